"""Layer norm and the q/k prologue without a GPU: what is refused at the edges of their ranges."""
from __future__ import annotations

import pytest

from h3attn import block


def test_no_rows_of_weights():
    """A [0, C] weight is no weight for the rows, not a missing one."""
    for segments, rows in ((None, 6), (None, 0), ((0, 0), 0)):
        with pytest.raises(ValueError, match="one segment at least"):
            block._bounds(segments, rows, 0)
    assert list(block._bounds(None, 6, None)) == list(block._bounds(None, 6, 1)) == [0, 6]
