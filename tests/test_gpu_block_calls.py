"""Layer norm and the q/k prologue on the GPU: calls that are easily got wrong."""
from __future__ import annotations

import pytest
import torch

import h3attn
from h3attn import autograd

pytestmark = pytest.mark.gpu


def test_weights_for_no_segment(gpu):
    x, none = torch.randn(6, 64, device=gpu), torch.empty(0, 64, device=gpu)
    for fn in (h3attn.layer_norm_fwd, autograd.layer_norm):
        for args in ((none,), (none, none), (None, none)):
            with pytest.raises(ValueError, match="one segment at least"):
                fn(x, *args)
    _, mean, rstd = h3attn.layer_norm_fwd(x, return_stats=True)
    with pytest.raises(ValueError, match="one segment at least"):
        h3attn.layer_norm_bwd(x, x, none, mean, rstd)
