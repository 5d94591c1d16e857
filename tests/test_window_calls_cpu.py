"""Windowed attention without a GPU: what the entry points take and refuse at the edges of their ranges."""
from __future__ import annotations

import ctypes

from h3attn import _lib

S3 = _lib.strides3
ROW = S3(0, 0, 128)


def test_backward_rows_apart():
    """dout's and q's rows past a sequence's end have to read as zeros: rows that overlap are refused."""
    L = _lib.lib()
    n, w = ctypes.c_size_t(0), _lib.Window(3, 3, 1, 0, 0, None, None)
    assert L.h3a_attn_bwd_window_workspace_size(1, 2, 1, 4, 4, 128, ctypes.byref(w), ctypes.byref(n)) == 0
    for i, name in ((0, b"dout"), (1, b"q")):
        for stride in (0, 64, 120):
            st = tuple(S3(0, 0, stride) if i == j else ROW for j in range(8))
            assert L.h3a_attn_bwd_window(*(16,) * 9, 1, 2, 1, 4, 4, 128, *st, ctypes.byref(w), 0.1, None, n.value,
                                         None) == _lib.H3A_ERR_INVALID_ARG
            assert name + b" sequence stride" in L.h3a_last_error()
