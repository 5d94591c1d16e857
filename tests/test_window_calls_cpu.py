"""Windowed attention without a GPU: what the entry points take and refuse at the edges of their ranges."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from h3attn import _lib, autograd, window

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


def test_workspace_size_knows_no_positions():
    """Starts given per sequence may put more rows than keys; how many bytes a call needs does not depend on them."""
    L = _lib.lib()
    for fn in (L.h3a_attn_fwd_window_workspace_size, L.h3a_attn_bwd_window_workspace_size):
        if fn is L.h3a_attn_fwd_window_workspace_size:
            sizes = (1, 2, 1, 9000, 100, 128)  # (up to 8192 rows it asks the device)
        else:
            sizes = (1, 2, 1, 140, 100, 128)
        got = []
        for start, starts in ((0, None), (0, 16), (7, None)):
            n = ctypes.c_size_t(1)
            assert fn(*sizes, ctypes.byref(_lib.Window(3, 3, 1, 0, start, starts, None)), ctypes.byref(n)) == 0
            got.append(n.value)
        assert len(set(got)) == 1
    window._workspace_bytes.cache_clear()
    for _ in range(3):
        window._workspace_bytes("h3a_attn_bwd_window_workspace_size", (1, 2, 1, 140, 100, 128), (3, 3, 1, 0), 0)
    assert window._workspace_bytes.cache_info().misses == 1
    # A launch still checks where its rows are.
    w = _lib.Window(3, 3, 1, 0, 0, None, None)
    assert L.h3a_attn_fwd_window(16, 16, 16, 16, None, 1, 2, 1, 140, 100, 128, *(ROW,) * 4, ctypes.byref(w), 0.1, None,
                                 0, None) == _lib.H3A_ERR_INVALID_ARG
    assert b"rows must lie at positions" in L.h3a_last_error()


def test_the_backward_pass_sees_the_forwards_arguments(monkeypatch):
    """A start or a flag that is written to between the passes (numpy scalars, 0-d arrays) is read once."""
    calls = []
    monkeypatch.setattr(autograd._WindowAttention, "apply", lambda q, k, v, kw: calls.append(kw))
    start, causal = np.array(3), np.array(True)
    autograd.window_attention(None, None, None, (4, 0), causal=causal, q_start=start)
    start[...], causal[...] = 9, False
    assert calls[0]["q_start"] == 3 and type(calls[0]["q_start"]) is int and calls[0]["causal"] is True
    with pytest.raises(ValueError, match="q_start must be a whole number"):
        autograd.window_attention(None, None, None, (4, 0), q_start=1.5)
    lens = torch.zeros(2, dtype=torch.int32)
    autograd.window_attention(None, None, None, (4, 0), q_start=lens, kv_lens=lens)
    assert calls[1]["q_start"] is lens and calls[1]["causal"] is False
