"""Windowed attention without a GPU: what is refused, before any HIP call."""
from __future__ import annotations

import ctypes

import pytest
import torch

import h3attn
from h3attn import _lib

S3 = _lib.strides3
ROW = S3(0, 0, 128)


def _fwd(L, q=16, k=16, v=16, o=16, lse=None, B=1, H=2, Hkv=1, Sq=4, Skv=4, D=128, st=(ROW,) * 4,
         w=(3, 3, 1, 0, 0), starts=None, lens=None, scale=0.1):
    win = None if w is None else ctypes.byref(_lib.Window(*w, starts, lens))
    return L.h3a_attn_fwd_window(q, k, v, o, lse, B, H, Hkv, Sq, Skv, D, *st, win, scale, None, 0, None)


def test_forward_refusals():
    L = _lib.lib()
    bad, unsup, align = _lib.H3A_ERR_INVALID_ARG, _lib.H3A_ERR_UNSUPPORTED, _lib.H3A_ERR_ALIGNMENT
    assert _fwd(L, q=None) == bad
    assert _fwd(L, w=None) == bad
    for size in ("B", "H", "Hkv", "Sq", "Skv"):
        assert _fwd(L, **{size: 0}) == bad
    assert _fwd(L, H=3, Hkv=2) == bad
    assert _fwd(L, D=64) == unsup
    assert _fwd(L, B=1 << 16, H=1 << 16) == unsup
    assert _fwd(L, Skv=(1 << 29) + 1) == bad
    for w in ((-1, 0, 0, 0, 0), (0, -1, 0, 0, 0), (0, 0, -1, 0, 0), (0, 0, 0, 0, 1), (0, 0, 0, 0, -1)):
        assert _fwd(L, w=w) == bad
    assert _fwd(L, Sq=5) == bad  # more rows than positions
    assert _fwd(L, scale=0.0) == bad and _fwd(L, scale=float("inf")) == bad
    assert _fwd(L, q=24) == align and _fwd(L, lse=18) == align and _fwd(L, lens=18) == align
    assert _fwd(L, st=(S3(0, 0, 12), ROW, ROW, ROW)) == align
    for i in range(4):
        st = [ROW] * 4
        st[i] = S3(0, 0, 1 << 24)
        assert _fwd(L, st=tuple(st)) == unsup
        assert b"sequence stride" in L.h3a_last_error()
    assert _fwd(L, st=(ROW, ROW, ROW, S3(0, 0, 120))) == bad
    assert b"rows overlap" in L.h3a_last_error()


def test_workspace_refusals():
    L = _lib.lib()
    n = ctypes.c_size_t(7)
    w = ctypes.byref(_lib.Window(3, 3, 1, 0, 0, None, None))
    size = L.h3a_attn_fwd_window_workspace_size
    assert size(1, 2, 1, 40, 40, 128, w, None) == _lib.H3A_ERR_INVALID_ARG
    assert size(1, 2, 1, 40, 40, 128, None, ctypes.byref(n)) == _lib.H3A_ERR_INVALID_ARG
    assert size(1, 2, 1, 40, 40, 64, w, ctypes.byref(n)) == _lib.H3A_ERR_UNSUPPORTED
    assert n.value == 7
    assert size(1, 2, 1, 8193, 8193, 128, w, ctypes.byref(n)) == 0 and n.value == 0  # more than 8192 rows: no split


def test_backward_refusals():
    L = _lib.lib()
    n = ctypes.c_size_t(0)
    w = ctypes.byref(_lib.Window(3, 3, 1, 0, 0, None, None))
    size = L.h3a_attn_bwd_window_workspace_size
    assert size(1, 2, 1, 4, 4, 128, w, None) == _lib.H3A_ERR_INVALID_ARG
    assert size(1, 2, 1, 4, 4, 128, None, ctypes.byref(n)) == _lib.H3A_ERR_INVALID_ARG
    assert size(1, 2, 1, 4, 4, 64, w, ctypes.byref(n)) == _lib.H3A_ERR_UNSUPPORTED
    assert size(1, 2, 1, 4, 4, 128, w, ctypes.byref(n)) == 0 and n.value > 0

    def bwd(ptrs=(16,) * 9, st=(ROW,) * 8, ws=16, nbytes=n.value):
        win = _lib.Window(3, 3, 1, 0, 0, None, None)
        return L.h3a_attn_bwd_window(*ptrs, 1, 2, 1, 4, 4, 128, *st, ctypes.byref(win), 0.1, ws, nbytes, None)

    for i in range(9):
        assert bwd(ptrs=tuple(None if i == j else 16 for j in range(9))) == _lib.H3A_ERR_INVALID_ARG
    for i in range(8):
        assert bwd(st=tuple(S3(0, 0, 12) if i == j else ROW for j in range(8))) == _lib.H3A_ERR_ALIGNMENT
    for i in (5, 6, 7):
        assert bwd(st=tuple(S3(0, 0, 64) if i == j else ROW for j in range(8))) == _lib.H3A_ERR_INVALID_ARG
    assert bwd(ws=None) == _lib.H3A_ERR_INVALID_ARG
    assert bwd(nbytes=n.value - 1) == _lib.H3A_ERR_INVALID_ARG
    assert bwd(ws=24) == _lib.H3A_ERR_ALIGNMENT


def test_python_refusals(monkeypatch):
    from h3attn import window
    q = torch.zeros(2, 4, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        h3attn.attn_fwd_window(q, q, q, (1, 1))
    monkeypatch.setattr(window, "_as_kernel_input", lambda name, t: (t, S3(*t.stride()[:3])))

    def refused(match, q=q, k=q, v=q, window=(1, 1), **kw):
        with pytest.raises(ValueError, match=match):
            h3attn.attn_fwd_window(q, k, v, window, **kw)

    refused("mismatch", k=q[:, :3], v=q[:, :3])
    refused("mismatch", k=q[:1], v=q[:1])
    refused("mismatch", v=q[:, :, :7])
    refused("empty", q=q[:, :, :0])
    refused("pair", window=3)
    refused("left side", window=(-1, 0))
    refused("right side", window=(0, 1.5))
    refused("sinks", sinks=-2)
    refused("causal", window=(4, 2), causal=True)
    refused("q_start", q_start=1)
    refused("q_start", q=q[:, :, :3], q_start=6)
    refused("needs q_start", q=q[:, :, :3], kv_lens=torch.zeros(2, dtype=torch.int32))
    refused("kv_lens", kv_lens=torch.zeros(2, dtype=torch.int64))
    refused("kv_lens", kv_lens=torch.zeros(3, dtype=torch.int32))
    refused("q_start", q_start=torch.zeros(4, dtype=torch.int32)[::2])
    refused("out must", out=q.float())
    lse = torch.zeros(2, 4, 8)
    with pytest.raises(ValueError, match="dout"):
        h3attn.attn_bwd_window(q.float(), q, q, q, q, lse, (1, 1))
    with pytest.raises(ValueError, match="lse"):
        h3attn.attn_bwd_window(q, q, q, q, q, lse[:, :, :7], (1, 1))


class Count:
    """A whole number that can be written to, as a 0-d tensor can."""

    def __init__(self, n):
        self.n = n

    def __index__(self):
        return self.n


def test_arguments_are_read_at_each_call():
    from h3attn import autograd, block, window
    cpu, n = torch.device("cpu"), Count(2)
    read = lambda: window._window([n, n], n, False, n, None, 1, 4, 16, cpu)[1]  # noqa: E731
    assert read() == (2, 2, 2, 0, 2)
    n.n = 3
    assert read() == (3, 3, 3, 0, 3)
    t = torch.tensor(5)
    assert window.mask_args((t, None), t) == ((5, None), 5)
    t += 1
    assert window.mask_args((t, None), t) == ((6, None), 6)
    pos = torch.zeros(4, 1, dtype=torch.int32)
    n.n = 32
    assert block._positions(pos, [n], 1e4, 1, 4, cpu)[1].dims[0] == 32
    n.n = 64
    assert block._positions(pos, [n], 1e4, 1, 4, cpu)[1].dims[0] == 64
    assert block.whole_numbers("segments", torch.tensor([0, 4, 9])) == (0, 4, 9)
    for bad in ([0, 1.5], [0, None], ["0"]):
        with pytest.raises(ValueError, match="segments must be whole numbers"):
            block.whole_numbers("segments", bad)
    q = torch.zeros(1, 1, 4, 128, dtype=torch.bfloat16)
    for kw in ({"window": (1, 0.5)}, {"window": (1, 1), "sinks": 2.0}, {"window": 4}):
        with pytest.raises(ValueError, match="window|sinks"):
            autograd.window_attention(q, q, q, **kw)


def test_backward_workspace_is_bounded():
    """First keys are cut into runs of queries that leave partial sums: a bounded number of them."""
    L = _lib.lib()
    n = ctypes.c_size_t(0)

    def size(B, H, Hkv, S, left, right, sinks):
        w = _lib.Window(left, right, sinks, 0, 0, None, None)
        assert L.h3a_attn_bwd_window_workspace_size(B, H, Hkv, S, S, 128, ctypes.byref(w), ctypes.byref(n)) == 0
        return n.value - 2 * 4 * B * H * S  # beside the rows' statistics

    run = 2 * 128 * 128 * 4
    for args in ((1, 56, 56, 42120, 0, 0, 42120), (1, 56, 8, 42120, 64, 64, 4096), (1, 1, 1, 1 << 22, 0, 0, 1 << 20),
                 (2, 56, 8, 8192, 16, 16, 256), (16, 56, 56, 8192, 0, 0, 2 ** 31 - 1), (1, 1, 1, 1 << 29, 0, 0, 1 << 29)):
        B, H, Hkv, S, left, right, sinks = args
        tiles = B * Hkv * ((min(sinks, S) + 127) // 128)
        assert 0 <= size(*args) <= (1024 + min(tiles, 1024)) * run + 512, args


def test_tiles_past_a_launch_are_refused():
    L = _lib.lib()
    assert _fwd(L, B=1 << 11, H=1 << 11, Hkv=1 << 11, w=None) == _lib.H3A_ERR_INVALID_ARG  # 2^22: sizes pass
    assert _fwd(L, B=(1 << 11) + 1, H=1 << 11, Hkv=1 << 11) == _lib.H3A_ERR_UNSUPPORTED
    assert _fwd(L, B=1 << 20, H=4, Hkv=4, Sq=129, Skv=129) == _lib.H3A_ERR_UNSUPPORTED
    assert b"tiles" in L.h3a_last_error()
