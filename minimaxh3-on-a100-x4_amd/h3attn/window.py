"""Attention over a sliding window with a few first keys that stay visible, forward and backward.

For windowed layers of the DiT, whose text tokens come first in the packed sequence
and are seen by every video token, and for the single new token of a causal model
against its cache of keys.  The gradients are those of the same mask; h3attn.autograd
wraps both in a differentiable function.
"""
from __future__ import annotations

import ctypes
import functools
import math
import operator

import torch

from . import _lib
from ._lib import check, lib, strides3
from .ops import HEAD_DIM, _as_kernel_input, _layout, _on_device, _stream


# Query rows up to which the forward may split the keys, and need a workspace.
SPLIT_ROWS = 8192


def whole_number(name: str, n) -> int:
    """n as a plain int: read now, whatever may be written to it later."""
    try:
        return operator.index(n)
    except TypeError:
        raise ValueError(f"{name} must be a whole number, got {n!r}") from None


def _side(name: str, n) -> int:
    """A window side; None is no limit."""
    if n is None:
        return 2 ** 31 - 1
    if n < 0:
        raise ValueError(f"{name} must be a whole number >= 0 (or None for no limit), got {n}")
    return min(n, 2 ** 31 - 1)


def mask_args(window, sinks):
    """The window and the number of first keys as plain ints (None: no limit)."""
    if not isinstance(window, (tuple, list)) or len(window) != 2:
        raise ValueError(f"window must be a pair (left, right), got {window!r}")
    left, right = window
    if type(left) is int and type(right) is int and type(sinks) is int:
        return (left, right), sinks
    if type(left) is not int and left is not None:
        left = whole_number("window's left side", left)
    if type(right) is not int and right is not None:
        right = whole_number("window's right side", right)
    if type(sinks) is not int and sinks is not None:
        sinks = whole_number("sinks", sinks)
    return (left, right), sinks


def _per_sequence(name: str, t: torch.Tensor, B: int, device) -> int:
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != B or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor [{B}] on q's device, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


@functools.lru_cache(maxsize=1024)
def _sides(window, sinks, causal, start, Sq, Skv):
    """(left, right, sinks, causal, start) of a checked window, all from plain values; start None: given per sequence."""
    left, right = _side("window's left side", window[0]), _side("window's right side", window[1])
    if causal and window[1] not in (0, None):
        raise ValueError(f"a causal window has no right side, got {window[1]}")
    if start is not None and not 0 <= start <= Skv - Sq:
        raise ValueError(f"q_start {start}: rows must lie at positions 0 .. Skv - 1 (Sq={Sq}, Skv={Skv})")
    return left, right, _side("sinks", sinks), 1 if causal else 0, 0 if start is None else start


def _window(window, sinks, causal, q_start, kv_lens, B, Sq, Skv, device):
    """The call's h3a_window, and its (left, right, sinks, causal, start), of which a workspace's size depends on the
    first four."""
    window, sinks = mask_args(window, sinks)
    lens = None if kv_lens is None else _per_sequence("kv_lens", kv_lens, B, device)
    starts = None
    if isinstance(q_start, torch.Tensor):
        starts, start = _per_sequence("q_start", q_start, B, device), None
    elif q_start is not None:
        start = whole_number("q_start", q_start)
    elif lens is not None and Sq != Skv:
        raise ValueError("kv_lens with Sq != Skv needs q_start: where the queries sit in the sequences")
    else:
        start = Skv - Sq
    sides = _sides(window, sinks, bool(causal), start, Sq, Skv)
    return _lib.Window(*sides, starts, lens), sides


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(fn: str, sizes: tuple, sides: tuple, device_index: int) -> int:
    """Workspace bytes of entry point fn on the device, which is the current one; sides: (left, right, sinks, causal)."""
    left, right, sinks, causal = sides
    w, n = _lib.Window(left, right, sinks, causal, 0, None, None), ctypes.c_size_t(0)
    check(fn, getattr(lib(), fn)(*sizes, ctypes.byref(w), ctypes.byref(n)))
    return n.value


def _prepare(q, k, v):
    q, qst = _as_kernel_input("q", q)
    k, kst = _as_kernel_input("k", k)
    v, vst = _as_kernel_input("v", v)
    B, H, Sq, D = q.shape
    Hkv, Skv = k.shape[1:3]
    if k.shape != v.shape or k.shape[0] != B or Hkv == 0 or H % Hkv:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)} k {tuple(k.shape)} v {tuple(v.shape)}")
    if 0 in (B, H, Sq, Skv):
        raise ValueError("empty attention input")
    if not (q.device == k.device == v.device):
        raise ValueError("q, k, v must be on the same device")
    return q, k, v, (B, H, Hkv, Sq, Skv, D), (qst, kst, vst)


def _check_like(name: str, t: torch.Tensor, q: torch.Tensor):
    if not isinstance(t, torch.Tensor) or t.shape != q.shape or t.dtype != torch.bfloat16 or t.device != q.device:
        raise ValueError(f"{name} must be a bf16 tensor {tuple(q.shape)} on its device")


def attn_fwd_window(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window, sinks: int = 0, causal: bool = False,
                    scale: float | None = None, out: torch.Tensor | None = None, q_start=None,
                    kv_lens: torch.Tensor | None = None, return_lse: bool = False):
    """Windowed attention, q [B,H,Sq,128], k/v [B,Hkv,Skv,128] bf16 (Hkv divides H) -> O [B,H,Sq,128].

    window: (left, right) keys seen to either side of a query's position, None for
    no limit; sinks: first keys seen from every position; causal: no key past the
    position (the window's right side is then 0 or None).
    q_start: position of the first query row, an int or an int32 GPU tensor [B];
    the default is Skv - Sq (the queries are the last rows), or 0 where Sq == Skv.
    kv_lens: int32 GPU tensor [B], the sequences' lengths in a padded batch or a
    cache; with Sq != Skv it needs q_start (kv_lens - 1 for one new token).  Rows
    at positions outside [0, kv_lens) give O = 0 and lse = -inf.
    return_lse: also the log-sum-exp of the scaled scores, fp32 [B,H,Sq], which
    attn_bwd_window takes.  Strides and `out` as for attn_fwd.
    """
    q, k, v, (B, H, Hkv, Sq, Skv, D), st = _prepare(q, k, v)
    w, sides = _window(window, sinks, causal, q_start, kv_lens, B, Sq, Skv, q.device)
    if out is None:
        out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
        ost = out.stride()[:3]
    else:
        _check_like("out", out, q)
        ost = _layout(out)
        if ost is None:
            raise ValueError("out must have unit last stride, 16-byte alignment and strides multiple of 8")
    lse = torch.empty((B, H, Sq), dtype=torch.float32, device=q.device) if return_lse else None
    sc = 1.0 / math.sqrt(D) if scale is None else float(scale)
    with _on_device(q):
        ws, nbytes = None, 0
        if Sq <= SPLIT_ROWS:
            nbytes = _workspace_bytes("h3a_attn_fwd_window_workspace_size", (B, H, Hkv, Sq, Skv, D), sides[:4],
                                      q.get_device())
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        rc = lib().h3a_attn_fwd_window(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                       None if lse is None else lse.data_ptr(), B, H, Hkv, Sq, Skv, D, *st,
                                       strides3(*ost), ctypes.byref(w), sc, None if ws is None else ws.data_ptr(), nbytes,
                                       _stream(q))
    check("h3a_attn_fwd_window", rc)
    return (out, lse) if return_lse else out


def _rows_apart(name: str, t: torch.Tensor):
    """t and its strides with rows that do not overlap and lie on the 16-byte grid, copied where they do not: a
    gradient may be expanded over the sequence (that of a mean) or a piece of a larger one (that of a concatenation)."""
    t, st = _as_kernel_input(name, t)
    if (t.shape[2] > 1 and st[2] < HEAD_DIM) or t.data_ptr() & 15:
        t, st = _as_kernel_input(name, t.clone(memory_format=torch.contiguous_format))
    return t, st


def _grad_like(t: torch.Tensor):
    """A tensor for t's gradient, in t's order of dimensions where the kernels can write it."""
    g = torch.empty_like(t)
    st = _layout(g)
    if st is None or (g.shape[2] > 1 and st[2] < HEAD_DIM):
        g = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        st = _layout(g)
    return g, strides3(*st)


def attn_bwd_window(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                    lse: torch.Tensor, window, sinks: int = 0, causal: bool = False, scale: float | None = None,
                    q_start=None, kv_lens: torch.Tensor | None = None):
    """Gradients (dq, dk, dv) of attn_fwd_window from dout, its inputs, its O and its lse (return_lse=True).

    window .. kv_lens as in the forward call.  dk and dv sum over the heads that
    share a key head.  The sums run in a fixed order: equal calls give equal bits.
    """
    q, k, v, (B, H, Hkv, Sq, Skv, D), st = _prepare(q, k, v)
    _check_like("dout", dout, q)
    _check_like("o", o, q)
    q, qst = _rows_apart("q", q)
    dout, gst = _rows_apart("dout", dout)
    o, ost = _as_kernel_input("o", o)
    if lse.shape != (B, H, Sq) or lse.dtype != torch.float32 or lse.device != q.device or not lse.is_contiguous():
        raise ValueError(f"lse must be the forward's fp32 [{B},{H},{Sq}] tensor")
    w, sides = _window(window, sinks, causal, q_start, kv_lens, B, Sq, Skv, q.device)
    (dq, dqst), (dk, dkst), (dv, dvst) = _grad_like(q), _grad_like(k), _grad_like(v)
    sc = 1.0 / math.sqrt(D) if scale is None else float(scale)
    with _on_device(q):
        nbytes = _workspace_bytes("h3a_attn_bwd_window_workspace_size", (B, H, Hkv, Sq, Skv, D), sides[:4],
                                  q.get_device())
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        rc = lib().h3a_attn_bwd_window(dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                       lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), B, H, Hkv, Sq,
                                       Skv, D, gst, qst, *st[1:], ost, dqst, dkst, dvst, ctypes.byref(w), sc, ws.data_ptr(),
                                       nbytes, _stream(q))
    check("h3a_attn_bwd_window", rc)
    return dq, dk, dv
