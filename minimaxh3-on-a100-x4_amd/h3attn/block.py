"""What stands around a DiT block's attention, forward and backward: the layer norm with a
scale and shift per segment of the packed sequence, and the q/k prologue from positions
on several axes.  (ops.qk_rmsnorm_rope_ is the prologue on a caller's rotation table.)
"""
from __future__ import annotations

import ctypes
import functools
import operator

import torch

from . import _lib
from ._lib import check, lib, strides3
from .ops import HEAD_DIM, _layout, _on_device, _stream

DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16, torch.float32: _lib.FP32}


def whole_numbers(name: str, values) -> tuple:
    """values as plain ints: read now, whatever may be written to them later."""
    try:
        return tuple(map(operator.index, values))
    except TypeError:
        raise ValueError(f"{name} must be whole numbers, got {values!r}") from None


# ---------------------------------------------------------------------------
# q/k RMSNorm + rotary embedding from positions
def _rope_input(name: str, t: torch.Tensor, device=None):
    """A bf16 [B,S,H,128] GPU tensor that can be read in place, or a copy, and its strides."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16 or t.dim() != 4 or t.shape[-1] != HEAD_DIM:
        raise ValueError(f"{name} must be a bf16 tensor [B,S,H,{HEAD_DIM}]")
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{name} must be a GPU tensor, all on one device")
    st = _layout(t)
    if st is None:
        t = t.clone(memory_format=torch.contiguous_format)
        st = t.stride()[:3]
    return t, strides3(*st)


def _rope_output(name: str, t, shape, device):
    if t is None:
        t = torch.empty(shape, dtype=torch.bfloat16, device=device)
    elif not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype != torch.bfloat16 or t.device != device:
        raise ValueError(f"{name} must be a bf16 tensor {tuple(shape)} on q's device")
    st = _layout(t)
    if st is None:
        raise ValueError(f"{name} must have unit last stride, 16-byte alignment and strides multiple of 8")
    return t, strides3(*st)


def _rope_weight(name: str, w: torch.Tensor, device) -> torch.Tensor:
    """The weights as the kernels read them: bf16, as in qk_rmsnorm_rope_ (a model's are; others are rounded)."""
    if w.numel() != HEAD_DIM:
        raise ValueError(f"{name} must have {HEAD_DIM} elements")
    if w.dtype != torch.bfloat16 or w.device != device or not w.is_contiguous() or w.data_ptr() & 15:
        w = w.detach().reshape(HEAD_DIM).to(device=device, dtype=torch.bfloat16, copy=True).contiguous()
    return w


@functools.lru_cache(maxsize=256)
def _axes_dims(axes: tuple):
    """Checked rotated dims of each axis as the entry points take them."""
    if not 1 <= len(axes) <= _lib.MAX_AXES:
        raise ValueError(f"axes must name the rotated dims of 1 to {_lib.MAX_AXES} axes, got {axes}")
    if any(d <= 0 or d % 2 for d in axes) or sum(axes) > HEAD_DIM or sum(axes) % 16:
        raise ValueError(f"axes {axes}: even dims that add up to a multiple of 16, at most {HEAD_DIM}")
    return (ctypes.c_int * _lib.MAX_AXES)(*axes)


def _positions(pos: torch.Tensor, axes, theta, B: int, S: int, device):
    axes = whole_numbers("axes", axes)
    dims, A, shape = _axes_dims(axes), len(axes), pos.shape
    if pos.dtype not in (torch.int32, torch.float32) or pos.device != device:
        raise ValueError(f"positions must be int32 or float32 on q's device, got {pos.dtype} on {pos.device}")
    if shape[-2:] != (S, A) or len(shape) > 3 or (len(shape) == 3 and shape[0] not in (1, B)):
        raise ValueError(f"positions {tuple(shape)} must be [S, axes] or [B, S, axes] (B={B}, S={S}, axes {axes})")
    pos = pos.contiguous()
    stride = S * A if len(shape) == 3 and shape[0] == B else 0
    return pos, _lib.Positions(pos.data_ptr(), stride, 1 if pos.dtype == torch.float32 else 0, A, dims, float(theta))


def _rope_prepare(q, k, pos, axes, qw, kw, theta):
    q, qst = _rope_input("q", q)
    k, kst = _rope_input("k", k, q.device)
    B, S, Hq, D = q.shape
    if tuple(k.shape[:2]) != (B, S):
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must share batch and sequence")
    if 0 in (B, S, Hq, k.shape[2]):
        raise ValueError("empty q or k")
    pos, p = _positions(pos, axes, theta, B, S, q.device)
    return (q, k, pos, _rope_weight("qw", qw, q.device), _rope_weight("kw", kw, q.device)), p, \
        (B, S, Hq, k.shape[2], D), (qst, kst)


def qk_rmsnorm_rope_axes(q: torch.Tensor, k: torch.Tensor, pos: torch.Tensor, axes, qw: torch.Tensor,
                         kw: torch.Tensor, eps: float = 1e-6, theta: float = 10000.0, out=None):
    """Per-head RMSNorm and split-half RoPE from positions: q [B,S,Hq,128], k [B,S,Hk,128] bf16 -> (q', k').

    pos: int32 or float32 [S, A] or [B, S, A], a token's position on each of A axes
    (time, height, width).  axes: rotated dims of each axis, even numbers whose sum
    rot is a multiple of 16; pair (i, i + rot/2) belongs to the axis whose dims/2
    pairs hold i, and as its n-th pair turns by pos * theta^(-2n/dims).  With one
    axis these are the rotations of rope_freqs.  Dims from rot on are only normalised.
    qw, kw: 128 weights, used in bf16: those of another dtype are rounded to it first.
    out: (q', k') to write, for instance (q, k) themselves.
    """
    (q, k, pos, qw, kw), p, sizes, (qst, kst) = _rope_prepare(q, k, pos, axes, qw, kw, theta)
    oq, ok = (None, None) if out is None else out
    oq, oqst = _rope_output("out[0]", oq, q.shape, q.device)
    ok, okst = _rope_output("out[1]", ok, k.shape, q.device)
    with _on_device(q):
        rc = lib().h3a_qk_rmsnorm_rope_axes(q.data_ptr(), k.data_ptr(), oq.data_ptr(), ok.data_ptr(), *sizes, qst, kst,
                                            oqst, okst, ctypes.byref(p), qw.data_ptr(), kw.data_ptr(), float(eps),
                                            _stream(q))
    check("h3a_qk_rmsnorm_rope_axes", rc)
    return oq, ok


@functools.lru_cache(maxsize=256)
def _rope_bwd_bytes(B: int, S: int) -> int:
    n = ctypes.c_size_t(0)
    check("h3a_qk_rmsnorm_rope_axes_bwd_workspace_size",
          lib().h3a_qk_rmsnorm_rope_axes_bwd_workspace_size(B, S, ctypes.byref(n)))
    return n.value


def qk_rmsnorm_rope_axes_bwd(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, pos: torch.Tensor,
                             axes, qw: torch.Tensor, kw: torch.Tensor, eps: float = 1e-6, theta: float = 10000.0):
    """Gradients of qk_rmsnorm_rope_axes from those of its outputs: (q's, k's, qw's, kw's).

    q and k are the forward's inputs.  The weights' gradients are fp32 [128], summed
    over all rows in a fixed order, at the weights as the forward uses them (in bf16).
    """
    (q, k, pos, qw, kw), p, (B, S, Hq, Hk, D), (qst, kst) = _rope_prepare(q, k, pos, axes, qw, kw, theta)
    if dq.shape != q.shape or dk.shape != k.shape:
        raise ValueError(f"gradients {tuple(dq.shape)}, {tuple(dk.shape)} must have the shapes of q and k")
    dq, dqst = _rope_input("dq", dq, q.device)
    dk, dkst = _rope_input("dk", dk, q.device)
    gq, gqst = _rope_output("dq", None, q.shape, q.device)
    gk, gkst = _rope_output("dk", None, k.shape, q.device)
    gqw, gkw = (torch.empty(D, dtype=torch.float32, device=q.device) for _ in range(2))
    nbytes = _rope_bwd_bytes(B, S)
    with _on_device(q):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        rc = lib().h3a_qk_rmsnorm_rope_axes_bwd(dq.data_ptr(), dk.data_ptr(), q.data_ptr(), k.data_ptr(), gq.data_ptr(),
                                                gk.data_ptr(), gqw.data_ptr(), gkw.data_ptr(), B, S, Hq, Hk, D,
                                                dqst, dkst, qst, kst, gqst, gkst, ctypes.byref(p), qw.data_ptr(),
                                                kw.data_ptr(), float(eps), ws.data_ptr(), nbytes, _stream(q))
    check("h3a_qk_rmsnorm_rope_axes_bwd", rc)
    return gq, gk, gqw, gkw


# ---------------------------------------------------------------------------
# layer norm
@functools.lru_cache(maxsize=256)
def _bounds(segments, rows: int, groups):
    """Checked bounds of the segments as the entry points take them; None: `groups` equal ones."""
    if rows > 2 ** 30:
        raise ValueError(f"{rows} rows unsupported (at most 2^30)")
    if groups == 0:
        raise ValueError("weight and bias must have a row for one segment at least")
    if segments is None:
        groups = groups or 1
        if rows % groups:
            raise ValueError(f"{rows} rows do not split evenly into {groups} segments: pass their bounds")
        segments = tuple(i * (rows // groups) for i in range(groups + 1))
    if len(segments) < 2 or segments[0] != 0 or segments[-1] != rows or \
            any(b < a for a, b in zip(segments, segments[1:])):
        raise ValueError(f"segments must be non-decreasing bounds from 0 to {rows} rows, got {segments}")
    if groups is not None and groups != len(segments) - 1:
        raise ValueError(f"{len(segments) - 1} segments, but weights for {groups}")
    return (ctypes.c_int * len(segments))(*segments)


@functools.lru_cache(maxsize=256)
def _norm_bwd_bytes(split: tuple, C: int) -> int:
    """Workspace bytes of the weights' gradients; split: the arguments of _bounds."""
    bounds, n = _bounds(*split), ctypes.c_size_t(0)
    check("h3a_layer_norm_bwd_workspace_size",
          lib().h3a_layer_norm_bwd_workspace_size(bounds, len(bounds) - 1, C, ctypes.byref(n)))
    return n.value


def _norm_rows(name: str, t: torch.Tensor, C: int) -> torch.Tensor:
    """t as [rows, C] with unit last stride and rows that do not overlap, copied where it has to be."""
    if t.dim() == 2 and t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) >= C):
        return t
    t2 = t.reshape(-1, C) if t.numel() else t.new_empty((t.numel() // max(C, 1), C))
    if (t2.stride(1) == 1 or C == 1) and (t2.shape[0] <= 1 or t2.stride(0) >= C):
        return t2
    return t2.contiguous()


def _norm_prepare(x, weight, bias, segments):
    if not isinstance(x, torch.Tensor) or x.dtype not in DTYPES or x.dim() < 1:
        raise ValueError("x must be a bf16, fp16 or fp32 tensor [..., C]")
    if not x.is_cuda:
        raise ValueError("x must be a GPU tensor (libh3attn has no CPU path)")
    C = x.shape[-1]
    if not 0 < C <= 16384:
        raise ValueError(f"{C} channels unsupported (1 to 16384)")
    rows = x.numel() // C
    groups = None
    affine = [(n, t) for n, t in (("weight", weight), ("bias", bias)) if t is not None]
    for name, t in affine:
        if t.dtype not in DTYPES or t.device != x.device or t.dim() not in (1, 2) or t.shape[-1] != C:
            raise ValueError(f"{name} must be a bf16, fp16 or fp32 tensor [{C}] or [segments, {C}] on x's device")
        if t.dtype != affine[0][1].dtype:
            raise ValueError("weight and bias must share a dtype")
        n = t.shape[0] if t.dim() == 2 else 1
        if groups is not None and n != groups:
            raise ValueError("weight and bias must have the same segments")
        groups = n
    split = (None if segments is None else whole_numbers("segments", segments), rows, groups)
    dt = DTYPES[affine[0][1].dtype] if affine else _lib.FP32
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    return rows, C, split, _bounds(*split), dt, weight, bias


def _ptr(t):
    return None if t is None else t.data_ptr()


def layer_norm_fwd(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                   eps: float = 1e-6, segments=None, modulate: bool = False, return_stats: bool = False):
    """Layer norm of x [..., C] over C: (x - mean) * rstd * weight + bias, in x's dtype.

    weight, bias: [C], or [n, C] with a row for each of n contiguous segments of x's
    rows.  segments: their n + 1 bounds, from 0 to the number of rows (empty ones
    allowed); without it the rows split evenly, as samples of a batch.  modulate:
    (1 + weight) in weight's place, as adaLN scales.  x: bf16, fp16 or fp32, C up to
    16384; weight and bias any of these.  Returns y, with return_stats (y, mean, rstd),
    the fp32 [rows] statistics that layer_norm_bwd takes.
    """
    rows, C, _, bounds, dt, weight, bias = _norm_prepare(x, weight, bias, segments)
    x2 = _norm_rows("x", x, C)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean, rstd = (torch.empty(rows, dtype=torch.float32, device=x.device) if return_stats else None for _ in range(2))
    with _on_device(x):
        rc = lib().h3a_layer_norm_fwd(x2.data_ptr(), x2.stride(0), _ptr(weight), _ptr(bias), y.data_ptr(), C,
                                      _ptr(mean), _ptr(rstd), rows, C,
                                      DTYPES[x.dtype], dt, bounds, len(bounds) - 1, 1 if modulate else 0,
                                      float(eps), _stream(x))
    check("h3a_layer_norm_fwd", rc)
    return (y, mean, rstd) if return_stats else y


def layer_norm_bwd(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None, mean: torch.Tensor,
                   rstd: torch.Tensor, segments=None, modulate: bool = False, param_grads: bool = True):
    """Gradients (dx, dweight, dbias) of layer_norm_fwd from dy, its x and weight and its statistics.

    dx in x's dtype.  dweight and dbias are fp32, summed over each segment's rows in
    a fixed order, [C], or [n, C] where weight is or segments are given; None without
    param_grads.
    """
    rows, C, split, bounds, dt, weight, _ = _norm_prepare(x, weight, None, segments)
    if not isinstance(dy, torch.Tensor) or dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError("dy must be a tensor like x")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.shape != (rows,) or t.dtype != torch.float32 or t.device != x.device or not t.is_contiguous():
            raise ValueError(f"{name} must be the forward's fp32 [{rows}] statistics")
    x2, dy2 = _norm_rows("x", x, C), _norm_rows("dy", dy, C)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    n = len(bounds) - 1
    dw = db = ws = None
    nbytes = 0
    with _on_device(x):
        if param_grads:
            shape = C if n == 1 and (weight is None or weight.dim() == 1) else (n, C)
            dw, db = (torch.empty(shape, dtype=torch.float32, device=x.device) for _ in range(2))
            nbytes = _norm_bwd_bytes(split, C)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        rc = lib().h3a_layer_norm_bwd(dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), x2.stride(0), _ptr(weight),
                                      mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), C, _ptr(dw), _ptr(db), rows, C,
                                      DTYPES[x.dtype], dt, bounds, n, 1 if modulate else 0, _ptr(ws), nbytes,
                                      _stream(x))
    check("h3a_layer_norm_bwd", rc)
    return dx, dw, db
