"""Differentiable forms of the operators that have a backward pass, for training.

Each is a torch.autograd.Function over the forward and backward entry points: inputs are
saved as they are given, statistics in fp32, and nothing is recomputed but what the
backward kernels recompute themselves.  Gradients that are not asked for are not returned;
the attention's and the prologue's backward passes take their full time all the same (the
layer norm's leaves its weights' gradients out).

A backward pass is captured into a HIP graph as torch's own are: on leaves that no eager
graph still alive holds (torch.autograd.grad on fresh leaves, or after such graphs are
gone), since their accumulation would run on the other graph's stream.
"""
from __future__ import annotations

import torch

from .block import layer_norm_bwd, layer_norm_fwd, qk_rmsnorm_rope_axes, qk_rmsnorm_rope_axes_bwd, whole_numbers
from .window import attn_bwd_window, attn_fwd_window, mask_args, whole_number


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kw):
        o, lse = attn_fwd_window(q, k, v, return_lse=True, **kw)
        # kv_lens and q_start take part in the backward pass: saved, so that a later write to
        # them is noticed.
        tensors = {n: t for n, t in kw.items() if isinstance(t, torch.Tensor)}
        ctx.kw = {n: t for n, t in kw.items() if n not in tensors}
        ctx.names = tuple(tensors)
        ctx.save_for_backward(q, k, v, o, lse, *tensors.values())
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, *tensors = ctx.saved_tensors
        dq, dk, dv = attn_bwd_window(do, q, k, v, o, lse, **ctx.kw, **dict(zip(ctx.names, tensors)))
        need = ctx.needs_input_grad
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None


def window_attention(q, k, v, window, sinks: int = 0, causal: bool = False, scale: float | None = None,
                     q_start=None, kv_lens=None) -> torch.Tensor:
    """attn_fwd_window with gradients for q, k and v."""
    window, sinks = mask_args(window, sinks)
    scale = None if scale is None else float(scale)
    if q_start is not None and not isinstance(q_start, torch.Tensor):
        q_start = whole_number("q_start", q_start)
    kw = dict(window=window, sinks=sinks, causal=bool(causal), scale=scale, q_start=q_start, kv_lens=kv_lens)
    return _WindowAttention.apply(q, k, v, kw)


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, qw, kw, axes, eps, theta):
        ctx.save_for_backward(q, k, pos, qw, kw)
        ctx.args = (axes, eps, theta)
        return qk_rmsnorm_rope_axes(q, k, pos, axes, qw, kw, eps=eps, theta=theta)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        q, k, pos, qw, kw = ctx.saved_tensors
        axes, eps, theta = ctx.args
        gq, gk, gqw, gkw = qk_rmsnorm_rope_axes_bwd(dq, dk, q, k, pos, axes, qw, kw, eps=eps, theta=theta)
        need = ctx.needs_input_grad
        return (gq if need[0] else None, gk if need[1] else None, None,
                gqw.to(qw.dtype).view_as(qw) if need[3] else None, gkw.to(kw.dtype).view_as(kw) if need[4] else None,
                None, None, None)


def qk_norm_rope(q, k, pos, axes, qw, kw, eps: float = 1e-6, theta: float = 10000.0):
    """qk_rmsnorm_rope_axes (out of place) with gradients for q, k and the weights, those in the weights' dtype.

    Weights kept in fp32 take part rounded to bf16, in both passes: their gradients are
    not rounded, but an update of less than half a bf16 step (2^-8 of the weight) shows in
    the output only once such updates have added up to it.
    """
    return _QkNormRope.apply(q, k, pos, qw, kw, whole_numbers("axes", axes), float(eps), float(theta))


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, segments, modulate):
        y, mean, rstd = layer_norm_fwd(x, weight, bias, eps=eps, segments=segments, modulate=modulate, return_stats=True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.args = (segments, modulate)
        ctx.params = tuple(None if t is None else (t.dtype, t.shape) for t in (weight, bias))
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        segments, modulate = ctx.args
        need = ctx.needs_input_grad
        if segments is None and weight is None and ctx.params[1] is not None:
            # The bias alone says how the rows split.
            n, rows = (1 if len(ctx.params[1][1]) == 1 else ctx.params[1][1][0]), mean.shape[0]
            segments = tuple(i * (rows // n) for i in range(n + 1))
        dx, dw, db = layer_norm_bwd(dy, x, weight, mean, rstd, segments=segments, modulate=modulate,
                                    param_grads=need[1] or need[2])
        grads = [None if not want else g.to(p[0]).reshape(p[1]) for want, g, p in
                 zip(need[1:3], (dw, db), ctx.params)]
        return dx if need[0] else None, *grads, None, None, None


def layer_norm(x, weight=None, bias=None, eps: float = 1e-6, segments=None, modulate: bool = False) -> torch.Tensor:
    """layer_norm_fwd with gradients for x, weight and bias, each in its own dtype."""
    segments = None if segments is None else whole_numbers("segments", segments)
    return _LayerNorm.apply(x, weight, bias, float(eps), segments, bool(modulate))
