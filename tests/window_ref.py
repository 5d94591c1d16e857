"""Windowed attention and its gradients from their definition, in float64 on the CPU.

Written over an explicit mask and torch.autograd-free formulas; the tests also compare
them with central differences.
"""
from __future__ import annotations

import math

import torch


def visible(B, Sq, Skv, window, sinks, causal, q_start, kv_lens):
    """bool [B,Sq,Skv]: which keys a row sees."""
    left, right = (math.inf if n is None else n for n in window)
    starts = [Skv - Sq if q_start is None else q_start] * B if not isinstance(q_start, (list, tuple)) else q_start
    lens = [Skv] * B if kv_lens is None else [min(max(n, 0), Skv) for n in kv_lens]
    m = torch.zeros(B, Sq, Skv, dtype=torch.bool)
    for b in range(B):
        pos = starts[b] + torch.arange(Sq)[:, None]
        j = torch.arange(Skv)[None, :]
        see = ((j >= pos - left) & (j <= pos + right)) | (j < sinks)
        if causal:
            see &= j <= pos
        m[b] = see & (j < lens[b]) & (pos >= 0) & (pos < lens[b])
    return m


def forward(q, k, v, mask, scale):
    """-> O, lse, P in float64 (heads of k and v repeated to q's)."""
    rep = q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
    s = (q @ k.transpose(2, 3)) * scale
    s = s.masked_fill(~mask[:, None], -math.inf)
    lse = torch.logsumexp(s, dim=-1)
    p = torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[..., None])
    p = p.masked_fill(~mask[:, None], 0.0)
    return p @ v, lse, p


def backward(do, q, k, v, mask, scale):
    """-> dq, dk, dv in float64."""
    Hkv = k.shape[1]
    rep = q.shape[1] // Hkv
    o, _, p = forward(q, k, v, mask, scale)
    do, q = do.double() * mask.any(-1)[:, None, :, None], q.double()
    kk, vv = k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
    ds = p * (do @ vv.transpose(2, 3) - (do * o).sum(-1, keepdim=True)) * scale
    dk, dv = ds.transpose(2, 3) @ q, p.transpose(2, 3) @ do
    B, _, S, D = k.shape
    return ds @ kk, dk.view(B, Hkv, rep, S, D).sum(2), dv.view(B, Hkv, rep, S, D).sum(2)


# Rounding to bf16 is off by at most half a step: 2^-8 of the value.  P and dS are
# rounded for their products, results once more; everything else is fp32, whose
# share (the score's sum of 128 products, exp2, long sums) is bounded by FP32 of the
# sums of absolute values: 128 * 2^-24 for a dot product, and a score error e
# changes p by a factor of 1 + e, with |score| * 2^-22 below 2^-15 for |score| < 128.
BF16, FP32 = 2.0 ** -8, 2.0 ** -13


def forward_bound(q, k, v, mask, scale):
    """Largest |O - exact| that the roundings allow, per element."""
    o, _, p = forward(q, k, v, mask, scale)
    rep = q.shape[1] // k.shape[1]
    return (BF16 + FP32) * (p @ v.double().abs().repeat_interleave(rep, 1)) + (BF16 + FP32) * o.abs() + 1e-30


def backward_bounds(do, q, k, v, mask, scale):
    """The same for dq, dk, dv."""
    Hkv = k.shape[1]
    rep = q.shape[1] // Hkv
    o, _, p = forward(q, k, v, mask, scale)
    do, qa = do.double() * mask.any(-1)[:, None, :, None], q.double().abs()
    kk, vv = k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
    delta = (do * o).sum(-1, keepdim=True)
    dp = do @ vv.transpose(2, 3)
    ds = p * (dp - delta)
    # delta is taken from the rounded O, whose own error is forward_bound.
    e_delta = (do.abs() * forward_bound(q, k, v, mask, scale)).sum(-1, keepdim=True)
    size = do.abs() @ vv.abs().transpose(2, 3) + delta.abs()
    e_ds = BF16 * ds.abs() + p * (e_delta + 2 * FP32 * size)
    gq, gk, gv = backward(do, q, k, v, mask, scale)
    B, _, S, D = k.shape
    fold = lambda x: x.view(B, Hkv, rep, S, D).sum(2)  # noqa: E731
    bq = scale * (e_ds @ kk.abs() + FP32 * (ds.abs() @ kk.abs())) + (BF16 + FP32) * gq.abs()
    bk = scale * fold((e_ds + FP32 * ds.abs()).transpose(2, 3) @ qa) + (BF16 + FP32) * gk.abs()
    bv = (BF16 + 2 * FP32) * fold(p.transpose(2, 3) @ do.abs()) + (BF16 + FP32) * gv.abs()
    return bq + 1e-30, bk + 1e-30, bv + 1e-30
