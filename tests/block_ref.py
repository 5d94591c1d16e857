"""Layer norm and the q/k prologue from positions, with their gradients, from the
definitions in float64 on the CPU, and the largest errors their roundings allow.

u is half a step of the stored type; sums of up to n fp32 terms are off by at most
n * 2^-24 of the sum of absolute values.
"""
from __future__ import annotations

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def norm(x, w, b, bounds, eps, add):
    """x [rows, C], w, b [segments, C] or None -> y, xhat, rstd, w per row."""
    x = x.double()
    wr = torch.ones_like(x) if w is None else torch.cat(
        [(w[s].double() + add).expand(bounds[s + 1] - bounds[s], -1) for s in range(len(bounds) - 1)])
    br = torch.zeros_like(x) if b is None else torch.cat(
        [b[s].double().expand(bounds[s + 1] - bounds[s], -1) for s in range(len(bounds) - 1)])
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).pow(2).mean(1, keepdim=True) + eps).rsqrt()
    xh = (x - mean) * rstd
    return xh * wr + br, xh, mean, rstd, wr, br


def norm_xhat_error(x, xh, rstd):
    """A row's sums have at most 64 serial and 12 tree steps: mean off by 2^-17 of the largest |x|,
    the variance by 2^-17 of itself (and the square of the former)."""
    return 2.0 ** -16 * (xh.abs() + x.double().abs().amax(1, keepdim=True) * rstd)


def norm_bound(x, y, xh, rstd, wr, br):
    return U[x.dtype] * y.abs() + norm_xhat_error(x, xh, rstd) * wr.abs() + 2.0 ** -22 * br.abs() + 1e-30


def norm_grads(dy, x, w, bounds, eps, add):
    """-> (dx, dw, db), bounds of their errors."""
    _, xh, _, rstd, wr, _ = norm(x, w, None, bounds, eps, add)
    dy = dy.double()
    a = dy * wr
    m1, m2 = a.mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
    dx = rstd * (a - m1 - xh * m2)
    seg = lambda t: torch.stack([t[bounds[s]:bounds[s + 1]].sum(0) for s in range(len(bounds) - 1)])  # noqa: E731
    ex = norm_xhat_error(x, xh, rstd)
    size = a.abs() + a.abs().mean(1, keepdim=True) + xh.abs() * (a * xh).abs().mean(1, keepdim=True)
    bx = U[x.dtype] * dx.abs() + rstd * (2.0 ** -15 * size + ex * m2.abs()
                                         + xh.abs() * (a.abs() * ex).mean(1, keepdim=True)) + 1e-30
    bw = seg(dy.abs() * (ex + 2.0 ** -16 * xh.abs())) + 1e-30
    bb = 2.0 ** -16 * seg(dy.abs()) + 1e-30
    return (dx, seg(dy * xh), seg(dy)), (bx, bw, bb)


def angles(pos, axes, theta):
    """pos [B, S, A] -> [B, S, 1, rot/2] angles."""
    out = []
    for a, d in enumerate(axes):
        n = torch.arange(d // 2, dtype=torch.float64)
        out.append(pos[..., a].double()[..., None] * theta ** (-2 * n / d))
    return torch.cat(out, -1)[:, :, None, :]


def rotate(x, ang):
    h = ang.shape[-1]
    a, b, rest = x[..., :h], x[..., h:2 * h], x[..., 2 * h:]
    c, s = ang.cos(), ang.sin()
    return torch.cat([a * c - b * s, a * s + b * c, rest], -1)


def pair_size(x, h):
    """|x_i| + |x_partner|: what a rotated value's fp32 error is relative to."""
    a, b, rest = x[..., :h].abs(), x[..., h:2 * h].abs(), x[..., 2 * h:].abs()
    return torch.cat([a + b, a + b, rest], -1)


def rope(x, ang, w, eps):
    """-> y and its bound.  The angle's sine and cosine and the norm are off by a few 2^-23."""
    x, w = x.double(), w.double()
    n = x * (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * w
    y = rotate(n, ang)
    return y, 2.0 ** -8 * y.abs() + 2.0 ** -19 * pair_size(n, ang.shape[-1]) + 1e-30


def rope_grads(dy, x, ang, w, eps):
    """-> (dx, dw), bounds."""
    dy, x, w = dy.double(), x.double(), w.double()
    h = ang.shape[-1]
    r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    g = rotate(dy, -ang)
    gs = pair_size(dy, h)
    gw = g * w
    dx = r * (gw - x * r * r * (x * gw).mean(-1, keepdim=True))
    bx = 2.0 ** -8 * dx.abs() + 2.0 ** -18 * r * (
        gs * w.abs() + x.abs() * r * r * (x.abs() * gs * w.abs()).mean(-1, keepdim=True)) + 1e-30
    return (dx, (g * x * r).sum((0, 1, 2))), (bx, 2.0 ** -16 * (gs * x.abs() * r).sum((0, 1, 2)) + 1e-30)
