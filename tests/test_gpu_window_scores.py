"""Windowed attention on the GPU with scores whose maximum moves along the sequence, and other scales.

Scores rise, fall and peak from stage to stage by up to 160 log2 units in some rows of a
wave and by none in others, so running maxima are refreshed, sums rescaled and partial
results of far-apart maxima merged; unit normal inputs do none of it.
"""
from __future__ import annotations

import math

import pytest
import torch

import h3attn
import window_ref as ref
from h3attn import autograd

pytestmark = pytest.mark.gpu
BF16, FP32 = ref.BF16, ref.FP32
DEFAULT = 1 / math.sqrt(128)
ROW_FACTORS = torch.tensor([0.0, 0.05, 1.0, -1.0, 4.0, -4.0, 0.3, -0.05, 2.0, 0.1, 4.0])
SHAPES = {
    "rise": lambda t: 2.5 * t,
    "fall": lambda t: 2.5 * (t.max() - t),
    "peaks": lambda t: torch.tensor([0.0, 6.0, 1.0, 6.0, 0.0, 3.0, 6.0])[t.long() % 7],
    "last": lambda t: torch.where(t == t.max(), 9.0, 0.0),
}


def inputs(gpu, B, H, Hkv, Sq, Skv, shape, scale, seed):
    """q, k, v, dout: scores of a row follow the shape over 64-key stages, times the row's factor (11.3 * factor * shape)."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    u = torch.randint(0, 2, (B, 1, Hkv, 128), generator=g) * 2.0 - 1
    b = SHAPES[shape](torch.arange(Skv) // 64).float()[None, :, None, None]
    a = ROW_FACTORS[(torch.arange(Sq)[:, None] + torch.arange(H)) % len(ROW_FACTORS)][None, :, :, None]
    q = a * u.repeat_interleave(H // Hkv, 2) + 0.3 * rnd(B, Sq, H, 128)
    k = (b * u + 0.3 * rnd(B, Skv, Hkv, 128)) * (DEFAULT / (scale or DEFAULT))
    return [t.to(torch.bfloat16).to(gpu).transpose(1, 2) for t in (q, k, rnd(B, Skv, Hkv, 128), rnd(B, Sq, H, 128))]


def by_definition(q, k, v, do, mask, scale):
    """One batch entry's heads of a key head: O, lse, dq, dk, dv and their bounds, in float64.

    A score's products and sum are off by 132 * 2^-24 of the absolute values' sum, its
    scaling by 2^-22 of itself; a weight by a factor of 1 + that, and as much again for the
    row's sum of weights (or its lse, 2^-21 of which its two roundings add); the factor 1.1
    is for e^x - 1 > x, x < 0.15.  The rest as in window_ref.
    """
    q, k, v, do = (t.double() for t in (q, k, v, do))
    s = q @ k.mT * scale
    hidden = s.masked_fill(~mask, -math.inf)
    lse = torch.logsumexp(hidden, -1, keepdim=True)
    p = torch.exp(hidden - lse)
    o = p @ v
    e = 132 * 2.0 ** -24 * (q.abs() @ k.abs().mT) * scale + 2.0 ** -22 * s.abs()
    e_row = (p * e).sum(-1, keepdim=True)
    assert (e + e_row)[p > 1e-9].max() < 0.1
    r = 1.1 * (e + e_row) + 2.0 ** -18
    bo = (p * (BF16 + FP32 + r)) @ v.abs() + (BF16 + FP32) * o.abs()
    r = r + 1.1 * 2.0 ** -21 * lse.abs()
    dp, delta = do @ v.mT, (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    size = do.abs() @ v.abs().mT
    e_delta = (do.abs() * bo).sum(-1, keepdim=True)
    e_ds = BF16 * ds.abs() + p * (r * (dp - delta).abs() + e_delta + 2 * FP32 * (size + delta.abs()))
    dq, dk, dv = scale * (ds @ k), scale * (ds.mT @ q).sum(0), (p.mT @ do).sum(0)
    bq = scale * ((e_ds + FP32 * ds.abs()) @ k.abs()) + (BF16 + FP32) * dq.abs()
    bk = scale * ((e_ds + FP32 * ds.abs()).mT @ q.abs()).sum(0) + (BF16 + FP32) * dk.abs()
    bv = ((p * (BF16 + 2 * FP32 + r)).mT @ do.abs()).sum(0) + (BF16 + FP32) * dv.abs()
    bl = 1.1 * e_row + 2.0 ** -21 * lse.abs() + 2.0 ** -18
    return {"O": (o, bo), "lse": (lse[..., 0], bl[..., 0]), "dq": (dq, bq), "dk": (dk, bk), "dv": (dv, bv)}


def stage_rises(q, k, mask, scale):
    """Largest rise of a row's score from the best of the earlier 64-key stages to a stage, in log2 units, by row."""
    s = (q.double() @ k.double().mT * scale / math.log(2)).masked_fill(~mask, -math.inf)
    top = torch.stack([t.amax(-1) for t in s.split(64, -1)], -1)
    before = torch.cummax(top, -1)[0][..., :-1]
    rise = (top[..., 1:] - before)[..., :]
    return torch.where(torch.isfinite(rise), rise, torch.zeros_like(rise)).amax(-1)


def check(gpu, B, H, Hkv, Sq, Skv, window, sinks, shape, scale=None, causal=False, grads=True, seed=0):
    q, k, v, do = inputs(gpu, B, H, Hkv, Sq, Skv, shape, scale, seed)
    kw = dict(window=window, sinks=sinks, causal=causal, scale=scale)
    got = dict(zip(("O", "lse"), h3attn.attn_fwd_window(q, k, v, return_lse=True, **kw)))
    if grads:
        got.update(zip(("dq", "dk", "dv"), h3attn.attn_bwd_window(do, q, k, v, got["O"], got["lse"], **kw)))
    mask = ref.visible(B, Sq, Skv, window, sinks, causal, None, None)
    rep, rises = H // Hkv, []
    for b, hk in {(0, 0), (B - 1, Hkv - 1), (0, Hkv // 2)}:
        heads = slice(hk * rep, (hk + 1) * rep)
        c = [t.cpu() for t in (q[b, heads], k[b, hk], v[b, hk], do[b, heads])]
        rises.append(stage_rises(c[0], c[1], mask[b], scale or DEFAULT).flatten())
        for name, (want, bound) in by_definition(*c, mask[b], scale or DEFAULT).items():
            if name in got:
                x = got[name][b, hk if name in ("dk", "dv") else heads].cpu().double()
                assert torch.isfinite(x).all(), name
                worst = ((x - want).abs() / (bound + 1e-30)).max().item()
                assert worst <= 1, f"{name} of head {hk}: error {worst:.3f} of what the roundings allow"
    return torch.cat(rises)


@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("B,H,Hkv,S", [(1, 2, 1, 700), (4, 40, 8, 700)], ids=["split", "tiles"])
@pytest.mark.parametrize("window,sinks,causal", [((None, None), 0, False), ((300, 150), 70, False), ((None, 0), 0, True)])
def test_moving_maxima(gpu, B, H, Hkv, S, window, sinks, causal, shape):
    rise = check(gpu, B, H, Hkv, S, S, window, sinks, shape, causal=causal, seed=S + H)
    if shape in ("rise", "last"):
        assert (rise > 128).any() and ((rise > 16) & (rise < 128)).any() and (rise < 8).any()


@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("B,H,Hkv,Sq,Skv", [(1, 28, 4, 1, 3000), (3, 14, 14, 1, 700), (1, 8, 1, 33, 2100), (2, 4, 2, 5, 1030)])
def test_moving_maxima_of_few_rows(gpu, B, H, Hkv, Sq, Skv, shape):
    """Pieces and waves whose maxima are far apart, merged."""
    check(gpu, B, H, Hkv, Sq, Skv, (None, 0), 0, shape if Skv < 1000 or shape != "rise" else "peaks", causal=True,
          grads=Sq > 1, seed=Skv)
    check(gpu, B, H, Hkv, Sq, Skv, (600, 0), 130, "last", causal=True, grads=False, seed=Skv + 1)


@pytest.mark.parametrize("scale", [0.03, 0.4, 1.0])
@pytest.mark.parametrize("B,H,Hkv,S", [(1, 2, 1, 300), (4, 40, 8, 300)], ids=["split", "tiles"])
@pytest.mark.parametrize("shape", ["peaks", "rise"])
def test_other_scales(gpu, B, H, Hkv, S, scale, shape):
    check(gpu, B, H, Hkv, S, S, (120, 90), 5, shape, scale=scale, seed=3)
    check(gpu, B, H, Hkv, 1, S, (120, 0), 5, shape, scale=scale, causal=True, grads=False, seed=4)


def test_autograd_passes_its_arguments_on(gpu):
    """Scale, eps and theta other than the defaults reach both passes."""
    q, k, v, do = inputs(gpu, 2, 4, 2, 150, 150, "peaks", 0.2, 1)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    kw = dict(window=(40, 20), sinks=3, scale=0.2)
    o = autograd.window_attention(*leaves, **kw)
    o.backward(do)
    want, lse = h3attn.attn_fwd_window(q, k, v, return_lse=True, **kw)
    assert torch.equal(o, want)
    for t, g in zip(leaves, h3attn.attn_bwd_window(do, q, k, v, want, lse, **kw)):
        assert torch.equal(t.grad, g)
    assert not torch.equal(o, h3attn.attn_fwd_window(q, k, v, window=(40, 20), sinks=3))
    pos = torch.arange(150, dtype=torch.int32, device=gpu)[:, None]
    w = torch.rand(128, device=gpu).to(torch.bfloat16).requires_grad_()
    qs, ks = (t.transpose(1, 2).clone().requires_grad_() for t in (q, k))
    kw = dict(eps=0.05, theta=300.0)
    yq, yk = autograd.qk_norm_rope(qs, ks, pos, (96,), w, w.detach(), **kw)
    dq, dk = torch.randn_like(yq), torch.randn_like(yk)
    torch.autograd.backward((yq, yk), (dq, dk))
    args = (qs.detach(), ks.detach(), pos, (96,), w.detach(), w.detach())
    for a, b in zip((yq, yk), h3attn.qk_rmsnorm_rope_axes(*args, **kw)):
        assert torch.equal(a, b)
    gq, gk, gw, _ = h3attn.qk_rmsnorm_rope_axes_bwd(dq, dk, *args, **kw)
    assert torch.equal(qs.grad, gq) and torch.equal(ks.grad, gk) and torch.equal(w.grad, gw.bfloat16())
    assert not torch.equal(yq, h3attn.qk_rmsnorm_rope_axes(*args)[0])
    x, s, b = (torch.randn(n, 64, device=gpu) for n in (12, 3, 3))
    xl, sl, bl = (t.clone().requires_grad_() for t in (x, s, b))
    y = autograd.layer_norm(xl, sl, bl, eps=0.3, segments=[0, 2, 7, 12], modulate=True)
    y.backward(dy := torch.randn_like(y))
    want, mean, rstd = h3attn.layer_norm_fwd(x, s, b, eps=0.3, segments=[0, 2, 7, 12], modulate=True, return_stats=True)
    assert torch.equal(y, want)
    for t, g in zip((xl, sl, bl), h3attn.layer_norm_bwd(dy, x, s, mean, rstd, segments=[0, 2, 7, 12], modulate=True)):
        assert torch.equal(t.grad, g)
