"""Windowed attention on the GPU: infinities and NaN that are seen, and what they cost."""
from __future__ import annotations

import math

import pytest
import torch

import h3attn
import window_ref as ref
from test_gpu_window import SCALE, make

pytestmark = pytest.mark.gpu
BF16, FP32 = ref.BF16, ref.FP32


def seen_sum(w, y, mask):
    """sum over j of w[i,j] * y[j] over the pairs of the mask alone, for each i (float64)."""
    out = torch.empty(w.shape[0], y.shape[1], dtype=torch.float64)
    for i in range(w.shape[0]):
        at = mask[i]
        out[i] = (w[i, at, None] * y[at]).sum(0)
    return out


def by_definition(q, k, v, do, mask):
    """One query head: O, dq and its parts of dk and dv, over pairs that see each other; and their error bounds.

    As window_ref, but a hidden pair is no term at all (there 0 times what it holds).
    """
    q, k, v, do = (t.double() for t in (q, k, v, do))
    p = torch.softmax((q @ k.T * SCALE).masked_fill(~mask, -math.inf), -1)
    o = seen_sum(p, v, mask)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (do @ v.T - delta)
    outs = [o, seen_sum(ds, k, mask) * SCALE, seen_sum(ds.T, q, mask.T) * SCALE, seen_sum(p.T, do, mask.T)]
    bo = (BF16 + FP32) * (seen_sum(p, v.abs(), mask) + o.abs())
    size = do.abs() @ v.abs().T + delta.abs()
    e_ds = BF16 * ds.abs() + p * ((do.abs() * bo).sum(-1, keepdim=True) + 2 * FP32 * size)
    bounds = [bo, SCALE * seen_sum(e_ds + FP32 * ds.abs(), k.abs(), mask),
              SCALE * seen_sum((e_ds + FP32 * ds.abs()).T, q.abs(), mask.T),
              (BF16 + 2 * FP32) * seen_sum(p.T, do.abs(), mask.T)]
    return outs, bounds


# H, Hkv, S, window, first keys: key ranges split over workgroups, short and long; tiles of the many-headed launch.
SHAPES = [(1, 2, 1, 200, (20, 20), 3), (1, 1, 1, 700, (40, 30), 130), (4, 40, 8, 200, (20, 20), 3)]


@pytest.mark.parametrize("B,H,Hkv,S,window,sinks", SHAPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("what", ["q", "k", "v", "do"])
@pytest.mark.parametrize("whole", [True, False], ids=["row", "element"])
def test_bad_values_reach_who_sees_them(gpu, B, H, Hkv, S, window, sinks, bad, what, whole):
    """Outputs are finite, and right, exactly where the definition's are: element by element."""
    t = dict(zip("q k v do".split(), make(gpu, B, H, Hkv, S, S, 7)))
    for n, at in enumerate((1, sinks + 5, S // 2, S - 1)):
        dims = slice(None) if whole else slice(11 + 30 * n, 12 + 30 * n)
        t[what][:, :, at, dims] = bad
    kw = dict(window=window, sinks=sinks)
    o, lse = h3attn.attn_fwd_window(t["q"], t["k"], t["v"], return_lse=True, **kw)
    dq, dk, dv = h3attn.attn_bwd_window(t["do"], t["q"], t["k"], t["v"], o, lse, **kw)
    mask = ref.visible(B, S, S, window, sinks, False, None, None)
    rep = H // Hkv
    c = {n: x.cpu() for n, x in t.items()}
    spread = 0
    for b, hk in {(0, 0), (B - 1, Hkv - 1)}:
        kv_out, kv_bound = [0, 0], [0, 0]
        for h in range(hk * rep, (hk + 1) * rep):
            outs, bounds = by_definition(c["q"][b, h], c["k"][b, hk], c["v"][b, hk], c["do"][b, h], mask[b])
            kv_out = [x + y for x, y in zip(kv_out, outs[2:])]
            kv_bound = [x + y for x, y in zip(kv_bound, bounds[2:])]
            for name, got, want, bound in (("O", o[b, h], outs[0], bounds[0]), ("dq", dq[b, h], outs[1], bounds[1])):
                spread += compare(name, got, want, bound)
        for name, got, want, bound in (("dk", dk[b, hk], kv_out[0], kv_bound[0]), ("dv", dv[b, hk], kv_out[1], kv_bound[1])):
            spread += compare(name, got, want, bound)
    assert spread  # the bad values are seen by someone


def compare(name, got, want, bound):
    got = got.cpu().double()
    fine = torch.isfinite(want)
    differ = torch.isfinite(got) != fine
    assert not differ.any(), f"{name}: {differ.sum()} of {differ.numel()} differ, first at {differ.nonzero()[0].tolist()}"
    err = (got - want).abs()[fine]
    limit = (bound + (BF16 + FP32) * want.abs() + 1e-30)[fine]
    assert (err <= limit).all(), f"{name}: error {(err / limit).max():.3f} of what the roundings allow"
    return (~fine).sum().item()
