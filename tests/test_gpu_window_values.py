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


@pytest.mark.parametrize("B,H,Hkv,S,window,sinks", SHAPES)
def test_a_key_that_no_row_takes(gpu, B, H, Hkv, S, window, sinks):
    """A key whose scores are all -inf has weight 0: O, dk and dv are as without it, dq is NaN where 0 meets its infinity."""
    q, k, v, do = make(gpu, B, H, Hkv, S, S, 9)
    q[..., 11] = -q[..., 11].abs() - 0.125
    spots = (sinks + 1, S // 2, S - 1)
    for at in spots:
        k[:, :, at, 11] = float("inf")
    mask = ref.visible(B, S, S, window, sinks, False, None, None)
    kw = dict(window=window, sinks=sinks)
    o, lse = h3attn.attn_fwd_window(q, k, v, return_lse=True, **kw)
    dq, dk, dv = h3attn.attn_bwd_window(do, q, k, v, o, lse, **kw)
    assert torch.isfinite(o).all() and torch.isfinite(lse).all() and torch.isfinite(dk).all() and torch.isfinite(dv).all()
    assert (dk[:, :, spots] == 0).all() and (dv[:, :, spots] == 0).all()
    rep = H // Hkv
    for b, hk in {(0, 0), (B - 1, Hkv - 1)}:
        kv_out, kv_bound = [0, 0], [0, 0]
        for h in range(hk * rep, (hk + 1) * rep):
            outs, bounds = by_definition(*(t.cpu() for t in (q[b, h], k[b, hk], v[b, hk], do[b, h])), mask[b])
            assert torch.isnan(outs[1]).any()
            kv_out = [x + y for x, y in zip(kv_out, outs[2:])]
            kv_bound = [x + y for x, y in zip(kv_bound, bounds[2:])]
            compare("O", o[b, h], outs[0], bounds[0])
            compare("dq", dq[b, h], outs[1], bounds[1])
        compare("dk", dk[b, hk], kv_out[0], kv_bound[0])
        compare("dv", dv[b, hk], kv_out[1], kv_bound[1])


@pytest.mark.parametrize("S", [200, 700])
def test_infinities_keep_their_sign(gpu, S):
    """A weight is never negative: +inf in v, or in dout, is +inf in O, or dv, and NaN only where -inf meets it."""
    q, k, v, do = make(gpu, 1, 2, 2, S, S, 5)
    inf, at = float("inf"), S // 2
    for t in (v, do):
        t[:, :, at, 3], t[:, :, at, 4], t[:, :, at, 5] = inf, -inf, inf
        t[:, :, at + 1, 5] = -inf
        t[:, :, at + 30, 6] = inf  # hidden from half of those that see the others
    o, lse = h3attn.attn_fwd_window(q, k, v, (20, 20), return_lse=True)
    near = slice(at - 8, at + 9)
    far = torch.ones(S, dtype=torch.bool)
    far[at - 20:at + 51] = False
    for name, t in (("O", o), ("dv", h3attn.attn_bwd_window(do, q, k, k, o := h3attn.attn_fwd_window(q, k, k, (20, 20)),
                                                             lse, (20, 20))[2])):
        assert (t[:, :, near, 3] == inf).all() and (t[:, :, near, 4] == -inf).all(), name
        assert torch.isnan(t[:, :, near, 5]).all() and torch.isfinite(t[:, :, near, 6]).all(), name
        assert torch.isfinite(t[:, :, near, 7:]).all() and torch.isfinite(t[:, :, far.to(t.device)]).all(), name


def compare(name, got, want, bound):
    got = got.cpu().double()
    fine = torch.isfinite(want)
    differ = torch.isfinite(got) != fine
    assert not differ.any(), f"{name}: {differ.sum()} of {differ.numel()} differ, first at {differ.nonzero()[0].tolist()}"
    err = (got - want).abs()[fine]
    limit = (bound + (BF16 + FP32) * want.abs() + 1e-30)[fine]
    assert (err <= limit).all(), f"{name}: error {(err / limit).max():.3f} of what the roundings allow"
    return (~fine).sum().item()


def pass_time(fn):
    """Milliseconds of a call, the best of four."""
    fn()
    times = []
    for _ in range(4):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        fn()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


# As many heads as fill the chip with tiles, one whose keys are split, and rows of one token each.
@pytest.mark.parametrize("B,H,Hkv,Sq,S", [(1, 16, 16, 4096, 4096), (1, 1, 1, 2048, 2048), (16, 28, 4, 1, 4096)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("what,where", [("do", "all"), ("do", "row"), ("do", "element"), ("do", "last"), ("q", "all"),
                                        ("q", "row"), ("q", "element"), ("k", "all"), ("k", "row"), ("k", "element"),
                                        ("v", "all"), ("v", "row"), ("v", "element"), ("v", "channel")])
def test_bad_values_that_are_seen_cost_little(gpu, B, H, Hkv, Sq, S, bad, what, where):
    """A step whose gradient overflowed, or one bad token, takes some times a clean one's time, not hundreds.

    A tile with a sum that is not finite is walked once more, in simpler loops (two to three times
    as long) that note every bad row (a few times as long again if each row is one).
    """
    t = dict(zip("q k v do".split(), make(gpu, B, H, Hkv, Sq, S, 3)))
    kw = dict(window=(511, 0 if Sq == 1 else 511), sinks=40)
    kw.update(q_start=torch.full((B,), S - 1, dtype=torch.int32, device=gpu) if Sq == 1 else None)

    def fwd():
        return h3attn.attn_fwd_window(t["q"], t["k"], t["v"], return_lse=True, **kw)

    def bwd():
        return h3attn.attn_bwd_window(t["do"], t["q"], t["k"], t["v"], *out, **kw)

    out = fwd()
    clean = [pass_time(fwd), pass_time(bwd)]
    n = t[what].shape[2]
    mid = n - 1 if where == "last" or n > Sq else n // 2
    if where == "all":
        t[what].fill_(bad)
    elif where == "channel":
        t[what][..., 77] = bad
    elif where == "element":
        t[what][:, :, mid, 77] = bad
    else:
        t[what][:, :, mid] = bad
    out = fwd()
    spoiled = [pass_time(fwd), pass_time(bwd)]
    print(f"{what} {where} {bad}: forward {clean[0]:.3f} -> {spoiled[0]:.3f} ms, backward {clean[1]:.3f} -> {spoiled[1]:.3f}")
    assert spoiled[0] <= 20 * clean[0] + 0.05 and spoiled[1] <= 20 * clean[1] + 0.05
