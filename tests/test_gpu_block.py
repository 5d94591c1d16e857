"""Layer norm and the q/k prologue from positions on the GPU, forward and backward, against float64."""
from __future__ import annotations

import pytest
import torch

import block_ref as ref
import h3attn

pytestmark = pytest.mark.gpu
EPS = 1e-6


def close(got, want, bound, what):
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    assert torch.isfinite(got).all(), f"{what}: non-finite"
    worst = ((got.double().cpu() - want).abs() / bound).max().item() if got.numel() else 0
    assert worst <= 1, f"{what}: error {worst:.3f} of what the roundings allow"


def norm_case(gpu, rows, C, dtype, wdtype, segments, seed=0, offset=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, C, generator=g) * torch.exp(torch.randn(C, generator=g)) + offset).to(dtype)
    w, b = ((torch.randn(segments, C, generator=g) * 0.3).to(wdtype) for _ in range(2))
    dy = torch.randn(rows, C, generator=g).to(dtype)
    return [t.to(gpu) for t in (x, w, b, dy)]


def check_norm(x, w, b, dy, bounds=None, modulate=True):
    rows, C = x.shape
    y, mean, rstd = h3attn.layer_norm_fwd(x, w, b, eps=EPS, segments=bounds, modulate=modulate, return_stats=True)
    assert y.dtype == x.dtype
    cb = [0, rows] if bounds is None else bounds
    cx, cdy = x.cpu(), dy.cpu()
    cw, cbias = (None if t is None else t.cpu().reshape(len(cb) - 1, C) for t in (w, b))
    add = 1.0 if modulate and w is not None else 0.0
    want, xh, wmean, wr, wrow, brow = ref.norm(cx, cw, cbias, cb, EPS, add)
    close(y, want, ref.norm_bound(cx, want, xh, wr, wrow, brow), "y")
    close(mean, wmean[:, 0], 2.0 ** -16 * cx.double().abs().amax(1) + 1e-30, "mean")
    close(rstd, wr[:, 0], wr[:, 0] * (2.0 ** -16 + (2.0 ** -17 * cx.double().abs().amax(1) * wr[:, 0]) ** 2), "rstd")
    dx, dw, db = h3attn.layer_norm_bwd(dy, x, w, mean, rstd, segments=bounds, modulate=modulate)
    grads, tol = ref.norm_grads(cdy, cx, cw, cb, EPS, add)
    close(dx, grads[0], tol[0], "dx")
    assert dw.dtype == db.dtype == torch.float32
    close(dw.reshape(-1, C), grads[1], tol[1], "dw")
    close(db.reshape(-1, C), grads[2], tol[2], "db")
    only, none, none_b = h3attn.layer_norm_bwd(dy, x, w, mean, rstd, segments=bounds, modulate=modulate,
                                               param_grads=False)
    assert none is None and none_b is None and torch.equal(only, dx)
    return y


@pytest.mark.parametrize("C", [1, 7, 8, 64, 65, 511, 512, 513, 1000, 1024, 1025, 1536, 2048, 2056, 4096, 4099, 5376,
                               6144, 6152, 8192, 8193, 12000, 16384])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norm_channels(gpu, C, dtype):
    check_norm(*norm_case(gpu, 19, C, dtype, dtype, 1, seed=C))


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 64, 513, 2049, 4111])
@pytest.mark.parametrize("C", [72, 1100])
def test_norm_rows(gpu, rows, C):
    check_norm(*norm_case(gpu, rows, C, torch.bfloat16, torch.float32, 1, seed=rows), modulate=False)


@pytest.mark.parametrize("C", [40, 1300])
def test_norm_segments(gpu, C):
    """Uneven segments, empty ones at both ends and between, more than one launch's worth."""
    x, w, b, dy = norm_case(gpu, 300, C, torch.bfloat16, torch.bfloat16, 7)
    check_norm(x, w, b, dy, [0, 0, 1, 50, 50, 51, 300, 300])
    x, w, b, dy = norm_case(gpu, 700, C, torch.bfloat16, torch.float16, 150)
    check_norm(x, w, b, dy, sorted([0, 700] + [(37 * i * i) % 701 for i in range(149)]))


def test_norm_without_affine(gpu):
    x, w, b, dy = norm_case(gpu, 33, 200, torch.float32, torch.float32, 1)
    check_norm(x, None, None, dy, modulate=False)
    check_norm(x, w[0], None, dy, modulate=False)
    check_norm(x, None, b[0], dy)


def test_norm_batch_of_samples(gpu):
    """[B,S,C] with a scale and shift per sample, as adaLN: the rows split evenly."""
    x, w, b, dy = norm_case(gpu, 60, 384, torch.bfloat16, torch.bfloat16, 4)
    y = h3attn.layer_norm_fwd(x.view(4, 15, 384), w, b, modulate=True)
    assert torch.equal(y.view(60, 384), check_norm(x, w, b, dy, [0, 15, 30, 45, 60]))


def test_norm_strided_rows_and_offsets(gpu):
    """Rows of a wider buffer, at bases off the 16-byte grid, and rows past 2^31 elements."""
    x, w, b, dy = norm_case(gpu, 21, 264, torch.bfloat16, torch.bfloat16, 1)
    want = check_norm(x, w, b, dy)
    for shift in (0, 1, 8):
        wide = torch.full((21, 300), float("nan"), dtype=torch.bfloat16, device=gpu)
        view = wide[:, shift:shift + 264]
        view.copy_(x)
        y, mean, rstd = h3attn.layer_norm_fwd(view, w, b, eps=EPS, modulate=True, return_stats=True)
        assert torch.equal(y, want)
        a = h3attn.layer_norm_bwd(view, view, w, mean, rstd, modulate=True)
        c = h3attn.layer_norm_bwd(x, x, w, mean, rstd, modulate=True)
        assert all(torch.equal(p, q) for p, q in zip(a, c))
    big = torch.empty((1 << 31) + 4096, dtype=torch.bfloat16, device=gpu)
    far = torch.as_strided(big, (2, 264), (1 << 31, 1))
    far.copy_(x[:2])
    assert torch.equal(h3attn.layer_norm_fwd(far, w, b, eps=EPS, modulate=True), want[:2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_far_from_zero(gpu, dtype):
    """A large common offset, constant rows, one huge channel: the variance is taken about the mean."""
    x, w, b, dy = norm_case(gpu, 40, 1024, dtype, torch.float32, 1, offset=100.0)
    x[3] = 5.0
    x[4] = 0.0
    x[5, 7] = 30000.0
    check_norm(x, w, b, dy)


def test_norm_no_rows(gpu):
    x = torch.empty(0, 64, device=gpu)
    w = torch.ones(3, 64, device=gpu)
    y, mean, rstd = h3attn.layer_norm_fwd(x, w, w, segments=[0, 0, 0, 0], return_stats=True)
    assert y.shape == (0, 64) and mean.shape == (0,)
    dx, dw, db = h3attn.layer_norm_bwd(y, x, w, mean, rstd, segments=[0, 0, 0, 0])
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all() and dw.shape == (3, 64)


def test_norm_bad_rows_stay_alone(gpu):
    """A row with NaN or infinities spoils its own output and nothing else's."""
    x, w, b, dy = norm_case(gpu, 12, 1300, torch.bfloat16, torch.bfloat16, 1)
    good = h3attn.layer_norm_fwd(x, w, b)
    x[5, 9], x[7, 1] = float("nan"), float("inf")
    y = h3attn.layer_norm_fwd(x, w, b)
    keep = [i for i in range(12) if i not in (5, 7)]
    assert torch.equal(y[keep], good[keep]) and torch.isnan(y[[5, 7]].float()).all()


# ---------------------------------------------------------------------------
def rope_case(gpu, B, S, Hq, Hk, axes, seed=0, pos_dtype=torch.int32, batched=False, top=50000):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B, S, (Hq + 2 * Hk) * 128, generator=g).to(torch.bfloat16).to(gpu)
    q = qkv[..., :Hq * 128].view(B, S, Hq, 128)
    k = qkv[..., Hq * 128:(Hq + Hk) * 128].view(B, S, Hk, 128)
    pos = torch.randint(-top, top, (B if batched else 1, S, len(axes)), generator=g)
    pos = pos.to(torch.int32) if pos_dtype == torch.int32 else pos.float() + 0.37
    qw, kw = ((1 + 0.2 * torch.randn(128, generator=g)).to(torch.bfloat16).to(gpu) for _ in range(2))
    dq, dk = (torch.randn(B, S, h, 128, generator=g).to(torch.bfloat16).to(gpu) for h in (Hq, Hk))
    return q, k, (pos if batched else pos[0]).to(gpu), qw, kw, dq, dk


def check_rope(q, k, pos, axes, qw, kw, dq, dk, theta=10000.0):
    got = h3attn.qk_rmsnorm_rope_axes(q, k, pos, axes, qw, kw, eps=EPS, theta=theta)
    grads = h3attn.qk_rmsnorm_rope_axes_bwd(dq, dk, q, k, pos, axes, qw, kw, eps=EPS, theta=theta)
    ang = ref.angles((pos if pos.dim() == 3 else pos[None]).cpu(), axes, theta)
    for i, (x, w, d, name) in enumerate(((q, qw, dq, "q"), (k, kw, dk, "k"))):
        y, tol = ref.rope(x.cpu(), ang, w.cpu(), EPS)
        close(got[i], y, tol, name)
        (dx, dw), (tx, tw) = ref.rope_grads(d.cpu(), x.cpu(), ang, w.cpu(), EPS)
        close(grads[i], dx, tx, "d" + name)
        close(grads[2 + i], dw, tw, f"d{name}w")
    return got


@pytest.mark.parametrize("axes", [(128,), (64, 64), (44, 42, 42), (32, 32, 32), (2, 14), (16, 56, 56), (8, 8, 8, 8)])
@pytest.mark.parametrize("Hq,Hk", [(4, 4), (14, 2), (28, 28), (33, 1)])
def test_rope_axes(gpu, axes, Hq, Hk):
    check_rope(*(c := rope_case(gpu, 1, 37, Hq, Hk, axes, seed=Hq))[:3], axes, *c[3:])


@pytest.mark.parametrize("B,S", [(1, 1), (1, 2), (1, 3), (1, 5), (3, 7), (2, 300), (1, 4200)])
def test_rope_lengths(gpu, B, S):
    axes = (44, 42, 42)
    for dtype, batched in ((torch.int32, True), (torch.float32, False)):
        check_rope(*(c := rope_case(gpu, B, S, 3, 2, axes, S, dtype, batched))[:3], axes, *c[3:])


def test_rope_more_tokens_than_a_launch_walks_at_once(gpu):
    # 2^24 tokens are taken by 2^22 workgroups in one step; offsets pass 32 bits on the way.
    S = (1 << 24) + 7
    q, k = (torch.randn(1, S, 1, 128, device=gpu, dtype=torch.bfloat16) for _ in range(2))
    pos = (torch.arange(S, device=gpu, dtype=torch.int32) % 4099)[:, None].contiguous()
    w = torch.rand(128, device=gpu).to(torch.bfloat16) + 0.5
    oq, ok = h3attn.qk_rmsnorm_rope_axes(q, k, pos, (128,), w, w)
    for a, b in ((0, 9), (S // 2, S // 2 + 9), ((1 << 24) - 5, (1 << 24) + 3), (S - 7, S)):
        for whole, part in zip((oq, ok), h3attn.qk_rmsnorm_rope_axes(q[:, a:b], k[:, a:b], pos[a:b], (128,), w, w)):
            assert torch.equal(whole[:, a:b], part)


def test_rope_far_positions(gpu):
    """Positions up to 2^30: the angles stay those of the definition."""
    axes = (44, 42, 42)
    check_rope(*(c := rope_case(gpu, 1, 64, 2, 2, axes, 3, top=1 << 30))[:3], axes, *c[3:], theta=500.0)


def test_rope_axes_matches_the_table_form_and_works_in_place(gpu):
    """One axis of token numbers is rope_freqs; written over q and k it is qk_rmsnorm_rope_."""
    q, k, _, qw, kw, _, _ = rope_case(gpu, 1, 130, 4, 4, (128,))
    pos = torch.arange(130, dtype=torch.int32, device=gpu)[:, None]
    want = h3attn.qk_rmsnorm_rope_axes(q, k, pos, (128,), qw, kw, eps=EPS)
    tq, tk = q.clone(), k.clone()
    h3attn.qk_rmsnorm_rope_(tq, tk, h3attn.rope_freqs(130, 128, device=gpu), qw, kw, eps=EPS)
    for a, b in ((want[0], tq), (want[1], tk)):
        assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 1e-5).all()
    out = h3attn.qk_rmsnorm_rope_axes(q, k, pos, (128,), qw, kw, eps=EPS, out=(q, k))
    assert out[0].data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_rope_writes_only_its_rows(gpu):
    q, k, pos, qw, kw, _, _ = rope_case(gpu, 2, 9, 5, 3, (44, 42, 42))
    bufs = [torch.full((2, 13, h + 2, 144), 7.0, dtype=torch.bfloat16, device=gpu) for h in (5, 3)]
    views = [b[:, 2:11, 1:-1, 8:136] for b in bufs]
    got = h3attn.qk_rmsnorm_rope_axes(q, k, pos, (44, 42, 42), qw, kw, out=views)
    want = h3attn.qk_rmsnorm_rope_axes(q, k, pos, (44, 42, 42), qw, kw)
    for b, v, g, w in zip(bufs, views, got, want):
        assert torch.equal(g, w)
        v.fill_(7.0)
        assert (b == 7).all()


def test_block_ops_on_streams_and_in_graphs(gpu):
    """Side stream, capture and replays on new inputs, against eager calls; equal calls give equal bits."""
    x, w, b, dy = norm_case(gpu, 500, 1300, torch.bfloat16, torch.bfloat16, 2)
    q, k, pos, qw, kw, dq, dk = rope_case(gpu, 1, 300, 6, 2, (44, 42, 42))
    bounds = [0, 77, 500]

    def step():
        y, mean, rstd = h3attn.layer_norm_fwd(x, w, b, segments=bounds, modulate=True, return_stats=True)
        return (y, *h3attn.layer_norm_bwd(dy, x, w, mean, rstd, segments=bounds, modulate=True),
                *h3attn.qk_rmsnorm_rope_axes(q, k, pos, (44, 42, 42), qw, kw),
                *h3attn.qk_rmsnorm_rope_axes_bwd(dq, dk, q, k, pos, (44, 42, 42), qw, kw))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(p, r) for p, r in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        for dst, src in zip((x, w, b, dy), norm_case(gpu, 500, 1300, torch.bfloat16, torch.bfloat16, 2, seed)):
            dst.copy_(src)
        for dst, src in zip((q, k, pos, qw, kw, dq, dk), rope_case(gpu, 1, 300, 6, 2, (44, 42, 42), seed)):
            dst.copy_(src)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, r) for p, r in zip(want, out))
