"""Windowed attention on the GPU, forward and backward, against the definition in float64."""
from __future__ import annotations

import math

import pytest
import torch

import h3attn
import window_ref as ref

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)


def make(gpu, B, H, Hkv, Sq, Skv, seed=0, scale=1.0):
    """q, k, v, dout on the GPU as [B,H,S,128] views of sequence-major memory."""
    g = torch.Generator().manual_seed(seed)
    mk = lambda h, s: (torch.randn(B, s, h, 128, generator=g) * scale).to(torch.bfloat16).to(gpu).transpose(1, 2)  # noqa: E731
    return mk(H, Sq), mk(Hkv, Skv), mk(Hkv, Skv), mk(H, Sq)


def close(got, want, bound, what):
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all(), f"{what}: non-finite"
    worst = (err / bound).max().item()
    assert worst <= 1, f"{what}: error {worst:.3f} of what the roundings allow"


def check(gpu, B, H, Hkv, Sq, Skv, window, sinks, causal=False, q_start=None, kv_lens=None, seed=0, grads=True,
          tensors=None):
    q, k, v, do = tensors or make(gpu, B, H, Hkv, Sq, Skv, seed)
    mask = ref.visible(B, Sq, Skv, window, sinks, causal, q_start, kv_lens)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu) if isinstance(x, (list, tuple)) else x  # noqa: E731
    kw = dict(window=window, sinks=sinks, causal=causal, q_start=dev(q_start), kv_lens=dev(kv_lens))
    o, lse = h3attn.attn_fwd_window(q, k, v, return_lse=True, **kw)
    c = [t.cpu() for t in (q, k, v, do)]
    want, want_lse, _ = ref.forward(*c[:3], mask, SCALE)
    empty = ~mask.any(-1)[:, None].expand(B, H, Sq)
    close(o, want, ref.forward_bound(*c[:3], mask, SCALE), "O")
    assert (o.cpu()[empty] == 0).all()
    assert (lse.cpu()[empty] == -math.inf).all()
    assert ((lse.cpu().double() - want_lse)[~empty].abs() <= 2.0 ** -13 * (1 + want_lse[~empty].abs())).all()
    if grads:
        got = h3attn.attn_bwd_window(do, q, k, v, o, lse, **kw)
        for name, g, w, b in zip(("dq", "dk", "dv"), got, ref.backward(c[3], *c[:3], mask, SCALE),
                                 ref.backward_bounds(c[3], *c[:3], mask, SCALE)):
            close(g, w, b, name)
        assert (got[0].cpu()[empty] == 0).all(), "dq of rows that see nothing"
        unseen = ~mask.any(1)[:, None].expand(B, Hkv, Skv)
        assert (got[1].cpu()[unseen] == 0).all() and (got[2].cpu()[unseen] == 0).all(), "dk, dv of unseen keys"
    return o


@pytest.mark.parametrize("S", [1, 2, 31, 33, 64, 65, 128, 129, 300])
@pytest.mark.parametrize("window,sinks,causal", [((16, 16), 4, False), ((40, 0), 0, True), ((0, 0), 0, False),
                                                 ((None, None), 0, False), ((7, 90), 33, False)])
def test_lengths_and_windows(gpu, S, window, sinks, causal):
    check(gpu, 1, 2, 2, S, S, window, sinks, causal, seed=S)


@pytest.mark.parametrize("sinks", [0, 1, 5, 63, 64, 70, 130, 300, 699, 1000])
@pytest.mark.parametrize("causal", [False, True])
def test_sinks(gpu, sinks, causal):
    check(gpu, 1, 1, 1, 700, 700, (50, 0 if causal else 20), sinks, causal, seed=sinks)


@pytest.mark.parametrize("S", [1, 40, 300])
def test_rows_of_one_key_have_no_score_gradient(gpu, S):
    # P = 1, so dS = P (dP - P dP) = 0.  In fp32: s and lse agree to 2^-19 (|lse| < 8 in three
    # roundings, an exp2 and a log2 of an ulp), so |1 - P| < 2^-18 and |dS| < 2^-18 |dP|; the
    # roundings of dS and of the result add a 2^-7th of that.
    q, k, v, do = make(gpu, 1, 2, 2, S, S, seed=S)
    o, lse = h3attn.attn_fwd_window(q, k, v, (0, 0), return_lse=True)
    assert lse.abs().max() < 8
    dq, dk, _ = (t.double() for t in h3attn.attn_bwd_window(do, q, k, v, o, lse, (0, 0)))
    dp = (do.double() * v.double()).sum(-1, keepdim=True).abs()
    assert (dq.abs() <= 2.0 ** -17 * SCALE * dp * k.double().abs()).all()
    assert (dk.abs() <= 2.0 ** -17 * SCALE * dp * q.double().abs()).all()
    dq, _, _ = h3attn.attn_bwd_window(do, q, k, v, *h3attn.attn_fwd_window(q, k, v, (50, 0), causal=True, return_lse=True),
                                      (50, 0), causal=True)
    assert (dq[:, :, 0].double().abs() <= 2.0 ** -17 * SCALE * dp[:, :, 0] * k[:, :, 0].double().abs()).all()


def test_first_keys_of_many_heads(gpu):
    # Runs of queries longer than a window tile's: 4 of 7 stages each, 24 stages in all.
    check(gpu, 1, 28, 28, 1500, 1500, (0, 0), 2 ** 31 - 1, False, seed=5)


@pytest.mark.parametrize("B,H,S", [(40, 6, 3), (300, 2, 1), (9, 14, 128)])
def test_many_short_sequences(gpu, B, H, S):
    # More heads than runs of tiles: every head's tiles are dealt, and none twice.
    check(gpu, B, H, H // 2, S, S, (2, 1), 1, False, seed=B)


@pytest.mark.parametrize("window", [(0, 0), (1, 0), (63, 64), (64, 63), (200, 0), (0, 200), (511, 511), (2000, 2000)])
def test_window_sides(gpu, window):
    check(gpu, 1, 2, 1, 513, 513, window, 3, False, seed=window[0])


@pytest.mark.parametrize("H,Hkv", [(1, 1), (6, 1), (6, 2), (6, 3), (14, 2)])
def test_shared_heads(gpu, H, Hkv):
    check(gpu, 2, H, Hkv, 200, 200, (30, 30), 10, False, seed=H)


@pytest.mark.parametrize("causal", [False, True])
def test_padded_batch(gpu, causal):
    """Lengths of 0, 1, a tile's edge, all, and out of range (clamped)."""
    lens = [0, 1, 64, 127, 128, 129, 260, 999, -5]
    check(gpu, len(lens), 2, 1, 260, 260, (40, 0 if causal else 40), 6, causal, kv_lens=lens)


@pytest.mark.parametrize("S,window,sinks,causal", [(129, (30, 30), 5, False), (257, (0, 64), 0, False),
                                                   (300, (100, 0), 70, True), (300, (None, None), 0, False)])
@pytest.mark.parametrize("ragged", [False, True])
def test_many_heads(gpu, S, window, sinks, causal, ragged):
    """Launches of more tiles than a split of the keys is worth."""
    lens = [S, 1, S // 2, S - 1] if ragged else None
    check(gpu, 4, 40, 8, S, S, window, sinks, causal, kv_lens=lens, seed=S)


@pytest.mark.parametrize("B,H,Hkv,S,window,sinks", [(1, 2, 1, 200, (20, 20), 3), (1, 1, 1, 700, (40, 30), 130),
                                                    (4, 40, 8, 200, (20, 20), 3)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["kv", "q"])
def test_hidden_values_do_not_matter(gpu, B, H, Hkv, S, window, sinks, bad, where):
    """NaN and infinities in rows of k and v, or of q and dout, reach those who see them and nobody else."""
    q, k, v, do = make(gpu, B, H, Hkv, S, S, 4)
    mask = ref.visible(B, S, S, window, sinks, False, None, None)
    c = [t.cpu() for t in (q, k, v, do)]
    spots = [sinks + 5, S // 2, S - 1]
    if where == "kv":
        for n, t in enumerate((k, v)):
            t[:, :, spots[n:]] = bad
        rows = mask[:, :, spots].any(-1)        # rows that see a bad key
    else:
        for n, t in enumerate((q, do)):
            t[:, :, spots[n:]] = bad
        rows = torch.zeros(B, S, dtype=torch.bool)
        rows[:, spots] = True
    keys = (mask & rows[:, :, None]).any(1)     # keys seen by such rows
    if where == "kv":
        keys[:, spots] = True
    kw = dict(window=window, sinks=sinks)
    o, lse = h3attn.attn_fwd_window(q, k, v, return_lse=True, **kw)
    grads = h3attn.attn_bwd_window(do, q, k, v, o, lse, **kw)
    for name, got, want, bound, hit in zip(
            ("O", "dq", "dk", "dv"), (o, *grads),
            (ref.forward(*c[:3], mask, SCALE)[0], *ref.backward(c[3], *c[:3], mask, SCALE)),
            (ref.forward_bound(*c[:3], mask, SCALE), *ref.backward_bounds(c[3], *c[:3], mask, SCALE)),
            (rows, rows, keys, keys)):
        clean = ~hit[:, None, :].expand(*got.shape[:3])
        assert clean.any()
        close(got.cpu()[clean], want[clean], bound[clean], name)
    if bad != bad:
        assert torch.isnan(o.cpu().float()).any(-1)[rows[:, None].expand(B, H, S)].any()


def test_padding_holds_anything(gpu):
    """Rows and keys behind a sequence's end are NaN: outputs are 0 there and right elsewhere."""
    B, H, Hkv, S = 3, 4, 2, 190
    q, k, v, do = make(gpu, B, H, Hkv, S, S, 8)
    lens = [190, 70, 0]
    mask = ref.visible(B, S, S, (25, 25), 9, False, None, lens)
    c = [t.cpu() for t in (q, k, v, do)]
    for t in (q, k, v, do):
        for b, n in enumerate(lens):
            t[b, :, n:] = float("nan")
    kw = dict(window=(25, 25), sinks=9, kv_lens=torch.tensor(lens, dtype=torch.int32, device=gpu))
    o, lse = h3attn.attn_fwd_window(q, k, v, return_lse=True, **kw)
    close(o, ref.forward(*c[:3], mask, SCALE)[0], ref.forward_bound(*c[:3], mask, SCALE), "O")
    for name, g, w, b in zip(("dq", "dk", "dv"), h3attn.attn_bwd_window(do, q, k, v, o, lse, **kw),
                             ref.backward(c[3], *c[:3], mask, SCALE), ref.backward_bounds(c[3], *c[:3], mask, SCALE)):
        close(g, w, b, name)
    # One token: nothing past its length is read.
    n = torch.tensor([190, 70, 1], dtype=torch.int32, device=gpu)
    got = h3attn.attn_fwd_window(c[0][:, :, :1].to(gpu), k, v, (60, 0), sinks=4, causal=True, q_start=n - 1, kv_lens=n)
    mask = ref.visible(B, 1, S, (60, 0), 4, True, [189, 69, 0], [190, 70, 1])
    assert torch.isfinite(got[:2]).all()
    want = ref.forward(c[0][:, :, :1], *c[1:3], mask, SCALE)[0]
    close(got[:2], want[:2], ref.forward_bound(c[0][:, :, :1], *c[1:3], mask, SCALE)[:2], "one token")


@pytest.mark.parametrize("Sq,Skv,q_start", [(1, 300, None), (5, 300, None), (5, 300, 0), (130, 300, 100), (64, 65, 1)])
def test_chunk_of_queries(gpu, Sq, Skv, q_start):
    check(gpu, 1, 4, 2, Sq, Skv, (70, 0), 5, True, q_start=q_start)
    check(gpu, 1, 4, 2, Sq, Skv, (70, 30), 5, False, q_start=q_start)


def test_starts_per_sequence(gpu):
    """Chunks at their own places in a padded cache, some rows outside their sequence."""
    check(gpu, 6, 4, 2, 140, 400, (90, 10), 7, False, q_start=[0, 100, 260, -50, 390, 1000],
          kv_lens=[400, 200, 300, 300, 400, 400])


@pytest.mark.parametrize("H,Hkv", [(2, 2), (28, 4), (8, 1), (40, 1)])
@pytest.mark.parametrize("left,sinks", [(0, 0), (99, 4), (1000, 0), (5000, 130)])
def test_one_token(gpu, H, Hkv, left, sinks):
    lens = [1, 2, 65, 400, 777]
    check(gpu, 5, H, Hkv, 1, 777, (left, 0), sinks, True, q_start=[n - 1 for n in lens], kv_lens=lens, grads=H < 20)


def test_gradients_against_differences():
    """The float64 reference's gradients against central differences of its forward (on the CPU)."""
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(1, h, 9, 8, generator=g, dtype=torch.float64) for h in (2, 1, 1))
    do = torch.randn(1, 2, 9, 8, generator=g, dtype=torch.float64)
    mask = ref.visible(1, 9, 9, (2, 1), 1, False, None, [8])
    grads = ref.backward(do, q, k, v, mask, 0.3)
    h = 1e-6
    for t, grad in zip((q, k, v), grads):
        for at in [(0, 0, 0, 0), (0, 0, 4, 3), (0, 0, 7, 7), (0, 0, 8, 1)]:
            x = t[at].item()
            f = []
            for d in (h, -h):
                t[at] = x + d
                f.append((ref.forward(q, k, v, mask, 0.3)[0] * do * mask.any(-1)[:, None, :, None]).sum().item())
            t[at] = x
            assert abs((f[0] - f[1]) / (2 * h) - grad[at].item()) < 1e-7


def test_strided_views_and_out(gpu):
    """Views of a fused QKV projection in, a view of a larger buffer out: nothing else is written."""
    B, S, H, Hkv = 2, 150, 4, 2
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(B, S, (H + 2 * Hkv) * 128 + 16, generator=g).to(torch.bfloat16).to(gpu)[..., 8:-8]
    q, k, v = (t.view(B, S, -1, 128).transpose(1, 2) for t in qkv.split([H * 128, Hkv * 128, Hkv * 128], dim=-1))
    do = torch.randn(B, H, S, 128, generator=g).to(torch.bfloat16).to(gpu)
    mask = ref.visible(B, S, S, (20, 20), 3, False, None, None)
    buf = torch.full((B, S + 9, H, 192), 7.0, dtype=torch.bfloat16, device=gpu)
    out = buf[:, 4:4 + S, :, 32:160].transpose(1, 2)
    got, lse = h3attn.attn_fwd_window(q, k, v, (20, 20), sinks=3, out=out, return_lse=True)
    assert got.data_ptr() == out.data_ptr()
    c = [t.cpu() for t in (q, k, v, do)]
    close(out, ref.forward(*c[:3], mask, SCALE)[0], ref.forward_bound(*c[:3], mask, SCALE), "O")
    rest = torch.ones_like(buf, dtype=torch.bool)
    rest[:, 4:4 + S, :, 32:160] = False
    assert (buf[rest] == 7).all()
    grads = h3attn.attn_bwd_window(do, q, k, v, out, lse, (20, 20), sinks=3)
    for name, t, w, b in zip(("dq", "dk", "dv"), grads, ref.backward(c[3], *c[:3], mask, SCALE),
                             ref.backward_bounds(c[3], *c[:3], mask, SCALE)):
        close(t, w, b, name)
    # A dtype of rows that cannot be read in place is copied, with the same result.
    odd = torch.empty(B, H, S, 129, dtype=torch.bfloat16, device=gpu)[..., 1:]
    odd.copy_(q)
    assert torch.equal(h3attn.attn_fwd_window(odd, k, v, (20, 20), sinks=3), out)


def test_large_offsets(gpu):
    """A cache whose second sequence starts past 2^32 bytes and past 2^31 elements."""
    S, far = 200, (1 << 31) + 4096
    cache = torch.empty(far + S * 256, dtype=torch.bfloat16, device=gpu)
    view = lambda at: torch.as_strided(cache, (2, 1, S, 128), (far, 128, 256, 1), at)  # noqa: E731
    g = torch.Generator().manual_seed(2)
    k, v = view(0), view(128)
    k.copy_(torch.randn(2, 1, S, 128, generator=g).to(torch.bfloat16))
    v.copy_(torch.randn(2, 1, S, 128, generator=g).to(torch.bfloat16))
    q, do = (torch.randn(2, 2, S, 128, generator=g).to(torch.bfloat16).to(gpu) for _ in range(2))
    check(gpu, 2, 2, 1, S, S, (33, 12), 4, tensors=(q, k, v, do))
    check(gpu, 2, 2, 1, 1, S, (90, 0), 4, True, tensors=(q[:, :, :1], k, v, do[:, :, :1]))


def test_equal_calls_give_equal_bits_and_full_window_is_dense(gpu):
    q, k, v, do = make(gpu, 1, 4, 4, 700, 700, 9)
    kw = dict(window=(100, 100), sinks=70)
    runs = []
    for _ in range(3):
        o, lse = h3attn.attn_fwd_window(q, k, v, return_lse=True, **kw)
        runs.append((o, lse, *h3attn.attn_bwd_window(do, q, k, v, o, lse, **kw)))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))
    full, dense = h3attn.attn_fwd_window(q, k, v, (None, None)), h3attn.attn_fwd(q, k, v)
    mask = torch.ones(1, 700, 700, dtype=torch.bool)
    bound = ref.forward_bound(q.cpu(), k.cpu(), v.cpu(), mask, SCALE)
    close(full, dense.double().cpu(), 2 * bound, "full window against attn_fwd")


def test_stream_and_graph(gpu):
    """On a side stream, and captured and replayed on new inputs in place, against eager calls."""
    q, k, v, do = make(gpu, 2, 4, 2, 260, 260, 5)
    lens = torch.tensor([260, 100], dtype=torch.int32, device=gpu)
    kw = dict(window=(50, 50), sinks=9, kv_lens=lens)

    def step():
        o, lse = h3attn.attn_fwd_window(q, k, v, return_lse=True, **kw)
        return (o, lse, *h3attn.attn_bwd_window(do, q, k, v, o, lse, **kw))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (6, 7, 8):
        for dst, src in zip((q, k, v, do), make(gpu, 2, 4, 2, 260, 260, seed)):
            dst.copy_(src)
        lens.copy_(torch.tensor([seed * 30, 260 - seed], dtype=torch.int32))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out))


@pytest.mark.parametrize("H,Hkv,S,window,sinks,causal", [(8, 1, 600, (119, 26), 0, False), (14, 2, 513, (67, 0), 50, True),
                                                         (6, 1, 200, (300, 300), 0, False), (4, 1, 130, (3, 2), 129, False)])
def test_few_key_tiles(gpu, H, Hkv, S, window, sinks, causal):
    # Too few tiles to fill the chip: all of them cut into runs of queries, ragged ones too.
    check(gpu, 1, H, Hkv, S, S, window, sinks, causal, seed=S)
    check(gpu, 2, H, Hkv, S, S, window, sinks, causal, kv_lens=[S, S // 3], q_start=[0, 0], seed=S + 1)


def test_calls_at_once_on_two_streams(gpu):
    """Split keys and cut tiles leave partial results in workspaces: each call has its own."""
    sets = [make(gpu, 1, 8, 1, 300, 300, seed) for seed in (1, 2)]
    kw = dict(window=(40, 30), sinks=140)

    def step(q, k, v, do):
        one = h3attn.attn_fwd_window(q[:, :, -1:], k, v, **kw)
        o, lse = h3attn.attn_fwd_window(q, k, v, return_lse=True, **kw)
        return (one, o, lse, *h3attn.attn_bwd_window(do, q, k, v, o, lse, **kw))

    want = [step(*s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(want[i], g))
