"""The differentiable forms, alone and as one block: gradients against float64 and against differences."""
from __future__ import annotations

import math

import pytest
import torch

import block_ref
import h3attn
import window_ref
from h3attn import autograd as ag

pytestmark = pytest.mark.gpu
AXES, EPS = (44, 42, 42), 1e-6


def leaf(*shape, gpu, dtype=torch.bfloat16, scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(gpu).requires_grad_()


def test_functions_return_the_entry_points_gradients(gpu):
    B, H, Hkv, S, C = 2, 4, 2, 90, 192
    q, k, v = (leaf(B, h, S, 128, gpu=gpu, seed=i) for i, h in enumerate((H, Hkv, Hkv)))
    lens = torch.tensor([90, 41], dtype=torch.int32, device=gpu)
    kw = dict(window=(20, 20), sinks=4, kv_lens=lens)
    o = ag.window_attention(q, k, v, **kw)
    do = torch.randn_like(o)
    o.backward(do)
    o2, lse = h3attn.attn_fwd_window(q.detach(), k.detach(), v.detach(), return_lse=True, **kw)
    for got, want in zip((o, q.grad, k.grad, v.grad),
                         (o2, *h3attn.attn_bwd_window(do, q.detach(), k.detach(), v.detach(), o2, lse, **kw))):
        assert torch.equal(got, want)
    x, w, b = leaf(B, S, C, gpu=gpu), leaf(B, C, gpu=gpu, seed=5), leaf(B, C, gpu=gpu, seed=6)
    y = ag.layer_norm(x, w, b, modulate=True)
    y.backward(dy := torch.randn_like(y))
    _, mean, rstd = h3attn.layer_norm_fwd(x.detach(), w.detach(), b.detach(), modulate=True, return_stats=True)
    dx, dw, db = h3attn.layer_norm_bwd(dy, x.detach(), w.detach(), mean, rstd, modulate=True)
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw.bfloat16()) and torch.equal(b.grad, db.bfloat16())
    # A frozen weight, no weight, and only a bias per sample.
    for weight, bias in ((w.detach(), b), (None, b), (None, None)):
        x.grad = b.grad = None
        ag.layer_norm(x, weight, bias).backward(dy)
        assert x.grad is not None and (bias is None or torch.equal(b.grad, dy.float().sum(1).bfloat16()) or
                                       (b.grad.float() - dy.float().sum(1)).abs().max() < 0.1)
    qw, kw_ = leaf(128, gpu=gpu, dtype=torch.float32, seed=7), leaf(128, gpu=gpu, dtype=torch.float32, seed=8)
    pos = torch.randint(0, 99, (S, 3), dtype=torch.int32, device=gpu)
    qs, ks = leaf(1, S, 4, 128, gpu=gpu), leaf(1, S, 2, 128, gpu=gpu, seed=1)
    yq, yk = ag.qk_norm_rope(qs, ks, pos, AXES, qw, kw_)
    (yq.float().sum() + yk.float().square().sum()).backward()
    assert qw.grad.dtype == torch.float32 and qw.grad.shape == (128,) and torch.isfinite(kw_.grad).all()
    # Nothing is asked of a frozen input.
    q2 = q.detach()
    o = ag.window_attention(q2, k, v.detach(), (None, 0), causal=True)
    o.sum().backward()
    assert q2.grad is None and k.grad is not None


class Block(torch.nn.Module):
    """x + out(attention(rope(norm(x)))): the attention half of a DiT block over windows."""

    def __init__(self, dim, heads, seed, device):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        mk = lambda *s: torch.nn.Parameter((torch.randn(*s, generator=g) / math.sqrt(s[-1])).bfloat16().to(device))  # noqa: E731
        self.heads = heads
        self.qkv, self.out = mk(3 * heads * 128, dim), mk(dim, heads * 128)
        self.qw, self.kw = (torch.nn.Parameter((1 + 0.1 * torch.randn(128, generator=g)).bfloat16().to(device))
                            for _ in range(2))
        self.scale, self.shift = mk(2, dim), mk(2, dim)

    def forward(self, x, pos, bounds, window, sinks):
        S, H = x.shape[0], self.heads
        h = ag.layer_norm(x, self.scale, self.shift, eps=EPS, segments=bounds, modulate=True)
        q, k, v = (h @ self.qkv.T).view(1, S, 3, H, 128).unbind(2)
        q, k = ag.qk_norm_rope(q, k, pos, AXES, self.qw, self.kw, eps=EPS)
        o = ag.window_attention(*(t.transpose(1, 2) for t in (q, k, v)), window, sinks=sinks)
        return x + o.transpose(1, 2).reshape(S, H * 128) @ self.out.T


def block_in_float64(p, x, pos, bounds, window, sinks, heads):
    S = x.shape[0]
    y = block_ref.norm(x, p["scale"], p["shift"], bounds, EPS, 1.0)[0]
    q, k, v = (y @ p["qkv"].T).view(1, S, 3, heads, 128).unbind(2)
    ang = block_ref.angles(pos[None], AXES, 10000.0)
    rn = lambda t, w: block_ref.rotate(t * (t.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * w, ang)  # noqa: E731
    q, k, v = (t.transpose(1, 2) for t in (rn(q, p["qw"]), rn(k, p["kw"]), v))
    mask = window_ref.visible(1, S, S, window, sinks, False, None, None)
    s = (q @ k.transpose(2, 3) / math.sqrt(128)).masked_fill(~mask[:, None], -math.inf)
    o = torch.softmax(s, -1) @ v
    return x + o.transpose(1, 2).reshape(S, heads * 128) @ p["out"].T


def test_block_forward_backward(gpu):
    """A run of them, as a model has them: norm, prologue, attention, with the model's products between.

    The block rounds to bf16 seven times between x and its result, each time by at most
    2^-8 of a value whose own size enters the next step: the errors' norms add up to at
    most 7 * 2^-8 of the result's forward, and about twice as many roundings backward.
    """
    S, dim, H, bounds, window, sinks = 150, 320, 3, (0, 40, 150), (30, 30), 10
    block = Block(dim, H, 3, gpu)
    x = leaf(S, dim, gpu=gpu, seed=9)
    pos = torch.stack([torch.arange(S) // 30, torch.arange(S) // 6 % 5, torch.arange(S) % 6], 1).int().to(gpu)
    y = block(x, pos, bounds, window, sinks)
    dy = leaf(S, dim, gpu=gpu, seed=10).detach()
    y.backward(dy)
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in block.named_parameters()}
    x64 = x.detach().double().cpu().requires_grad_()
    want = block_in_float64(p, x64, pos.cpu(), list(bounds), window, sinks, H)
    want.backward(dy.double().cpu())
    rel = lambda a, b: ((a.double().cpu() - b).norm() / b.norm()).item()  # noqa: E731
    assert rel(y.detach(), want.detach()) <= 7 * 2.0 ** -8
    assert rel(x.grad, x64.grad) <= 14 * 2.0 ** -8
    for n, t in block.named_parameters():
        assert rel(t.grad, p[n].grad) <= 14 * 2.0 ** -8, n
    # The gradient of x against a difference of the float64 block along a direction.
    d = torch.randn(S, dim, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
    h = 1e-5
    f = lambda s: (block_in_float64({n: t.detach() for n, t in p.items()}, x64.detach() + s * d, pos.cpu(),  # noqa: E731
                                    list(bounds), window, sinks, H) * dy.double().cpu()).sum().item()
    slope = (f(h) - f(-h)) / (2 * h)
    # (An error vector of that norm has a component along a random direction of norm / sqrt(n)
    # standard deviations; six of them.)
    assert abs((x.grad.double().cpu() * d).sum().item() - slope) <= \
        14 * 2.0 ** -8 * x64.grad.norm().item() * d.norm().item() / math.sqrt(d.numel()) * 6


def test_block_step_captured_and_replayed(gpu):
    """Forward and backward of the block in one graph, on static inputs, against eager steps."""
    S, dim, H, bounds, window, sinks = 96, 256, 2, (0, 30, 96), (20, 20), 6
    block = Block(dim, H, 4, gpu)
    pos = torch.randint(0, 50, (S, 3), dtype=torch.int32, device=gpu)
    x, dy = leaf(S, dim, gpu=gpu).detach(), leaf(S, dim, gpu=gpu, seed=1).detach()
    params = list(block.parameters())

    def step():
        xi = x.detach().requires_grad_()
        y = block(xi, pos, bounds, window, sinks)
        return (y.detach(), *torch.autograd.grad(y, [xi, *params], dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (2, 3, 4):
        x.copy_(leaf(S, dim, gpu=gpu, seed=seed).detach())
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
