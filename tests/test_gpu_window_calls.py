"""Windowed attention on the GPU: calls that the documentation allows and that are easily got wrong."""
from __future__ import annotations

import pytest
import torch

import h3attn
import window_ref as ref
from h3attn import autograd
from test_gpu_window import SCALE, check, close, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,H,Hkv,S,window,sinks,lens", [(1, 2, 2, 40, (None, None), 0, None), (2, 4, 2, 200, (30, 30), 9, None),
                                                         (2, 4, 2, 200, (30, 30), 140, [150, 70]),
                                                         (3, 40, 8, 170, (20, 200), 0, [170, 3, 99])])
@pytest.mark.parametrize("which", ["dout", "q", "both", "overlapping"])
def test_rows_that_share_memory(gpu, B, H, Hkv, S, window, sinks, lens, which):
    """A gradient expanded over the sequence (that of a mean over it), one query for all rows, overlapping rows."""
    q, k, v, do = make(gpu, B, H, Hkv, S, S, seed=S)
    wide = lambda t: t[:, :, :1].expand(B, H, S, 128)  # noqa: E731
    if which == "overlapping":
        mem = do.contiguous().view(B, H, S * 128)
        do = mem.as_strided((B, H, S, 128), (H * S * 128, S * 128, 64, 1))
    else:
        do = wide(do) if which != "q" else do
        q = wide(q) if which != "dout" else q
    check(gpu, B, H, Hkv, S, S, window, sinks, kv_lens=lens, tensors=(q, k, v, do))


def test_gradient_of_a_mean_over_the_sequence(gpu):
    B, H, S = 1, 3, 150
    q, k, v, _ = (t.detach().requires_grad_() for t in make(gpu, B, H, H, S, S, seed=1))
    o = autograd.window_attention(q, k, v, (25, 25), sinks=5)
    o.sum(dim=2).backward(g := torch.ones(B, H, 128, dtype=torch.bfloat16, device=gpu))
    do = g[:, :, None].expand(B, H, S, 128).cpu()
    c = [t.detach().cpu() for t in (q, k, v)]
    mask = ref.visible(B, S, S, (25, 25), 5, False, None, None)
    for name, t, w, b in zip(("dq", "dk", "dv"), (q, k, v), ref.backward(do, *c, mask, SCALE),
                             ref.backward_bounds(do, *c, mask, SCALE)):
        close(t.grad, w, b, name)


@pytest.mark.parametrize("B,H,Hkv,Sq,Skv", [(2, 2, 1, 140, 100), (4, 40, 8, 300, 129), (1, 1, 1, 20, 1), (1, 1, 1, 8300, 70)])
@pytest.mark.parametrize("causal", [False, True])
def test_more_rows_than_keys(gpu, B, H, Hkv, Sq, Skv, causal):
    """Starts per sequence put a query buffer that is longer than the cache; rows outside it give zeros."""
    starts = [0, -Sq + 30, Skv - 5, -17][:B]
    check(gpu, B, H, Hkv, Sq, Skv, (40, 0 if causal else 25), 6, causal, q_start=starts)
    check(gpu, B, H, Hkv, Sq, Skv, (40, 0 if causal else 25), 6, causal, q_start=starts,
          kv_lens=[Skv - 1, Skv // 2, Skv, 0][:B])


@pytest.mark.parametrize("offset", [1, 3, 4, 8])
def test_gradient_off_the_16_byte_grid(gpu, offset):
    """The gradient of an output that was concatenated behind an odd number of other values is a piece of a larger one."""
    B, H, S = 1, 2, 70
    q, k, v, do = make(gpu, B, H, H, S, S, seed=2)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = autograd.window_attention(*leaves, (12, 12))
    both = torch.cat([torch.zeros(offset, dtype=torch.bfloat16, device=gpu), o.reshape(-1)])
    both.backward(torch.cat([torch.zeros(offset, dtype=torch.bfloat16, device=gpu), do.reshape(-1)]))
    o2, lse = h3attn.attn_fwd_window(q, k, v, (12, 12), return_lse=True)
    for t, want in zip(leaves, h3attn.attn_bwd_window(do, q, k, v, o2, lse, (12, 12))):
        assert torch.equal(t.grad, want)
