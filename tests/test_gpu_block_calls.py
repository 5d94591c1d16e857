"""Layer norm and the q/k prologue on the GPU: calls that are easily got wrong."""
from __future__ import annotations

import pytest
import torch

import h3attn
from h3attn import autograd

pytestmark = pytest.mark.gpu


def test_weights_for_no_segment(gpu):
    x, none = torch.randn(6, 64, device=gpu), torch.empty(0, 64, device=gpu)
    for fn in (h3attn.layer_norm_fwd, autograd.layer_norm):
        for args in ((none,), (none, none), (None, none)):
            with pytest.raises(ValueError, match="one segment at least"):
                fn(x, *args)
    _, mean, rstd = h3attn.layer_norm_fwd(x, return_stats=True)
    with pytest.raises(ValueError, match="one segment at least"):
        h3attn.layer_norm_bwd(x, x, none, mean, rstd)


def test_fp32_weights_are_used_in_bf16(gpu):
    """In both passes; their gradients stay fp32, and are those at the rounded weights."""
    g = torch.Generator().manual_seed(0)
    q, k, dq, dk = (torch.randn(2, 40, 3, 128, generator=g).to(torch.bfloat16).to(gpu) for _ in range(4))
    qw, kw = ((1 + 0.3 * torch.randn(128, generator=g)).to(gpu) for _ in range(2))
    pos = torch.arange(40, dtype=torch.int32, device=gpu)[:, None]
    wide = [t.clone().requires_grad_() for t in (q, k, qw, kw)]
    y = autograd.qk_norm_rope(wide[0], wide[1], pos, (128,), wide[2], wide[3])
    torch.autograd.backward(y, (dq, dk))
    args = (q, k, pos, (128,), qw.bfloat16(), kw.bfloat16())
    for got, want in zip(y, h3attn.qk_rmsnorm_rope_axes(*args)):
        assert torch.equal(got, want)
    for t, want in zip(wide, h3attn.qk_rmsnorm_rope_axes_bwd(dq, dk, *args)):
        assert t.grad.dtype == t.dtype and torch.equal(t.grad, want)
    assert wide[2].grad.dtype == torch.float32
    # Less than half a step of bf16 is no change, more than a step is one.
    with torch.no_grad():
        same = autograd.qk_norm_rope(q, k, pos, (128,), qw.bfloat16().float() * (1 + 2.0 ** -10), kw)
        other = autograd.qk_norm_rope(q, k, pos, (128,), qw * (1 + 2.0 ** -6), kw)
    assert torch.equal(same[0], y[0]) and not torch.equal(other[0], y[0])
