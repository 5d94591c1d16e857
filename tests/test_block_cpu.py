"""Layer norm and the prologue from positions without a GPU: refusals, and the float64 references
that the GPU tests use against central differences."""
from __future__ import annotations

import ctypes

import pytest
import torch

import block_ref as ref
import h3attn
from h3attn import _lib, block

S3 = _lib.strides3
ROW = S3(0, 128, 128)


def _rope(L, q=16, B=1, S=2, Hq=2, Hk=1, D=128, st=(ROW,) * 4, pos=16, axes=(44, 42, 42), n=None, theta=1e4,
          eps=1e-6, qw=16, stride=0):
    dims = (ctypes.c_int * 4)(*axes)
    p = _lib.Positions(pos, stride, 0, len(axes) if n is None else n, dims, theta)
    return L.h3a_qk_rmsnorm_rope_axes(q, 16, 16, 16, B, S, Hq, Hk, D, *st, ctypes.byref(p), qw, 16, eps, None)


def test_rope_refusals():
    L = _lib.lib()
    bad, unsup, align = _lib.H3A_ERR_INVALID_ARG, _lib.H3A_ERR_UNSUPPORTED, _lib.H3A_ERR_ALIGNMENT
    for kw in ({"B": 0}, {"S": -1}, {"Hq": 0}, {"Hk": 0}, {"q": None}, {"pos": None}, {"qw": None}, {"theta": 0.0},
               {"theta": float("nan")}, {"eps": -1.0}, {"stride": -1}):
        assert _rope(L, **kw) == bad, kw
    for kw in ({"D": 64}, {"axes": (43, 43, 42)}, {"axes": (64, 66)}, {"axes": (0, 128)}, {"axes": (20,)}, {"n": 0},
               {"n": 5}):
        assert _rope(L, **kw) == unsup, kw
    for kw in ({"q": 24}, {"qw": 8}, {"pos": 18}, {"st": (S3(0, 12, 128), ROW, ROW, ROW)}):
        assert _rope(L, **kw) == align, kw
    assert _rope(L, st=(ROW, ROW, S3(0, 64, 128), ROW)) == bad  # written rows overlap
    n = ctypes.c_size_t(0)
    size = L.h3a_qk_rmsnorm_rope_axes_bwd_workspace_size
    assert size(1, 2, None) == bad and size(0, 2, ctypes.byref(n)) == bad
    assert size(1, 2, ctypes.byref(n)) == 0 and n.value > 0
    dims = (ctypes.c_int * 4)(44, 42, 42)
    p = _lib.Positions(16, 0, 0, 3, dims, 1e4)

    def bwd(gw=16, ws=16, nbytes=n.value, dq=16):
        return L.h3a_qk_rmsnorm_rope_axes_bwd(dq, 16, 16, 16, 16, 16, gw, 16, 1, 2, 2, 1, 128, *(ROW,) * 6,
                                              ctypes.byref(p), 16, 16, 1e-6, ws, nbytes, None)

    assert bwd(dq=None) == bad and bwd(gw=None) == bad and bwd(ws=None) == bad and bwd(nbytes=n.value - 1) == bad
    assert bwd(gw=18) == align and bwd(ws=24) == align


def test_norm_refusals():
    L = _lib.lib()
    bad, unsup, align = _lib.H3A_ERR_INVALID_ARG, _lib.H3A_ERR_UNSUPPORTED, _lib.H3A_ERR_ALIGNMENT
    ints = lambda *b: (ctypes.c_int * len(b))(*b)  # noqa: E731

    def fwd(x=16, xs=64, y=16, ys=64, mean=None, rstd=None, rows=4, C=64, dt=0, wdt=2, bounds=(0, 4), eps=1e-6, w=16):
        return L.h3a_layer_norm_fwd(x, xs, w, 16, y, ys, mean, rstd, rows, C, dt, wdt, ints(*bounds), len(bounds) - 1,
                                    0, eps, None)

    for kw in ({"x": None}, {"y": None}, {"rows": -1}, {"C": 0}, {"mean": 16}, {"bounds": (0, 3)}, {"bounds": (1, 4)},
               {"bounds": (0, 3, 2, 4)}, {"bounds": (0,)}, {"ys": 63}, {"xs": -64}, {"eps": -1.0},
               {"eps": float("inf")}):
        assert fwd(**kw) == bad, kw
    for kw in ({"C": 16385}, {"dt": 3}, {"wdt": -1}):
        assert fwd(**kw) == unsup, kw
    for kw in ({"x": 17}, {"w": 18}):
        assert fwd(**kw) == align, kw
    n = ctypes.c_size_t(0)
    size = L.h3a_layer_norm_bwd_workspace_size
    assert size(None, 1, 64, ctypes.byref(n)) == bad and size(ints(0, 4), 1, 64, None) == bad
    assert size(ints(0, 4), 1, 64, ctypes.byref(n)) == 0 and n.value > 0

    def bwd(mean=16, dw=16, db=16, ws=16, nbytes=n.value, dy=16):
        return L.h3a_layer_norm_bwd(dy, 64, 16, 64, 16, mean, 16, 16, 64, dw, db, 4, 64, 0, 2, ints(0, 4), 1, 0, ws,
                                    nbytes, None)

    for kw in ({"mean": None}, {"dw": None}, {"ws": None}, {"nbytes": n.value - 1}, {"dy": None}):
        assert bwd(**kw) == bad, kw
    assert bwd(ws=24) == align


def test_python_refusals(monkeypatch):
    x = torch.zeros(6, 64)
    with pytest.raises(ValueError, match="GPU"):
        h3attn.layer_norm_fwd(x)
    q = torch.zeros(1, 4, 2, 128, dtype=torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16)
    pos = torch.zeros(4, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        h3attn.qk_rmsnorm_rope_axes(q, q, pos, (44, 42, 42), w, w)
    with pytest.raises(ValueError, match="bf16"):
        h3attn.qk_rmsnorm_rope_axes(q.float(), q, pos, (44, 42, 42), w, w)
    monkeypatch.setattr(block, "_rope_input", lambda name, t, device=None: (t, S3(*t.stride()[:3])))
    for match, p, axes in (("axes", pos, ()), ("axes", pos, (44, 42, 41)), ("axes", pos, (64, 64, 64)),
                           ("axes", pos, (44, 42, 44)), ("int32", pos.long(), (44, 42, 42)),
                           ("positions", pos, (64, 64)), ("positions", pos[:3], (44, 42, 42))):
        with pytest.raises(ValueError, match=match):
            h3attn.qk_rmsnorm_rope_axes(q, q, p, axes, w, w)
    with pytest.raises(ValueError, match="share batch"):
        h3attn.qk_rmsnorm_rope_axes(q, q[:, :3], pos, (44, 42, 42), w, w)
    with pytest.raises(ValueError, match="out"):
        h3attn.qk_rmsnorm_rope_axes(q, q, pos, (44, 42, 42), w, w, out=(q.float(), q))
    with pytest.raises(ValueError, match="128 elements"):
        h3attn.qk_rmsnorm_rope_axes(q, q, pos, (44, 42, 42), w[:64], w)


def test_references_against_differences():
    g = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, b, dy = rnd(5, 12), rnd(2, 12), rnd(2, 12), rnd(5, 12)
    bounds, h = [0, 3, 5], 1e-6
    f = lambda: (ref.norm(x, w, b, bounds, 1e-3, 1.0)[0] * dy).sum().item()  # noqa: E731
    ref.U[torch.float64] = 0.0
    grads, _ = ref.norm_grads(dy, x, w, bounds, 1e-3, 1.0)
    q, qw, dq = rnd(1, 3, 2, 128), rnd(128), rnd(1, 3, 2, 128)
    ang = ref.angles(torch.tensor([[[3, 5], [70, -2], [1000, 9]]]), (32, 64), 100.0)
    rf = lambda: (ref.rope(q, ang, qw, 1e-3)[0] * dq).sum().item()  # noqa: E731
    rgrads, _ = ref.rope_grads(dq, q, ang, qw, 1e-3)
    for fn, t, grad in ((f, x, grads[0]), (f, w, grads[1]), (f, b, grads[2]), (rf, q, rgrads[0]), (rf, qw, rgrads[1])):
        flat, gflat = t.view(-1), grad.reshape(-1)
        for i in range(0, flat.numel(), max(1, flat.numel() // 17)):
            v = flat[i].item()
            flat[i] = v + h
            up = fn()
            flat[i] = v - h
            down = fn()
            flat[i] = v
            assert abs((up - down) / (2 * h) - gflat[i].item()) < 1e-6 * (1 + abs(gflat[i].item()))


def test_norm_rows_past_the_limit():
    L = _lib.lib()
    rows = (1 << 30) + 1
    bounds = (ctypes.c_int * 2)(0, rows)
    assert L.h3a_layer_norm_fwd(16, 64, 16, 16, 16, 64, None, None, rows, 64, 0, 2, bounds, 1, 0, 1e-6,
                                None) == _lib.H3A_ERR_UNSUPPORTED
    assert L.h3a_layer_norm_bwd_workspace_size(bounds, 1, 64, ctypes.byref(ctypes.c_size_t(0))) == _lib.H3A_ERR_UNSUPPORTED
    with pytest.raises(ValueError, match="rows"):
        block._bounds(None, rows, None)
