"""The operators of one windowed DiT block, forward and backward, as cases that can be timed and compared.

A case is a dict of plain values; `prepare` makes its inputs on the GPU from a seed,
`run` makes one pass: through the public entry points where `own` is true, in plain
torch with 32-bit arithmetic where it is false.  `exact` restates it in 64 bits and
`work` gives the bytes and operations it cannot do without.  Kinds of case:

  window        attention over a sliding window and a few first keys that stay visible
  window_train  the same, forward and backward: O, dq, dk, dv
  window_token  one new token per sequence against a cache of keys and values
  rope          q/k RMSNorm and rotary embedding from (time, height, width) positions, on
                the strided views of a fused QKV projection
  rope_train    the same, forward and backward: q, k, their gradients and the weights'
  norm          layer norm of [rows, C] with a scale and shift per segment of rows
  norm_train    the same, forward and backward: y, dx and the scales' and shifts' gradients

H = 56 heads, 5376 channels and S = 42120 packed tokens are the video DiT's; 28 and 14
heads are a rank's share when 2 or 4 GPUs split the heads.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

D = 128
EPS = 1e-6
THETA = 10000.0
FULL_S, FULL_H, FULL_C = 42120, 56, 5376
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _h3attn():
    """The package under test; only looked up where `own` is true."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minimaxh3-on-a100-x4_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import h3attn
    return h3attn


# ---------------------------------------------------------------------------
# cases
def listed():
    return [
        # A short clip on two heads: what a call costs before any work.
        {"name": "window_h2_s300", "kind": "window", "B": 1, "H": 2, "Hkv": 2, "S": 300, "left": 64, "right": 64,
         "sinks": 16, "causal": False, "ragged": False},
        # A padded batch of ragged causal sequences with heads that share keys, as a text or caption tower has it.
        {"name": "window_b3_h28_causal_s4104", "kind": "window", "B": 3, "H": 28, "Hkv": 4, "S": 4104, "left": 1023,
         "right": 0, "sinks": 4, "causal": True, "ragged": True},
        # The full model's layer: 512 text tokens that every video token sees, 4096 tokens to either side.
        {"name": "window_h56_s42120", "kind": "window", "B": 1, "H": FULL_H, "Hkv": FULL_H, "S": FULL_S, "left": 4096,
         "right": 4096, "sinks": 512, "causal": False, "ragged": False},
        # Fine-tuning a short clip on a rank's heads.
        {"name": "window_train_h14_s4104", "kind": "window_train", "B": 1, "H": 14, "Hkv": 14, "S": 4104, "left": 512,
         "right": 512, "sinks": 128, "causal": False, "ragged": False},
        # A training step of a longer clip on all heads, two ragged samples, heads in groups of seven.
        {"name": "window_train_b2_h56_s8192", "kind": "window_train", "B": 2, "H": FULL_H, "Hkv": 8, "S": 8192,
         "left": 1024, "right": 1024, "sinks": 256, "causal": False, "ragged": True},
        # One request, one token: latency of a step against a long cache.
        {"name": "window_token_b1_s42120", "kind": "window_token", "B": 1, "H": 28, "Hkv": 4, "S": FULL_S,
         "left": 4095, "sinks": 4},
        # A serving batch of requests at different lengths.
        {"name": "window_token_b16_s8192", "kind": "window_token", "B": 16, "H": FULL_H, "Hkv": 8, "S": 8192,
         "left": 4095, "sinks": 4},
        # The prologue of a short clip.
        {"name": "rope_h4_s300", "kind": "rope", "B": 1, "H": 4, "Hkv": 4, "S": 300, "axes": "44,42,42"},
        # The full model's prologue, and a training step of a shorter clip with a part of the dims unrotated.
        {"name": "rope_h56_s42120", "kind": "rope", "B": 1, "H": FULL_H, "Hkv": FULL_H, "S": FULL_S,
         "axes": "44,42,42"},
        {"name": "rope_train_h56_s8192", "kind": "rope_train", "B": 1, "H": FULL_H, "Hkv": FULL_H, "S": 8192,
         "axes": "32,32,32"},
        # The norm in front of a layer over the packed sequence: 13 segments, each with its own scale and shift.
        {"name": "norm_s42120_c5376", "kind": "norm", "rows": FULL_S, "C": FULL_C, "segments": 13, "dtype": "bf16"},
        {"name": "norm_train_s42120_c5376", "kind": "norm_train", "rows": FULL_S, "C": FULL_C, "segments": 13,
         "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _head_pair(rng):
    return rng.choice([(2, 2), (4, 4), (14, 14), (14, 2), (28, 28), (28, 4), (56, 56), (56, 8), (8, 1), (24, 8)])


def draw(rng):
    kind = rng.choice(["window", "window", "window_train", "window_train", "window_token", "window_token", "rope",
                       "rope_train", "norm", "norm_train"])
    if kind in ("window", "window_train"):
        B = rng.choice([1, 1, 2, 3])
        H, Hkv = _head_pair(rng)
        S = _log_int(rng, 65, (FULL_S if kind == "window" else 8192) // B)
        causal = rng.random() < 0.4
        left = _log_int(rng, 16, 4096 if kind == "window" else 1024)
        return {"kind": kind, "B": B, "H": H, "Hkv": Hkv, "S": S, "left": left,
                "right": 0 if causal else rng.choice([left, left, _log_int(rng, 1, left)]),
                "sinks": rng.choice([0, 1, 4, _log_int(rng, 8, 512 if kind == "window" else 256)]), "causal": causal,
                "ragged": rng.random() < 0.4}
    if kind == "window_token":
        H, Hkv = rng.choice([(2, 2), (4, 4), (14, 2), (28, 4), (56, 8), (8, 1), (24, 8)])
        S = _log_int(rng, 300, FULL_S)
        return {"kind": kind, "B": _log_int(rng, 1, max(1, min(64, 65536 // S))), "H": H, "Hkv": Hkv, "S": S,
                "left": _log_int(rng, 127, 8191), "sinks": rng.choice([0, 4, 16])}
    if kind in ("rope", "rope_train"):
        H, Hkv = _head_pair(rng)
        return {"kind": kind, "B": 1, "H": H, "Hkv": Hkv, "S": _log_int(rng, 64, FULL_S if kind == "rope" else 8192),
                "axes": rng.choice(["44,42,42", "32,32,32", "16,56,56", "64,64", "128"])}
    C = rng.choice([FULL_C, _log_int(rng, 64, 8192), 8 * _log_int(rng, 8, 1024)])
    rows = _log_int(rng, 16, max(16, FULL_S * FULL_C // C // 2))
    return {"kind": kind, "rows": min(rows, 200000), "C": C, "segments": rng.choice([1, 1, 2, 13]),
            "dtype": rng.choice(["bf16", "bf16", "fp32", "fp16"])}


# ---------------------------------------------------------------------------
# inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFFFFFF)
    return g


def _lens(case):
    """Lengths of a batch's sequences, between a third of the buffer and all of it (the longest fills it)."""
    B, S = case["B"], case["S"]
    lens = [S // 3 + 104729 * b % (S - S // 3) for b in range(B)]
    lens[0] = S
    return lens


def _segments(case):
    """Bounds of the segments of rows: uneven, the text, condition and audio parts being shorter than the video's."""
    n, rows = case["segments"], case["rows"]
    return [rows * i * i // (n * n) for i in range(n + 1)]


def _axes(case):
    """Rotated dims of each position axis."""
    return tuple(int(d) for d in case["axes"].split(","))


def _positions(S, axes, gen):
    """(time, height, width) of packed tokens: text first, at one position after the other on every axis, then frames."""
    A = len(axes)
    text = min(S // 8, 512)
    n = torch.arange(S - text, device="cuda")
    w, h = 52, 30
    cols = {1: [n], 2: [n // w, n % w], 3: [n // (w * h), n // w % h, n % w]}[A]
    shift = torch.randint(0, 1000, (1,), generator=gen, device="cuda")
    video = torch.stack(cols, dim=1) + text + shift
    head = (torch.arange(text, device="cuda") + shift)[:, None].expand(text, A)
    return torch.cat([head, video]).to(torch.int32).contiguous()


def prepare(case, seed):
    gen = _gen(seed)
    kind = case["kind"]

    def randn(*shape, dtype=torch.bfloat16, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    st = dict(case)
    if kind.startswith("window"):
        B, H, Hkv, S = case["B"], case["H"], case["Hkv"], case["S"]
        Sq = 1 if kind == "window_token" else S
        # Sequence-major memory, as the projections leave it: [B,S,H,D] seen as [B,H,S,D].
        st["q"] = randn(B, Sq, H, D).transpose(1, 2)
        st["k"] = randn(B, S, Hkv, D).transpose(1, 2)
        st["v"] = randn(B, S, Hkv, D).transpose(1, 2)
        # Keys drift along the sequence and the first ones draw attention, as learned sinks do.
        st["k"][:, :, :4] *= 1.5
        st["kv_lens"] = st["q_start"] = None
        if kind == "window_token":
            lens = torch.tensor(_lens(case), device="cuda", dtype=torch.int32)
            st["kv_lens"], st["q_start"] = lens, lens - 1
        elif case["ragged"]:
            st["kv_lens"] = torch.tensor(_lens(case), device="cuda", dtype=torch.int32)
        if kind == "window_train":
            st["do"] = randn(B, Sq, H, D).transpose(1, 2)
        return st
    if kind.startswith("rope"):
        B, H, Hkv, S = case["B"], case["H"], case["Hkv"], case["S"]
        qkv = randn(B, S, (H + 2 * Hkv) * D)
        st["q"] = qkv[..., :H * D].view(B, S, H, D)
        st["k"] = qkv[..., H * D:(H + Hkv) * D].view(B, S, Hkv, D)
        st["axes"] = _axes(case)
        st["pos"] = _positions(S, st["axes"], gen)
        st["qw"] = (1 + randn(D, dtype=torch.float32, scale=0.1)).to(torch.bfloat16)
        st["kw"] = (1 + randn(D, dtype=torch.float32, scale=0.1)).to(torch.bfloat16)
        if kind == "rope_train":
            st["dq"], st["dk"] = randn(B, S, H, D), randn(B, S, Hkv, D)
        return st
    rows, C, dt = case["rows"], case["C"], DT[case["dtype"]]
    # A residual stream: channels of different scale, a few large, a common offset.
    scale = torch.exp(0.5 * torch.randn(C, generator=gen, device="cuda"))
    st["x"] = (torch.randn(rows, C, generator=gen, device="cuda") * scale + 0.3).to(dt)
    st["scale"] = randn(case["segments"], C, dtype=dt, scale=0.2)
    st["shift"] = randn(case["segments"], C, dtype=dt, scale=0.2)
    st["bounds"] = _segments(case)
    if kind == "norm_train":
        st["dy"] = randn(rows, C, dtype=dt)
    return st


# ---------------------------------------------------------------------------
# plain form: elementary torch operations in 32 bits, rounded once at the end
CHUNK = 512


def _repeat(x, n):
    return x.float().repeat_interleave(n, dim=1) if n > 1 else x.float().contiguous()


def _plain_ranges(s, i0, n):
    """Slices of keys that query rows i0 .. i0+n-1 can see: the first ones, and the window's."""
    S = s["k"].shape[2]
    if s["kind"] == "window_token":
        return [(0, S)]
    lo, hi, first = max(0, i0 - s["left"]), min(S, i0 + n + s["right"]), min(S, s["sinks"])
    return [(0, max(hi, first))] if first >= lo else [(0, first), (lo, hi)]


def _plain_scores(s, q, k, i0, n):
    """Visible-or-minus-infinity scores of a chunk of rows, and the key indices they are against."""
    dev = q.device
    B = q.shape[0]
    j = torch.cat([torch.arange(a, b, device=dev) for a, b in _plain_ranges(s, i0, n)])
    pos = torch.arange(i0, i0 + n, device=dev)[None, :].expand(B, n)
    if s["q_start"] is not None:
        pos = pos + s["q_start"][:, None]
    lens = torch.full((B,), k.shape[2], device=dev) if s["kv_lens"] is None else s["kv_lens"]
    p, jj, ll = pos[:, None, :, None], j[None, None, None, :], lens[:, None, None, None]
    seen = ((jj >= p - s["left"]) & (jj <= p + s.get("right", 0))) | (jj < s["sinks"])
    if s.get("causal", True):
        seen = seen & (jj <= p)
    seen = seen & (jj < ll) & (p < ll)
    sc = torch.matmul(q, k[:, :, j].transpose(2, 3).contiguous()) / math.sqrt(D)
    return torch.where(seen, sc, torch.full_like(sc, -math.inf)), j


def _plain_softmax(sc):
    top = sc.amax(dim=-1, keepdim=True)
    e = torch.exp(sc - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_window(s):
    H, Hkv = s["q"].shape[1], s["k"].shape[1]
    rep = H // Hkv
    q, k, v = s["q"].float().contiguous(), _repeat(s["k"], rep), _repeat(s["v"], rep)
    train = s["kind"] == "window_train"
    o = torch.empty_like(q)
    if train:
        do = s["do"].float().contiguous()
        dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    Sq = q.shape[2]
    for i0 in range(0, Sq, CHUNK):
        n = min(CHUNK, Sq - i0)
        qc = q[:, :, i0:i0 + n].contiguous()
        sc, j = _plain_scores(s, qc, k, i0, n)
        p = _plain_softmax(sc)
        vj = v[:, :, j]
        o[:, :, i0:i0 + n] = torch.matmul(p, vj)
        if train:
            g = do[:, :, i0:i0 + n].contiguous()
            dp = torch.matmul(g, vj.transpose(2, 3).contiguous())
            ds = p * (dp - (p * dp).sum(dim=-1, keepdim=True)) / math.sqrt(D)
            dq[:, :, i0:i0 + n] = torch.matmul(ds, k[:, :, j])
            dk.index_add_(2, j, torch.matmul(ds.transpose(2, 3).contiguous(), qc))
            dv.index_add_(2, j, torch.matmul(p.transpose(2, 3).contiguous(), g))
    dt = s["q"].dtype
    if not train:
        return o.to(dt)
    B, _, S, _ = k.shape
    dk = dk.view(B, Hkv, rep, S, D).sum(dim=2)
    dv = dv.view(B, Hkv, rep, S, D).sum(dim=2)
    return o.to(dt), dq.to(dt), dk.to(dt), dv.to(dt)


def _plain_cos_sin(pos, axes):
    """Cosine and sine of every pair's angle, the angles taken in 64 bits."""
    ang = []
    for a, d in enumerate(axes):
        freq = THETA ** (-2.0 * torch.arange(d // 2, device=pos.device, dtype=torch.float64) / d)
        ang.append(pos[:, a].double()[:, None] * freq[None, :])
    ang = torch.cat(ang, dim=1)
    return torch.cos(ang).float()[None, :, None, :], torch.sin(ang).float()[None, :, None, :]


def _plain_rope(s):
    c, sn = _plain_cos_sin(s["pos"], s["axes"])
    half = c.shape[-1]
    outs, grads, wgrads = [], [], []
    for name in ("q", "k"):
        x, w = s[name].float(), s[name + "w"].float()
        r = torch.rsqrt(x.pow(2).mean(dim=-1, keepdim=True) + EPS)
        y = x * r * w
        a, b, rest = y[..., :half], y[..., half:2 * half], y[..., 2 * half:]
        outs.append(torch.cat([a * c - b * sn, a * sn + b * c, rest], dim=-1).to(torch.bfloat16))
        if s["kind"] == "rope_train":
            g = s["d" + name].float()
            a, b, rest = g[..., :half], g[..., half:2 * half], g[..., 2 * half:]
            g = torch.cat([a * c + b * sn, b * c - a * sn, rest], dim=-1)
            wgrads.append((g * x * r).sum(dim=(0, 1, 2)))
            gw = g * w
            grads.append((r * (gw - x * r * r * (x * gw).mean(dim=-1, keepdim=True))).to(torch.bfloat16))
    return tuple(outs + grads + wgrads)


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(dim=1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt(xc.pow(2).mean(dim=1, keepdim=True) + EPS)
    xh = xc * rstd
    y, dx = torch.empty_like(x), torch.empty_like(x)
    b = s["bounds"]
    dscale, dshift = [], []
    for n in range(len(b) - 1):
        rows = slice(b[n], b[n + 1])
        w = 1 + s["scale"][n].float()
        y[rows] = xh[rows] * w + s["shift"][n].float()
        if s["kind"] == "norm_train":
            g = s["dy"][rows].float()
            dscale.append((g * xh[rows]).sum(dim=0))
            dshift.append(g.sum(dim=0))
            gw = g * w
            dx[rows] = rstd[rows] * (gw - gw.mean(dim=1, keepdim=True)
                                     - xh[rows] * (gw * xh[rows]).mean(dim=1, keepdim=True))
    dt = s["x"].dtype
    if s["kind"] == "norm":
        return y.to(dt)
    return y.to(dt), dx.to(dt), torch.stack(dscale), torch.stack(dshift)


# ---------------------------------------------------------------------------
# the framework's entry points
def _own_window(s):
    h3 = _h3attn()
    kw = dict(window=(s["left"], s.get("right", 0)), sinks=s["sinks"], causal=s.get("causal", True),
              q_start=s["q_start"], kv_lens=s["kv_lens"])
    if s["kind"] != "window_train":
        return h3.attn_fwd_window(s["q"], s["k"], s["v"], **kw)
    o, lse = h3.attn_fwd_window(s["q"], s["k"], s["v"], return_lse=True, **kw)
    dq, dk, dv = h3.attn_bwd_window(s["do"], s["q"], s["k"], s["v"], o, lse, **kw)
    return o, dq, dk, dv


def _own_rope(s):
    h3 = _h3attn()
    args = (s["q"], s["k"], s["pos"], s["axes"], s["qw"], s["kw"])
    q, k = h3.qk_rmsnorm_rope_axes(*args, eps=EPS, theta=THETA)
    if s["kind"] == "rope":
        return q, k
    dq, dk, dqw, dkw = h3.qk_rmsnorm_rope_axes_bwd(s["dq"], s["dk"], *args, eps=EPS, theta=THETA)
    return q, k, dq, dk, dqw, dkw


def _own_norm(s):
    h3 = _h3attn()
    kw = dict(segments=s["bounds"], modulate=True)
    if s["kind"] == "norm":
        return h3.layer_norm_fwd(s["x"], s["scale"], s["shift"], eps=EPS, **kw)
    y, mean, rstd = h3.layer_norm_fwd(s["x"], s["scale"], s["shift"], eps=EPS, return_stats=True, **kw)
    dx, dscale, dshift = h3.layer_norm_bwd(s["dy"], s["x"], s["scale"], mean, rstd, **kw)
    return y, dx, dscale, dshift


def run(state):
    kind = state["kind"].split("_")[0]
    if own:
        return {"window": _own_window, "rope": _own_rope, "norm": _own_norm}[kind](state)
    return {"window": _plain_window, "rope": _plain_rope, "norm": _plain_norm}[kind](state)


# ---------------------------------------------------------------------------
# 64-bit restatements, one head or one block of rows at a time
def _exact_window(case, s):
    B, H, Hkv = case["B"], case["H"], case["Hkv"]
    q, k, v = s["q"], s["k"], s["v"]
    Sq, S = q.shape[2], k.shape[2]
    token, train = case["kind"] == "window_token", case["kind"] == "window_train"
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    dq = torch.zeros_like(o) if train else None
    dk = torch.zeros(k.shape, dtype=torch.float64, device=q.device) if train else None
    dv = torch.zeros_like(dk) if train else None
    lens = [S] * B if s["kv_lens"] is None else s["kv_lens"].tolist()
    left, right, causal = case["left"], case.get("right", 0), case.get("causal", True)
    for b in range(B):
        start, n_keys = (lens[b] - 1 if token else 0), lens[b]
        for i0 in range(0, Sq, 2048):
            i1 = min(Sq, i0 + 2048, n_keys - start)
            if i1 <= i0:
                continue
            first, last = start + i0, start + i1 - 1
            lo, hi = max(0, first - left), min(n_keys, last + right + 1)
            idx = [x for x in range(min(case["sinks"], lo, n_keys))] + list(range(lo, hi))
            if lo < case["sinks"]:  # first keys past the window's end
                idx += [x for x in range(hi, min(case["sinks"], n_keys))]
            cols = torch.tensor(idx, device=q.device)
            pos = torch.arange(first, last + 1, device=q.device)[:, None]
            away = cols[None, :] - pos
            hidden = ((away < -left) | (away > right)) & (cols >= case["sinks"])[None, :]
            if causal:
                hidden |= away > 0
            for h in range(H):
                kh, vh = k[b, h * Hkv // H, cols].double(), v[b, h * Hkv // H, cols].double()
                qh = q[b, h, i0:i1].double()
                logits = (qh @ kh.T).mul_(D ** -0.5).masked_fill_(hidden, -math.inf)
                prob = torch.softmax(logits, dim=1)
                o[b, h, i0:i1] = prob @ vh
                if train:
                    gh = s["do"][b, h, i0:i1].double()
                    dlog = gh @ vh.T
                    dlog -= (gh * o[b, h, i0:i1]).sum(dim=1, keepdim=True)
                    dlog *= prob
                    dlog *= D ** -0.5
                    dq[b, h, i0:i1] = dlog @ kh
                    dk[b, h * Hkv // H].index_add_(0, cols, dlog.T @ qh)
                    dv[b, h * Hkv // H].index_add_(0, cols, prob.T @ gh)
    return (o, dq, dk, dv) if train else o


def _exact_rope(case, s):
    exps = torch.cat([torch.arange(d // 2, dtype=torch.float64) * (2.0 / d) for d in s["axes"]])
    axis = torch.cat([torch.full((d // 2,), a) for a, d in enumerate(s["axes"])]).to(s["pos"].device)
    ang = s["pos"].double()[:, axis] * torch.exp(-math.log(THETA) * exps).to(s["pos"].device)
    turn = torch.polar(torch.ones_like(ang), ang)[:, None, :]  # complex [S, 1, half]
    half = len(axis)
    outs, grads, wgrads = [], [], []
    for name in ("q", "k"):
        y_all, dx_all = [], []
        w = s[name + "w"].double()
        dw = torch.zeros_like(w)
        for i in range(0, case["S"], 4096):
            x, t = s[name][:, i:i + 4096].double(), turn[i:i + 4096]
            rms = (x.square().sum(dim=-1, keepdim=True) / D + EPS).sqrt()
            y = x / rms * w
            z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * t
            y_all.append(torch.cat([z.real, z.imag, y[..., 2 * half:]], dim=-1))
            if case["kind"] == "rope_train":
                g = s["d" + name][:, i:i + 4096].double()
                z = torch.complex(g[..., :half].contiguous(), g[..., half:2 * half].contiguous()) * t.conj()
                g = torch.cat([z.real, z.imag, g[..., 2 * half:]], dim=-1)
                dw += (g * x / rms).sum(dim=(0, 1, 2))
                gw = g * w
                dx_all.append(gw / rms - x * (x * gw).sum(dim=-1, keepdim=True) / (D * rms ** 3))
        outs.append(torch.cat(y_all, dim=1))
        if dx_all:
            grads.append(torch.cat(dx_all, dim=1))
            wgrads.append(dw)
    return tuple(outs + grads + wgrads)


def _exact_norm(case, s):
    train = case["kind"] == "norm_train"
    ys, dxs, dscales, dshifts = [], [], [], []
    b = s["bounds"]
    for n in range(case["segments"]):
        w, c = s["scale"][n].double() + 1, s["shift"][n].double()
        dw, db = torch.zeros_like(w), torch.zeros_like(w)
        for i in range(b[n], b[n + 1], 8192):
            x = s["x"][i:min(i + 8192, b[n + 1])].double()
            var, mu = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
            sd = (var + EPS).sqrt()
            z = (x - mu) / sd
            ys.append(z * w + c)
            if train:
                g = s["dy"][i:min(i + 8192, b[n + 1])].double()
                dw += (g * z).sum(dim=0)
                db += g.sum(dim=0)
                g = g * w
                dxs.append((g - g.mean(dim=1, keepdim=True) - z * (g * z).mean(dim=1, keepdim=True)) / sd)
        dscales.append(dw)
        dshifts.append(db)
    return (torch.cat(ys), torch.cat(dxs), torch.stack(dscales), torch.stack(dshifts)) if train else torch.cat(ys)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"].split("_")[0]
    return {"window": _exact_window, "rope": _exact_rope, "norm": _exact_norm}[kind](case, s)


# ---------------------------------------------------------------------------
# work
def _pairs(case):
    """Visible (query, key) pairs of one head over the batch, all sequences taken at full length unless ragged."""
    S = case["S"]
    left, right, sinks, causal = case["left"], case.get("right", 0), case["sinks"], case.get("causal", True)
    if causal:
        right = 0
    lens = [S] * case["B"] if not case.get("ragged") else _lens(case)
    total = 0
    for n in lens:
        for i in ([n - 1] if case["kind"] == "window_token" else range(n)):
            lo, hi = max(0, i - left), min(n - 1, i + right)
            total += hi - lo + 1
            top = min(sinks, n, i + 1 if causal else n)  # visible first keys
            total += max(0, min(top, lo)) + max(0, top - max(hi + 1, lo))
    return total


def work(case):
    kind = case["kind"]
    if kind.startswith("window"):
        B, H, Hkv, S = case["B"], case["H"], case["Hkv"], case["S"]
        pairs = _pairs(case)
        if kind == "window_token":
            keys = pairs  # per kv head, over the batch
            return {"bytes": 2 * keys * Hkv * D * 2 + 2 * B * H * D * 2, "flops": 4 * D * H * pairs}
        qo, kv = B * H * S * D * 2, B * Hkv * S * D * 2
        if kind == "window":
            return {"bytes": 2 * qo + 2 * kv, "flops": 4 * D * H * pairs}
        return {"bytes": 4 * qo + 4 * kv, "flops": 14 * D * H * pairs}
    if kind.startswith("rope"):
        row = case["B"] * case["S"] * (case["H"] + case["Hkv"]) * D
        n_axes = len(_axes(case))
        if kind == "rope":
            return {"bytes": 2 * 2 * row + 4 * case["S"] * n_axes, "flops": 8 * row}
        return {"bytes": 2 * 4 * row + 4 * case["S"] * n_axes, "flops": 24 * row}
    size = 2 if case["dtype"] != "fp32" else 4
    n = case["rows"] * case["C"]
    vec = case["segments"] * case["C"]
    if kind == "norm":
        return {"bytes": size * (2 * n + 2 * vec), "flops": 8 * n}
    return {"bytes": size * (4 * n + 2 * vec) + 8 * vec, "flops": 20 * n}
