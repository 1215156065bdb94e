"""What the operators of agents with a long memory are measured on: attention
with a decay for each head (``decay_attention``: over a set of rows, its
gradients, and one row at a time over a kept state) and the norms around a
block with its gate and residual scale (``residual_norm``, with gradients).

``run`` computes a case with elementary torch operations in fp32 (``own``
false) or through ``tarmac_b200.ops`` (``own`` true), on the same inputs.
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

own = False

EPS = 1e-6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CHUNK = 256  # rows that the plain form takes at once


def _ops():
    if "tarmac_b200.ops" in sys.modules:
        return sys.modules["tarmac_b200.ops"]
    pkg = str(Path(__file__).resolve().parents[1] / "topk-tarmac_b200")
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    from tarmac_b200 import ops
    return ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
# op "decay": B, N, H, Hk, d, dtype; state: starts from a kept state and
#   returns the new one; lens: ragged row counts; decay "slopes" (from half a
#   row to hundreds of rows), "strong" or "none"; train: the gradients too.
# op "norm": rows (as B, N), D, dtype; gate: with a gate; train: the gradients.

def _decay(B, N, H, Hk, d, dtype, state=False, lens=False, decay="slopes", train=False):
    return dict(op="decay", B=B, N=N, H=H, Hk=Hk, d=d, dtype=dtype, state=state, lens=lens,
                decay=decay, train=train)


def _norm(B, N, D, dtype, gate=True, train=False):
    return dict(op="norm", B=B, N=N, D=D, dtype=dtype, gate=gate, train=train)


def listed():
    cases = [
        # one environment step of a rollout: each of 256 episodes reads and
        # renews its memory
        ("decay_step", _decay(256, 1, 4, 4, 16, "f32", state=True)),
        # one new token for each of many long-lived sequences
        ("decay_step_many", _decay(512, 1, 16, 16, 128, "bf16", state=True)),
        # the agents of a small episode read as a sequence
        ("decay_short", _decay(256, 6, 4, 4, 16, "f32")),
        # a long history prepared in one call, its state kept for the steps
        ("decay_history", _decay(2, 8192, 16, 4, 128, "bf16", state=True)),
        # training at the single-head benchmark's sizes with four heads
        ("decay_train_agents", _decay(64, 512, 4, 4, 16, "f32", train=True)),
        # ragged episodes that go on from a state, odd sizes
        ("decay_train_ragged", _decay(7, 777, 6, 3, 80, "bf16", True, True, train=True)),
        # training with wide messages among many agents
        ("decay_train_wide", _decay(32, 1024, 8, 8, 64, "bf16", train=True)),
        # training on long histories
        ("decay_train_long", _decay(2, 8192, 16, 16, 128, "bf16", train=True)),
        # the messages of the same environment step join the agents' streams
        ("norm_step", _norm(256, 6, 64, "f32")),
        # the same for a long history of wide rows
        ("norm_history", _norm(4, 8192, 2048, "bf16")),
        # training, sizes off every grid
        ("norm_train_odd", _norm(37, 333, 250, "f32", False, True)),
        # training on a large batch of 512-agent episodes
        ("norm_train_large", _norm(1024, 512, 256, "bf16", True, True)),
    ]
    return [dict(c, name=n) for n, c in cases]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    dtype = rng.choice(["f32", "bf16", "bf16"])
    train = rng.random() < 0.5
    if rng.random() < 0.35:
        D = _log_int(rng, 16, 8192)
        if rng.random() < 0.6:
            D = max(16, D // 64 * 64 if D >= 128 else D // 8 * 8)
        N = _log_int(rng, 1, 8192)
        rows = _log_int(rng, 256, (130_000_000 if dtype == "bf16" else 65_000_000) // D)
        return _norm(max(1, rows // N), N, D, dtype, rng.random() < 0.7, train)
    Hk = rng.choice([1, 2, 3, 4, 8])
    H = Hk * rng.choice([1, 1, 2, 4])
    # fp32 messages stay at the agents' widths
    d = rng.choice([16, 32, 64] if dtype == "f32" else [16, 32, 64, 64, 80, 96, 128])
    if rng.random() < 0.25:
        d = rng.randrange(8, d + 1, 8)
    decay = rng.choice(["slopes", "slopes", "slopes", "strong", "none"])
    if rng.random() < 0.25:  # one new row, or a few, over a kept state
        B = max(1, min(_log_int(rng, 1, 1024), 134_000_000 // (H * d * d)))
        return _decay(B, rng.choice([1, 1, 1, 2, 5]), H, Hk, d, dtype, True, False, decay)
    N = _log_int(rng, 2, 2048 if dtype == "f32" else 32768)
    most = 4_000_000 if dtype == "f32" else 33_000_000
    B = max(1, min(_log_int(rng, 1, 512), most // (N * H * d)))
    if B * N * H * d > most:
        N = most // (H * d)
    state = rng.random() < 0.4
    return _decay(B, N, H, Hk, d, dtype, state, rng.random() < 0.3, decay, train)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lens(case, seed):
    """Stratified row counts over [1, N], their order from the seed."""
    B, N = case["B"], case["N"]
    base = [max(1, -(-N * (2 * b + 1) // (2 * B))) for b in range(B)]
    g = torch.Generator().manual_seed(seed)
    return torch.tensor(base, dtype=torch.int32)[torch.randperm(B, generator=g)]


def _rows(g, B, N, heads, d, dtype):
    """The column blocks of one projection's output, as [B, N, h, d] views."""
    x = torch.randn(B, N, sum(heads) * d, generator=g, device="cuda").to(dtype)
    parts = x.split([h * d for h in heads], dim=-1)
    return [p.unflatten(-1, (h, d)) for p, h in zip(parts, heads)]


def _rates(case, g):
    """log of each head's decay, fp32 [H]."""
    H = case["H"]
    u = torch.rand(H, generator=g, device="cuda")
    h = torch.arange(1, H + 1, device="cuda")
    if case["decay"] == "slopes":
        return -(2.0 ** (-8.0 * h / H)) * (0.75 + 0.5 * u)
    if case["decay"] == "strong":
        return -0.5 - 6.0 * u
    return torch.zeros(H, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]
    B, N = case["B"], case["N"]
    st = {"case": case}
    if case["op"] == "norm":
        D = case["D"]

        def rows():
            return torch.randn(B, N, D, generator=g, device="cuda").to(t)

        st["x"], st["y"] = rows(), rows()
        st["gate"] = rows() if case["gate"] else None
        for w, at in (("w_post", 1.0), ("w_pre", 1.0), ("scale", 0.5)):
            st[w] = at + 0.1 * torch.randn(D, generator=g, device="cuda")
        if case["train"]:
            st["dh"], st["dz"] = rows(), rows()
        return st
    H, Hk, d = case["H"], case["Hk"], case["d"]
    st["q"], st["k"], st["v"] = _rows(g, B, N, (H, Hk, Hk), d, t)
    st["log_decay"] = _rates(case, g)
    st["lens"] = _lens(case, seed).cuda() if case["lens"] else None
    st["state"] = st["next"] = None
    if case["state"]:
        st["state"] = torch.randn(B, H, d, d, generator=g, device="cuda")
        st["next"] = torch.empty_like(st["state"])  # the new state's place
    if case["train"]:
        st["dout"] = torch.randn(B, N, H, d, generator=g, device="cuda").to(t)
        st["dnext"] = None
        if case["state"]:
            st["dnext"] = torch.randn(B, H, d, d, generator=g, device="cuda")
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

class _Chunk:
    """Rows [t0, t1) of every head in fp32 ([B, H, c, d], rows from lens on
    zero), with the powers of the decays that they need."""

    def __init__(self, st, t0, t1, names):
        case = st["case"]
        B, H = case["B"], case["H"]
        c = t1 - t0
        i = torch.arange(c, device="cuda")
        n = torch.full((B,), c, device="cuda")
        if st["lens"] is not None:
            n = (st["lens"].long() - t0).clamp(0, c)
        live = i < n[:, None]
        for name in names:
            x = st[name][:, t0:t1].float()
            if st["lens"] is not None:
                x = torch.where(live[:, :, None, None], x, 0.0)
            x = x.permute(0, 2, 1, 3)
            setattr(self, name, x if x.shape[1] == H else x.repeat_interleave(H // x.shape[1], 1))
        rate = st["log_decay"][:, None, None]
        gap = (i[:, None] - i).float()
        self.w = torch.where(gap >= 0, torch.exp(rate * gap.clamp_min(0.0)), 0.0)  # [H, c, c]
        self.first = torch.exp(rate * (i + 1)[:, None])  # [H, c, 1]
        left = (n[:, None] - 1 - i)[:, None, :, None]    # [B, 1, c, 1]
        self.last = torch.where(left >= 0, torch.exp(rate * left.clamp_min(0)), 0.0)
        self.all = torch.exp(rate * n[:, None, None, None])


def _starts(N):
    return [(t, min(t + CHUNK, N)) for t in range(0, N, CHUNK)]


def _decay_plain(st):
    case = st["case"]
    B, N, H, Hk, d = (case[x] for x in ("B", "N", "H", "Hk", "d"))
    t, scale = st["q"].dtype, 1.0 / d ** 0.5
    S = st["state"]
    if S is None:
        S = torch.zeros(B, H, d, d, device="cuda")
    S0s, outs = [], []
    for t0, t1 in _starts(N):
        x = _Chunk(st, t0, t1, ("q", "k", "v"))
        if case["train"]:
            S0s.append(S)
        o = torch.matmul(torch.matmul(x.q, x.k.transpose(-1, -2)) * x.w, x.v)
        o = (o + torch.matmul(x.q, S) * x.first) * scale
        outs.append(o.permute(0, 2, 1, 3))
        S = S * x.all + torch.matmul((x.k * x.last).transpose(-1, -2), x.v)
    res = {"out": torch.cat(outs, 1).to(t)}
    if case["state"]:
        res["state"] = S
    if not case["train"]:
        return res
    R = st["dnext"]
    if R is None:
        R = torch.zeros(B, H, d, d, device="cuda")
    grads = []
    for (t0, t1), S in zip(reversed(_starts(N)), reversed(S0s)):
        x = _Chunk(st, t0, t1, ("q", "k", "v", "dout"))
        g = x.dout * scale
        pv = torch.matmul(g, x.v.transpose(-1, -2)) * x.w
        pk = torch.matmul(x.q, x.k.transpose(-1, -2)) * x.w
        dq = torch.matmul(pv, x.k) + torch.matmul(g * x.first, S.transpose(-1, -2))
        dk = torch.matmul(pv.transpose(-1, -2), x.q) + \
            torch.matmul(x.v * x.last, R.transpose(-1, -2))
        dv = torch.matmul(pk.transpose(-1, -2), g) + torch.matmul(x.k * x.last, R)
        R = R * x.all + torch.matmul((x.q * x.first).transpose(-1, -2), g)
        dk, dv = (y.unflatten(1, (Hk, H // Hk)).sum(2) for y in (dk, dv))
        grads.append([y.permute(0, 2, 1, 3) for y in (dq, dk, dv)])
    for name, parts in zip(("dq", "dk", "dv"), zip(*reversed(grads))):
        res[name] = torch.cat(parts, 1).to(t)
    if case["state"]:
        res["dstate"] = R
    return res


def _norm_plain(st):
    case = st["case"]
    x, y = st["x"].float(), st["y"].float()
    gate = 1.0 if st["gate"] is None else torch.sigmoid(st["gate"].float())
    ry = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
    yn = y * ry
    u = yn * st["w_post"]
    h = x + st["scale"] * gate * u
    rh = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    hn = h * rh
    t = st["x"].dtype
    res = {"h": h.to(t), "z": (hn * st["w_pre"]).to(t)}
    if not case["train"]:
        return res
    dz = st["dz"].float()
    a = dz * st["w_pre"]
    e = st["dh"].float() + rh * (a - hn * (a * hn).mean(-1, keepdim=True))
    res["dx"] = e.to(t)
    if st["gate"] is not None:
        res["dgate"] = (e * st["scale"] * u * gate * (1.0 - gate)).to(t)
    b = e * st["scale"] * gate
    res["dw_post"] = (b * yn).sum((0, 1))
    res["dw_pre"] = (dz * hn).sum((0, 1))
    res["dscale"] = (e * gate * u).sum((0, 1))
    b = b * st["w_post"]
    res["dy"] = (ry * (b - yn * (b * yn).mean(-1, keepdim=True))).to(t)
    return res


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    case = st["case"]
    if not own:
        return _norm_plain(st) if case["op"] == "norm" else _decay_plain(st)
    ops = _ops()
    if case["op"] == "norm":
        args = (st["x"], st["y"], st["w_post"], st["w_pre"], st["gate"], st["scale"])
        h, z = ops.residual_norm(*args, eps=EPS)
        res = {"h": h, "z": z}
        if case["train"]:
            grads = ops.residual_norm_backward(*args, st["dh"], st["dz"], eps=EPS)
            for name, g in zip(("dx", "dy", "dw_post", "dw_pre", "dgate", "dscale"), grads):
                if g is not None:
                    res[name] = g
        return res
    args = (st["q"], st["k"], st["v"], st["log_decay"])
    res = {}
    if case["state"]:
        res["out"], res["state"] = ops.decay_attention(
            *args, state=st["state"], lens=st["lens"], state_out=st["next"])
    else:
        res["out"] = ops.decay_attention(*args, lens=st["lens"])
    if case["train"]:
        res["dq"], res["dk"], res["dv"], dstate = ops.decay_attention_backward(
            *args, st["dout"], state=st["state"], dstate=st["dnext"], lens=st["lens"])
        if dstate is not None:
            res["dstate"] = dstate
    return res


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    B, N = case["B"], case["N"]
    if case["op"] == "norm":
        x, D = B * N * case["D"], case["D"]
        tiles = 4 + case["gate"]
        flops = 14 * x
        if case["train"]:  # x, y and the gate are read already
            tiles += 4 + case["gate"]
            flops += 30 * x
        return {"bytes": tiles * x * es + 4 * D * (6 if case["train"] else 3), "flops": flops}
    H, Hk, d = case["H"], case["Hk"], case["d"]
    rows = sum(_lens(case, 0).tolist()) if case["lens"] else B * N
    state = 4 * B * H * d * d if case["state"] else 0
    # q, k, v in, out out; the recurrent form's products
    moved = rows * (H + 2 * Hk) * d * es + B * N * H * d * es + 2 * state
    flops = rows * H * 5 * d * d
    if case["train"]:  # dout and the new state's gradient in, gradients out
        moved += rows * H * d * es + B * N * (H + 2 * Hk) * d * es + 2 * state
        flops += rows * H * 9 * d * d
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _exact_norm(st):
    case = st["case"]
    D = case["D"]
    x, y = st["x"].double(), st["y"].double()
    wo, wi, s = (st[n].double() for n in ("w_post", "w_pre", "scale"))
    gate = torch.ones_like(x) if st["gate"] is None else 1 / (1 + torch.exp(-st["gate"].double()))
    ny = (y.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt()
    unit = y / ny
    h = x + unit * wo * gate * s
    nh = (h.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt()
    top = h / nh
    res = {"h": h, "z": top * wi}
    if case["train"]:
        dz = st["dz"].double()
        e = dz * wi / nh
        e = st["dh"].double() + e - top * (top * e).sum(-1, keepdim=True) / D
        res["dx"] = e
        if st["gate"] is not None:
            res["dgate"] = e * s * unit * wo * gate * (1 - gate)
        res["dw_pre"] = torch.einsum("bnd,bnd->d", dz, top)
        e = e * gate
        res["dscale"] = torch.einsum("bnd,bnd->d", e, unit) * wo
        res["dw_post"] = torch.einsum("bnd,bnd->d", e, unit) * s
        f = e * s * wo / ny
        res["dy"] = f - unit * (unit * f).sum(-1, keepdim=True) / D
    return res


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(st)
    B, N, H, Hk, d = (case[x] for x in ("B", "N", "H", "Hk", "d"))
    if N * (1.0 + B * H * d * d / 4e6) * (3 if case["train"] else 1) > 2e5:
        return None  # over about 20 seconds
    # row by row: S = lambda S + k v^T, out = scale S^T q; gradients back
    # through the same steps
    lam = torch.exp(st["log_decay"].double())[:, None, None]
    scale = d ** -0.5
    share = torch.arange(H, device="cuda") * Hk // H

    def live(t):  # which episodes have a row t
        if st["lens"] is None:
            return torch.ones(B, 1, 1, dtype=torch.bool, device="cuda")
        return (st["lens"] > t)[:, None, None]

    def row(name, t):
        x = st[name][:, t].double()
        x = torch.where(live(t), x, 0.0)
        return x if x.shape[1] == H else x[:, share]

    S = torch.zeros(B, H, d, d, dtype=torch.float64, device="cuda")
    if st["state"] is not None:
        S = st["state"].double()
    res = {"out": torch.zeros(B, N, H, d, dtype=torch.float64, device="cuda")}
    if case["train"]:
        res["dq"] = torch.zeros_like(res["out"])
    for t in range(N):
        new = lam * S + row("k", t)[..., :, None] * row("v", t)[..., None, :]
        S = torch.where(live(t)[..., None], new, S)
        res["out"][:, t] = scale * (row("q", t)[..., None] * S).sum(-2)
        if case["train"]:
            res["dq"][:, t] = scale * (row("dout", t)[..., None, :] * S).sum(-1)
    if case["state"]:
        res["state"] = S
    if case["train"]:
        R = torch.zeros_like(S) if st["dnext"] is None else st["dnext"].double()
        for name in ("dk", "dv"):
            res[name] = torch.zeros(B, N, Hk, d, dtype=torch.float64, device="cuda")
        for t in range(N - 1, -1, -1):
            R = R + scale * row("q", t)[..., :, None] * row("dout", t)[..., None, :]
            dk = (R * row("v", t)[..., None, :]).sum(-1)
            dv = (R * row("k", t)[..., :, None]).sum(-2)
            for name, x in (("dk", dk), ("dv", dv)):
                res[name][:, t] = x.unflatten(1, (Hk, H // Hk)).sum(2)
            R = torch.where(live(t)[..., None], lam * R, R)
        if case["state"]:
            res["dstate"] = R
    return res
