"""What the multi-head operators are measured on: head norms with the position
rotation (``qk_norm_rotate``) and masked attention with heads
(``head_attention``), forward and with their gradients.

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


def _ops():
    pkg = str(Path(__file__).resolve().parents[1] / "topk-tarmac_b200")
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    from tarmac_b200 import ops
    return ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
# op "rotate": B, N, H, Hk, d, dtype; r columns rotated; pairs "halves" or
#   "adjacent"; table "shared" (positions are time steps, one table) or "own"
#   (each episode has its agents' positions).
# op "attend": B, Nq, Nk, H, Hk, d, dtype; peers "all", "others" (an agent
#   leaves itself out) or "past"; lens: ragged key lengths; seen: share of the
#   pairs that a visibility mask leaves (1.0: no mask; with a mask every 17th
#   row sees nobody).
# train: the gradients too.

def _rotate(B, N, H, Hk, d, r, dtype, pairs="halves", table="shared", train=False):
    return dict(op="rotate", B=B, N=N, H=H, Hk=Hk, d=d, r=r, dtype=dtype,
                pairs=pairs, table=table, train=train)


def _attend(B, Nq, Nk, H, Hk, d, dtype, peers="others", lens=False, seen=1.0, train=False):
    return dict(op="attend", B=B, Nq=Nq, Nk=Nk, H=H, Hk=Hk, d=d, dtype=dtype,
                peers=peers, lens=lens, seen=seen, train=train)


def listed():
    cases = [
        # one environment step of a rollout: 256 episodes of 6 agents
        ("rotate_step", _rotate(256, 6, 4, 4, 16, 16, "f32", table="own")),
        # a long history prepared in one call
        ("rotate_history", _rotate(4, 8192, 16, 4, 128, 128, "bf16")),
        # training, part of the columns rotated, sizes off every grid
        ("rotate_train_odd", _rotate(37, 333, 6, 2, 40, 24, "f32", "adjacent", "own", True)),
        # training on a large batch of 512-agent episodes
        ("rotate_train_large", _rotate(1024, 512, 4, 2, 64, 32, "bf16", table="own", train=True)),
        # the attention of the same environment step
        ("attend_step", _attend(256, 6, 6, 4, 4, 16, "f32")),
        # agents with a limited field of view
        ("attend_seen", _attend(256, 512, 512, 4, 2, 64, "bf16", seen=0.25)),
        # one new token per episode over ragged histories
        ("attend_token", _attend(32, 1, 16384, 16, 2, 128, "bf16", "all", lens=True)),
        # a long history read in one call
        ("attend_long", _attend(2, 8192, 8192, 16, 4, 128, "bf16", "past")),
        # training at the single-head benchmark's sizes with four heads
        ("train_agents", _attend(64, 512, 512, 4, 4, 16, "f32", train=True)),
        # ragged episodes with a field of view, empty rows, odd sizes
        ("train_ragged", _attend(7, 777, 777, 6, 3, 80, "bf16", "past", True, 0.5, True)),
        # training with wide messages among many agents
        ("train_wide", _attend(32, 1024, 1024, 8, 8, 64, "bf16", train=True)),
        # training on long histories
        ("train_long", _attend(1, 8192, 8192, 16, 4, 128, "bf16", "past", train=True)),
    ]
    return [dict(c, name=n) for n, c in cases]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    dtype = rng.choice(["f32", "bf16", "bf16"])
    Hk = rng.choice([1, 2, 3, 4, 8])
    H = Hk * rng.choice([1, 1, 2, 4])
    # fp32 messages stay at the agents' widths
    d = rng.choice([16, 32, 64] if dtype == "f32" else [16, 32, 64, 64, 80, 96, 128])
    if rng.random() < 0.25:
        d = rng.randrange(8, d + 1, 8)
    train = rng.random() < 0.5
    if rng.random() < 0.4:
        N = _log_int(rng, 1, 8192)
        rows = _log_int(rng, 256, 100_000_000 // ((H + Hk) * d))
        return _rotate(max(1, rows // N), N, H, Hk, d, rng.choice([d, max(2, d // 4 * 2)]),
                       dtype, rng.choice(["halves", "adjacent"]),
                       rng.choice(["shared", "own"]), train)
    if rng.random() < 0.3:  # few new tokens over a history
        Nk = _log_int(rng, 64, 32768)
        B = max(1, min(_log_int(rng, 1, 128), 130_000_000 // (Nk * Hk * d)))
        return _attend(B, rng.choice([1, 1, 2, 5]), Nk, H, Hk, d, dtype,
                       rng.choice(["all", "past"]), rng.random() < 0.6)
    N = _log_int(rng, 2, 1024 if dtype == "f32" else 8192)
    B = max(1, min(_log_int(rng, 1, 512), 500_000_000 // (N * N * H),
                   100_000_000 // (N * H * d)))
    if H * N * N > 500_000_000:
        H = Hk = 4
    return _attend(B, N, N, H, Hk, d, dtype, rng.choice(["all", "others", "past"]),
                   rng.random() < 0.3, rng.choice([1.0, 1.0, 0.3, 0.7]), train)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lens(case, seed):
    """Stratified key lengths over [1, Nk], their order from the seed."""
    B, Nk = case["B"], case["Nk"]
    base = [max(1, -(-Nk * (2 * b + 1) // (2 * B))) for b in range(B)]
    g = torch.Generator().manual_seed(seed)
    return torch.tensor(base, dtype=torch.int32)[torch.randperm(B, generator=g)]


def _rows(g, B, N, heads, d, dtype):
    """The column blocks of one projection's output, as [B, N, h, d] views."""
    x = torch.randn(B, N, sum(heads) * d, generator=g, device="cuda").to(dtype)
    parts = x.split([h * d for h in heads], dim=-1)
    return [p.unflatten(-1, (h, d)) for p, h in zip(parts, heads)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]
    B, H, Hk, d = case["B"], case["H"], case["Hk"], case["d"]
    st = {"case": case}
    if case["op"] == "rotate":
        N, half = case["N"], case["r"] // 2
        st["q"], st["k"], _ = _rows(g, B, N, (H, Hk, Hk), d, t)
        for w in ("wq", "wk"):
            st[w] = 1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")
        freq = 10000.0 ** (-torch.arange(half, device="cuda") / half)
        pos = torch.arange(N, device="cuda").float()[None]
        if case["table"] == "own":
            pos = 100.0 * torch.rand(B, N, generator=g, device="cuda")
        angle = pos[..., None] * freq
        st["cos"], st["sin"] = angle.cos(), angle.sin()
        if case["train"]:
            st["dq"] = torch.randn(B, N, H, d, generator=g, device="cuda").to(t)
            st["dk"] = torch.randn(B, N, Hk, d, generator=g, device="cuda").to(t)
        return st
    Nq, Nk = case["Nq"], case["Nk"]
    if Nq == Nk:
        st["q"], st["k"], st["v"] = _rows(g, B, Nq, (H, Hk, Hk), d, t)
    else:  # new tokens beside a history kept as keys and values
        st["q"], = _rows(g, B, Nq, (H,), d, t)
        st["k"], = _rows(g, B, Nk, (Hk,), d, t)
        st["v"], = _rows(g, B, Nk, (Hk,), d, t)
    st["key_len"] = _lens(case, seed).cuda() if case["lens"] else None
    st["q_start"] = None
    if case["lens"] and Nq != Nk:  # the new tokens are each history's last
        st["q_start"] = (st["key_len"] - Nq).to(torch.int32)
    st["visible"] = None
    if case["seen"] < 1.0:
        st["visible"] = torch.rand(B, Nq, Nk, generator=g, device="cuda") < case["seen"]
        st["visible"][:, ::17] = False
    if case["train"]:
        st["dout"] = torch.randn(B, Nq, H, d, generator=g, device="cuda").to(t)
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _turn(z, cos, sin, pairs, back=False):
    """Rotate the first 2 * cos.shape[-1] columns of z [B, N, h, d]."""
    r = 2 * cos.shape[-1]
    c, s = cos[:, :, None], sin[:, :, None]
    if back:
        s = -s
    head, tail = z[..., :r], z[..., r:]
    if pairs == "halves":
        a, b = head[..., :r // 2], head[..., r // 2:]
        head = torch.cat([a * c - b * s, a * s + b * c], -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    return torch.cat([head, tail], -1)


def _rotate_plain(x, w, st):
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    return _turn(y, st["cos"], st["sin"], st["case"]["pairs"])


def _rotate_grad_plain(x, w, dy, st):
    x = x.float()
    s = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    dz = _turn(dy.float(), st["cos"], st["sin"], st["case"]["pairs"], back=True)
    xs = x * s
    dw = (dz * xs).sum((0, 1, 2))
    g = dz * w
    return s * (g - xs * (g * xs).mean(-1, keepdim=True)), dw


def _mask(st):
    """[B or 1, Nq, Nk] truth values, or None where every pair counts."""
    case = st["case"]
    Nq, Nk = case["Nq"], case["Nk"]
    j = torch.arange(Nk, device="cuda")
    i = torch.arange(Nq, device="cuda")[None, :, None]
    start = Nk - Nq if st["q_start"] is None else st["q_start"][:, None, None]
    m = st["visible"]
    if case["peers"] != "all":
        own_rule = j != start + i if case["peers"] == "others" else j <= start + i
        m = own_rule if m is None else m & own_rule
    if st["key_len"] is not None:
        inside = j < st["key_len"][:, None, None]
        m = inside if m is None else m & inside
    return m


def _attend_plain(st):
    case = st["case"]
    H, Hk, d = case["H"], case["Hk"], case["d"]
    q = st["q"].float().unflatten(2, (Hk, H // Hk)).permute(0, 2, 3, 1, 4)
    k = st["k"].float().permute(0, 2, 1, 3)[:, :, None]
    v = st["v"].float().permute(0, 2, 1, 3)[:, :, None]
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / d ** 0.5)  # [B, Hk, G, Nq, Nk]
    m = _mask(st)
    if m is not None:
        s = s.masked_fill(~m[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top.clamp_min(torch.finfo(torch.float32).min))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return q, k, v, p, torch.matmul(p, v)


def _heads_last(x, dtype):
    """[B, Hk, G, N, d] -> [B, N, Hk * G, d]."""
    return x.permute(0, 3, 1, 2, 4).flatten(2, 3).to(dtype)


def _attend_grad_plain(st, q, k, v, p, out):
    case = st["case"]
    H, Hk, d = case["H"], case["Hk"], case["d"]
    do = st["dout"].float().unflatten(2, (Hk, H // Hk)).permute(0, 2, 3, 1, 4)
    dv = torch.matmul(p.flatten(2, 3).transpose(-1, -2), do.flatten(2, 3))
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds = (ds - (do * out).sum(-1, keepdim=True)) * p
    dq = torch.matmul(ds, k) * (1.0 / d ** 0.5)
    dk = torch.matmul(ds.flatten(2, 3).transpose(-1, -2), q.flatten(2, 3)) * (1.0 / d ** 0.5)
    t = st["q"].dtype
    return (_heads_last(dq, t), dk.transpose(1, 2).to(t), dv.transpose(1, 2).to(t))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    case = st["case"]
    if own:
        return _run_own(_ops(), case, st)
    t = st["q"].dtype
    if case["op"] == "rotate":
        out = {"q": _rotate_plain(st["q"], st["wq"], st).to(t),
               "k": _rotate_plain(st["k"], st["wk"], st).to(t)}
        if case["train"]:
            dq, out["dwq"] = _rotate_grad_plain(st["q"], st["wq"], st["dq"], st)
            dk, out["dwk"] = _rotate_grad_plain(st["k"], st["wk"], st["dk"], st)
            out["dq"], out["dk"] = dq.to(t), dk.to(t)
        return out
    q, k, v, p, o = _attend_plain(st)
    out = {"out": _heads_last(o, t)}
    if case["train"]:
        out["dq"], out["dk"], out["dv"] = _attend_grad_plain(st, q, k, v, p, o)
    return out


def _run_own(ops, case, st):
    if case["op"] == "rotate":
        args = (st["q"], st["k"], st["wq"], st["wk"], st["cos"], st["sin"])
        adjacent = case["pairs"] == "adjacent"
        q, k = ops.qk_norm_rotate(*args, eps=EPS, interleaved=adjacent)
        out = {"q": q, "k": k}
        if case["train"]:
            out["dq"], out["dk"], out["dwq"], out["dwk"] = ops.qk_norm_rotate_backward(
                *args, st["dq"], st["dk"], eps=EPS, interleaved=adjacent)
        return out
    how = dict(peers=case["peers"], key_len=st["key_len"], q_start=st["q_start"],
               visible=st["visible"])
    if not case["train"]:
        return {"out": ops.head_attention(st["q"], st["k"], st["v"], **how)}
    if st["visible"] is not None:
        how["visible"] = ops.pack_visibility(st["visible"])
    o, lse = ops.head_attention(st["q"], st["k"], st["v"], return_lse=True, **how)
    dq, dk, dv = ops.head_attention_backward(st["q"], st["k"], st["v"], o, lse,
                                             st["dout"], **how)
    return {"out": o, "dq": dq, "dk": dk, "dv": dv}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    B, H, Hk, d = case["B"], case["H"], case["Hk"], case["d"]
    if case["op"] == "rotate":
        N = case["N"]
        x = B * N * (H + Hk) * d
        table = (B if case["table"] == "own" else 1) * N * case["r"] * 4
        # forward reads and writes x; the gradients read x (already read) and
        # dy and write dx
        moved = 2 * x * es + table + 8 * d
        if case["train"]:
            moved += 2 * x * es + 8 * d
        return {"bytes": moved, "flops": x * (22 if case["train"] else 8)}
    Nq, Nk = case["Nq"], case["Nk"]
    lens = _lens(case, 0).tolist() if case["lens"] else [Nk] * B
    pairs = 0
    for n in lens:
        start = (n - Nq) if case["lens"] and Nq != Nk else Nk - Nq
        if case["peers"] == "past":
            # rows see min(n, start + i + 1) keys
            full = max(0, min(Nq, Nq - (n - start - 1)))
            part = Nq - full
            first = start + 1
            lost = max(0, min(part, -start))  # rows before the first key
            part, first = part - lost, first + lost
            pairs += full * n + part * first + part * (part - 1) // 2
        else:
            pairs += Nq * n - (Nq if case["peers"] == "others" else 0)
    if case["seen"] < 1.0:
        pairs = int(pairs * case["seen"] * 16 / 17)
    rows_q, rows_k = B * Nq * H * d, sum(lens) * Hk * d
    seen = B * Nq * Nk if case["seen"] < 1.0 else 0
    moved = (2 * rows_q + 2 * rows_k) * es + seen
    flops = 4 * pairs * H * d
    if case["train"]:
        moved += (2 * rows_q + 2 * B * Nk * Hk * d) * es
        flops += 10 * pairs * H * d
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _exact_rotate(x, w, st, dy=None):
    case = st["case"]
    d, half = case["d"], case["r"] // 2
    x = x.double()
    i = torch.arange(half, device="cuda")
    a, b = (2 * i, 2 * i + 1) if case["pairs"] == "adjacent" else (i, i + half)
    # the rotation as a complex number for each pair
    turn = torch.complex(st["cos"].double(), st["sin"].double())[:, :, None]
    norm = (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt()
    unit = x / norm
    if dy is None:
        y = unit * w.double()
        z = torch.complex(y[..., a], y[..., b]) * turn
        y[..., a], y[..., b] = z.real, z.imag
        return y
    g = dy.double().clone()
    z = torch.complex(g[..., a], g[..., b]) * turn.conj()
    g[..., a], g[..., b] = z.real, z.imag
    dw = torch.einsum("bnhd,bnhd->d", g, unit)
    g = g * w.double()
    return (g - unit * (unit * g).sum(-1, keepdim=True) / d) / norm, dw


def exact(case, seed):
    heads = case["B"] * case["H"]
    if case["op"] == "attend" and (
            heads > 20_000 or heads * case["Nq"] * case["Nk"] * case["d"] > 3e11):
        return None  # over about 20 seconds
    st = prepare(case, seed)
    if case["op"] == "rotate":
        res = {"q": _exact_rotate(st["q"], st["wq"], st),
               "k": _exact_rotate(st["k"], st["wk"], st)}
        if case["train"]:
            res["dq"], res["dwq"] = _exact_rotate(st["q"], st["wq"], st, st["dq"])
            res["dk"], res["dwk"] = _exact_rotate(st["k"], st["wk"], st, st["dk"])
        return res
    B, H, Hk, d, Nq, Nk = (case[x] for x in ("B", "H", "Hk", "d", "Nq", "Nk"))
    q, k, v = (st[x].double() for x in "qkv")
    res = {"out": torch.zeros(B, Nq, H, d, dtype=torch.float64, device="cuda")}
    if case["train"]:
        res |= {"dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    col = torch.arange(Nk, device="cuda").expand(Nq, Nk)
    row = torch.arange(Nq, device="cuda")[:, None]
    for b in range(B):
        at = row + (int(st["q_start"][b]) if st["q_start"] is not None else Nk - Nq)
        shut = torch.zeros(Nq, Nk, dtype=torch.bool, device="cuda")
        if st["key_len"] is not None:
            shut |= col >= int(st["key_len"][b])
        if case["peers"] == "others":
            shut |= col == at
        elif case["peers"] == "past":
            shut |= col > at
        if st["visible"] is not None:
            shut |= ~st["visible"][b]
        blind = shut.all(-1, keepdim=True)
        for h in range(H):
            c = h * Hk // H
            w = (q[b, :, h] @ k[b, :, c].T / d ** 0.5).masked_fill_(shut, float("-inf"))
            w = torch.softmax(w.masked_fill_(blind, 0.0), -1).masked_fill_(blind, 0.0)
            o = w @ v[b, :, c]
            res["out"][b, :, h] = o
            if case["train"]:
                g = st["dout"][b, :, h].double()
                res["dv"][b, :, c] += w.T @ g
                w *= g @ v[b, :, c].T - (g * o).sum(-1, keepdim=True)
                res["dq"][b, :, h] = w @ k[b, :, c] / d ** 0.5
                res["dk"][b, :, c] += w.T @ q[b, :, h] / d ** 0.5
    return res
