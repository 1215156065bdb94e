"""Attention with a decay for each head on the GPU against the 64-bit form:
one row and many, odd widths, shared heads, padding, states, gradients."""

from __future__ import annotations

import math

import pytest
import torch

import _decay64 as d64

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
NAN = float("nan")


def rates(H, kind):
    if kind == "slopes":
        return -(2.0 ** (-8.0 * torch.arange(1, H + 1) / H))
    if kind == "strong":
        return -0.5 - 6.0 * torch.linspace(0, 1, H)
    if kind == "ends":  # keeps nothing, keeps all
        return torch.tensor([-math.inf, 0.0] * H)[:H]
    return torch.zeros(H)


class Case:
    def __init__(self, B, N, H, Hk, d, dtype, state=True, lens=None, decay="slopes", seed=0):
        g = torch.Generator().manual_seed(1000 * N + 10 * d + H + seed)

        def rnd(*s, t=dtype):
            return torch.randn(*s, generator=g).to(t)

        self.q, self.k, self.v = rnd(B, N, H, d), rnd(B, N, Hk, d), rnd(B, N, Hk, d)
        self.dout = rnd(B, N, H, d)
        self.state = rnd(B, H, d, d, t=F32) if state else None
        self.dstate = rnd(B, H, d, d, t=F32) if state else None
        self.rate = rates(H, decay)
        self.lens = None if lens is None else torch.tensor(lens, dtype=torch.int32)
        self.scale, self.dtype = d ** -0.5, dtype
        n = torch.full((B,), N) if lens is None else self.lens.long().clamp(0, N)
        self.pad = torch.arange(N) >= n[:, None]  # [B, N]
        self.clean = [t.clone() for t in (self.q, self.k, self.v, self.dout)]
        for t in (self.q, self.k, self.v, self.dout):
            t[self.pad] = NAN

    def want(self):
        q, k, v, g = (t.double() for t in self.clean)
        S = None if self.state is None else self.state.double()
        dS = None if self.dstate is None else self.dstate.double()
        return d64.decay_grads(q, k, v, self.rate, self.scale, g, S, self.lens, dS)

    def mags(self):
        """The same sums over absolute values: what errors are relative to."""
        q, k, v, g = (t.double().abs() for t in self.clean)
        S = None if self.state is None else self.state.double().abs()
        dS = None if self.dstate is None else self.dstate.double().abs()
        return d64.decay_grads(q, k, v, self.rate, self.scale, g, S, self.lens, dS)

    def run(self, wrap=lambda t: t):
        from tarmac_b200 import ops
        q, k, v, g = (wrap(t.cuda()) for t in (self.q, self.k, self.v, self.dout))
        S, dS, lens = (None if t is None else t.cuda() for t in (self.state, self.dstate, self.lens))
        rate = self.rate.cuda()
        out, last = ops.decay_attention(q, k, v, rate, S, lens, return_state=True)
        dq, dk, dv, first = ops.decay_attention_backward(q, k, v, rate, g, S, dS, lens)
        assert (first is None) == (S is None)
        return out, last, dq, dk, dv, first

    def check(self, got):
        """fp32 1e-5 of the sum of absolute terms: exponents up to 88 before a
        power is zero (88 2^-24), 2^-24 for each product and addition that a
        term passes (a few dozen).
        bf16: a weight of P or of b is off by 2^-8 and then the output, by each
        term; as independent errors they leave at most 2^-8 of the
        tensor's norm (three roundings of rms 2^-8 / sqrt 3 each). States
        are fp32's for both types."""
        want, mags = self.want(), self.mags()
        for i, (a, b, m) in enumerate(zip(got, want, mags)):
            if a is None:
                continue
            is_state = i in (1, 5)
            assert a.dtype == (F32 if is_state else self.dtype) and a.is_contiguous()
            a = a.double().cpu()
            err = (a - b).abs()
            if self.dtype is F32 or is_state:
                tol = 1e-5 * m
            else:
                tol = (2 ** -8 + 1e-5) * (m + b.abs())
                if b.numel() > 500:
                    assert err.norm() <= 2 ** -8 * b.norm(), (i, err.norm() / b.norm())
            assert (err <= tol + 1e-30).all(), (i, (err - tol).max(), err.max())
        for a in (got[0], got[2], got[3], got[4]):
            assert (a.cpu()[self.pad] == 0).all()


WIDTHS = [1, 3, 8, 16, 24, 32, 40, 64, 80, 100, 128]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("N", [1, 5, 67])
def test_widths(N, d, dtype):
    c = Case(2, N, 4, 2, d, dtype)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N", [2, 8, 9, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 333])
@pytest.mark.parametrize("H,Hk,d", [(3, 3, 16), (2, 1, 64)])
def test_lengths(N, H, Hk, d, dtype):
    c = Case(3, N, H, Hk, d, dtype, lens=[N, max(0, N - 3), N // 2])
    c.check(c.run())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [16, 128])
@pytest.mark.parametrize("N", [6, 700])
def test_padding(N, d, dtype):
    """Lengths out of range act like the bounds; an episode of none keeps its
    state; padding holds NaN (Case)."""
    c = Case(6, N, 2, 2, d, dtype, lens=[0, -4, N, N + 9, 1, N // 3])
    got = c.run()
    c.check(got)
    for b in (0, 1):
        assert torch.equal(got[1][b].cpu(), c.state[b])
        assert torch.equal(got[5][b].cpu(), c.dstate[b])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("decay", ["slopes", "strong", "ends", "none"])
@pytest.mark.parametrize("N,d", [(5, 32), (150, 32), (150, 128)])
def test_decays(N, d, decay, dtype):
    c = Case(2, N, 4, 4, d, dtype, decay=decay)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,N,H,Hk,d,lens", [
    (1, 1100, 1, 1, 16, None), (1, 1500, 2, 1, 64, [1333]), (2, 900, 4, 4, 128, [900, 130]),
    (1, 2000, 2, 2, 40, None)])
def test_segments(B, N, H, Hk, d, lens, dtype):
    """Few heads: the row axis is cut in segments."""
    for state in (True, False):
        c = Case(B, N, H, Hk, d, dtype, state, lens)
        c.check(c.run())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N", [4, 70, 300])
def test_without_state(N, dtype):
    c = Case(2, N, 6, 2, 48, dtype, state=False)
    c.check(c.run())


def strided(t):
    """Heads and rows swapped in memory, every second row of a larger tensor."""
    B, N, h, d = t.shape
    wide = torch.zeros(B, h, 2 * N, d + 8, device=t.device, dtype=t.dtype)
    view = wide[:, :, ::2, :d].transpose(1, 2)
    view.copy_(t)
    return view


def off_grid(t):
    """One element off the vectors' grid."""
    flat = torch.zeros(t.numel() + 1, device=t.device, dtype=t.dtype)
    view = flat[1:].view(t.shape)
    view.copy_(t)
    return view


def columns_apart(t):
    return t.transpose(1, 3).contiguous().transpose(1, 3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("wrap", [strided, off_grid, columns_apart])
@pytest.mark.parametrize("N,d", [(3, 64), (140, 64), (140, 24)])
def test_layouts(N, d, wrap, dtype):
    c = Case(2, N, 4, 2, d, dtype)
    c.check(c.run(wrap))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N", [3, 130])
def test_broadcast_keys(N, dtype):
    """Keys and values of one episode read by all (stride 0)."""
    c = Case(3, N, 2, 2, 32, dtype)
    for i in (1, 2):  # k, v
        c.clean[i] = c.clean[i][:1].expand(3, -1, -1, -1)
    c.k, c.v = c.clean[1], c.clean[2]
    c.check(c.run(lambda t: t[:1].expand(3, -1, -1, -1) if (t[0] == t[1]).all() else t))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,N,d", [(2, 1, 16), (2, 3, 128), (2, 200, 64), (1, 1300, 64)])
def test_state_in_place(B, N, d, dtype):
    from tarmac_b200 import ops
    c = Case(B, N, 2, 1, d, dtype)
    q, k, v, S, rate = (t.cuda() for t in (c.q, c.k, c.v, c.state, c.rate))
    out, want = ops.decay_attention(q, k, v, rate, S, return_state=True)
    assert torch.equal(S.cpu(), c.state)  # read only
    out2, got = ops.decay_attention(q, k, v, rate, S, state_out=S)
    assert got is S and torch.equal(S, want) and torch.equal(out, out2)


@pytest.mark.parametrize("B,N,d,segments", [(2, 100, 16, 3), (3, 1300, 32, 41), (1, 9000, 16, 188)])
def test_state_in_place_by_segments(B, N, d, segments):
    """Up to 32 columns every segment reads the state before the first row; what
    the last one writes must not reach the others."""
    from tarmac_b200 import ops
    plan = ops.decay_attention_plan(B, N, 2, 1, d, F32, state=True)
    assert plan["kernel"] == "decay_scan" and plan["segments"] == segments
    c = Case(B, N, 2, 1, d, F32)
    q, k, v, S, rate = (t.cuda() for t in (c.q, c.k, c.v, c.state, c.rate))
    lens = torch.full((B,), N, dtype=torch.int32, device="cuda")
    lens[0] = 1
    out, want = ops.decay_attention(q, k, v, rate, S, lens, return_state=True)
    for _ in range(5):
        s = S.clone()
        out2, got = ops.decay_attention(q, k, v, rate, s, lens, state_out=s)
        assert got is s and torch.equal(s, want) and torch.equal(out, out2)


def test_state_in_place_captured():
    """A captured call that renews its state, replayed: call after call."""
    from tarmac_b200 import ops
    c = Case(2, 100, 2, 1, 16, F32)
    q, k, v, S, rate = (t.cuda() for t in (c.q, c.k, c.v, c.state, c.rate))
    want, s = S.clone(), S.clone()
    for _ in range(3):
        o, want = ops.decay_attention(q, k, v, rate, want, return_state=True)
    ops.decay_attention(q, k, v, rate, S.clone(), return_state=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, _ = ops.decay_attention(q, k, v, rate, s, state_out=s)
    s.copy_(S)
    for _ in range(3):
        g.replay()
    assert torch.equal(s, want) and torch.equal(out, o)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_parts_in_turn(dtype):
    """A history in calls of unequal size, the state handed on, against one
    call: the same sums in another order (the bounds of Case.check, twice)."""
    from tarmac_b200 import ops
    c = Case(2, 300, 4, 2, 64, dtype)
    q, k, v, S, rate = (t.cuda() for t in (c.q, c.k, c.v, c.state, c.rate))
    outs, t0 = [], 0
    for n in (1, 100, 7, 64, 127, 1):
        o, S = ops.decay_attention(*(t[:, t0:t0 + n] for t in (q, k, v)), rate, S,
                                   return_state=True)
        outs.append(o)
        t0 += n
    assert t0 == 300
    want, mags = c.want(), c.mags()
    tol = 1e-5 if dtype is F32 else 2 ** -8 + 1e-5
    got = torch.cat(outs, 1).double().cpu()
    assert ((got - want[0]).abs() <= tol * (mags[0] + want[0].abs())).all()
    assert ((S.double().cpu() - want[1]).abs() <= 2e-5 * mags[1]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N", [2, 150, 1300])
def test_same_bits(N, dtype):
    c = Case(1, N, 4, 1, 64, dtype)
    for a, b in zip(c.run(), c.run()):
        assert torch.equal(a, b)


def test_empty():
    from tarmac_b200 import ops
    rate = rates(2, "slopes").cuda()
    for B, N in ((0, 5), (2, 0)):
        q = torch.zeros(B, N, 2, 16, device="cuda")
        S = torch.randn(B, 2, 16, 16, device="cuda")
        out, last = ops.decay_attention(q, q, q, rate, S, return_state=True)
        assert out.shape == q.shape and torch.equal(last, S)
        dq, dk, dv, first = ops.decay_attention_backward(q, q, q, rate, q, S, S)
        assert dq.shape == q.shape and torch.equal(first, S)
    out, last = ops.decay_attention(q, q, q, rate, return_state=True)
    assert (last == 0).all()


def test_nan_stays_in_its_head():
    """A NaN in one head's rows reaches that head's later rows only."""
    from tarmac_b200 import ops
    for N in (4, 200):
        q, k, v = torch.randn(3, 2, N, 3, 32, device="cuda")
        k[1, N // 2, 1, 3] = NAN
        out, S = ops.decay_attention(q, k, v, rates(3, "slopes").cuda(), return_state=True)
        bad = torch.zeros(2, N, 3, dtype=torch.bool, device="cuda")
        bad[1, N // 2:, 1] = True
        assert torch.equal(out.isnan().any(-1), bad)
        assert torch.equal(S.isnan().any(-1).any(-1).nonzero(), torch.tensor([[1, 1]]).cuda())


def test_graph_and_stream():
    """Captured and replayed on new inputs, and on a stream of its own."""
    from tarmac_b200 import ops
    rate = rates(4, "slopes").cuda()
    for N, dtype in ((1, F32), (200, BF16), (1300, BF16)):
        x = torch.randn(1, N, 4, 3 * 64, device="cuda").to(dtype)
        q, k, v = x.split(64, -1)
        S = torch.randn(1, 4, 64, 64, device="cuda")

        def run():
            out, last = ops.decay_attention(q, k, v, rate, S, return_state=True)
            return [out, last, *ops.decay_attention_backward(q, k, v, rate, out, S, last)]

        run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = run()
        x.copy_(torch.randn_like(x))
        g.replay()
        want = run()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            other = run()
        side.synchronize()
        for a, b, c in zip(held, want, other):
            assert torch.equal(a, b) and torch.equal(b, c)


def test_long_offsets():
    """Rows that start beyond 2^31 elements of their tensor."""
    from tarmac_b200 import ops
    N, H, d = 70, 1, 64
    big = torch.zeros(2 ** 31 + 4 * N * d, device="cuda", dtype=BF16)
    c = Case(2, N, H, H, d, BF16, state=False)
    step = 2 ** 31 + N * d
    views = []
    for i, t in enumerate((c.q, c.k, c.v)):
        view = big.as_strided((2, N, H, d), (step, d, d, 1), i * N * d)
        view.copy_(t)
        views.append(view)
    rate = c.rate.cuda()
    want = ops.decay_attention(*(t.cuda() for t in (c.q, c.k, c.v)), rate)
    assert torch.equal(ops.decay_attention(*views, rate), want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,N,H,Hk,d", [(160, 70, 3, 3, 40), (90, 130, 5, 1, 24), (320, 40, 1, 1, 72)])
def test_many_units(B, N, H, Hk, d, dtype):
    """More heads than SMs, odd numbers of heads, lengths of every kind: blocks
    walk over several units."""
    lens = [(37 * b) % (N + 3) for b in range(B)]
    c = Case(B, N, H, Hk, d, dtype, state=False, lens=lens)
    c.check(c.run())


@pytest.mark.parametrize("N,H,Hk,d", [(260, 4, 2, 64), (260, 3, 1, 16), (390, 2, 2, 128)])
def test_several_chunks_and_strong_decays(N, H, Hk, d):
    for decay in ("strong", "ends"):
        for lens in (None, [N - 130, 1]):
            c = Case(2, N, H, Hk, d, BF16, lens=lens, decay=decay)
            c.check(c.run())


def test_two_streams_at_once():
    """Calls that overlap on two streams do not share anything."""
    from tarmac_b200 import ops
    cases = [Case(1, 1500, 4, 2, 64, BF16), Case(1, 1500, 4, 2, 32, F32)]
    for c in cases:
        args = [t.cuda() for t in (c.q, c.k, c.v, c.rate, c.state)]
        want = ops.decay_attention(*args, return_state=True)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got += [ops.decay_attention(*args, return_state=True) for _ in range(5)]
        torch.cuda.synchronize()
        for out, S in got:
            assert torch.equal(out, want[0]) and torch.equal(S, want[1])


@pytest.mark.parametrize("B,d", [(1480, 16), (600, 32), (222, 48), (74, 128)])
def test_slow_decays_in_one_walk(B, d):
    """fp32 rows, one walk over all of them, heads that keep about 128 rows. A term
    m rows old is off by 8 2^-25 inside 16 rows and by 2^-25 for each 16 (on
    average 16 2^-25 = 4.8e-7, random signs over heads and rows put aside), its
    sums by the roundings of the 64 rows or so after it (rms 2^-25 each, 8 of them
    as one: 2.4e-7) and of the output: 1e-6 of the norm. A decay off by 2^-25 in
    every row would be off by 128 2^-25 = 3.8e-6."""
    from tarmac_b200 import ops
    N, H, Hk, some = 512, 2, 1, 3
    for backward in (False, True):
        plan = ops.decay_attention_plan(B, N, H, Hk, d, F32, state=True, backward=backward)
        assert plan["kernel"] == "decay_scan" and plan["segments"] == 1
    g = torch.Generator().manual_seed(d)
    q, k, v, dout = (torch.randn(B, N, h, d, generator=g) for h in (H, Hk, Hk, H))
    S, dS = (torch.randn(B, H, d, d, generator=g) for _ in range(2))
    rate = -1.0 / torch.tensor([111.0, 143.0])
    gpu = [t.cuda() for t in (q, k, v, rate, dout, S, dS)]
    got = ops.decay_attention(*gpu[:4], gpu[5], return_state=True)
    got = (*got, *ops.decay_attention_backward(*gpu[:6], gpu[6]))
    q, k, v, dout, S, dS = (t[:some].double() for t in (q, k, v, dout, S, dS))
    want = d64.decay_grads(q, k, v, rate, d ** -0.5, dout, S, None, dS)
    for i, (a, b) in enumerate(zip(got, want)):
        assert (a[:some].double().cpu() - b).norm() <= 1e-6 * b.norm(), i
