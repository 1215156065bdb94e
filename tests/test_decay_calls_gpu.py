"""Calls of the operators with a memory of fixed size as programs make them: training
captured into graphs, inference mode, many heads, states and lengths of other
layouts and types, results used on other streams."""

from __future__ import annotations

import gc

import pytest
import torch

import _decay64 as d64

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def rows(B, N, H, d, dtype, n=3, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + N)
    return [torch.randn(B, N, H, d, generator=g, device="cuda").to(dtype) for _ in range(n)]


def rates(H):
    return -torch.linspace(0.01, 0.5, H, device="cuda")


@pytest.mark.parametrize("N,dtype", [(6, F32), (40, BF16), (700, F32), (1300, BF16)])
def test_training_captured(N, dtype):
    """Forward and backward in graphs give an eager call's bits, with an eager graph
    of other leaves alive."""
    from tarmac_b200 import autograd as ag
    rate, w = rates(2), torch.randn(32, device="cuda")

    def fn(q, k, v, S, w):
        out, last = ag.decay_attention(q, k, v, rate, S, return_state=True)
        y = out.flatten(2)
        return (*ag.residual_norm(y, y, w), last)

    def leaves(seed):
        S = torch.randn(2, 2, 16, 16, device="cuda")
        return [x.requires_grad_() for x in (*rows(2, N, 2, 16, dtype, seed=seed), S, w.clone())]

    gc.collect()  # graphs of earlier tests, whose release would end a capture
    graphed = torch.cuda.make_graphed_callables(fn, tuple(leaves(1)))
    for seed in (2, 3):
        a = leaves(seed)
        b = [x.detach().clone().requires_grad_() for x in a]
        want = fn(*b)
        got = graphed(*a)
        go = [torch.randn_like(x) for x in want]
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        for x, y in zip(torch.autograd.grad(got, a, go), torch.autograd.grad(want, b, go)):
            assert torch.equal(x, y)
    torch.cuda.synchronize()
    del graphed, got
    gc.collect()


@pytest.mark.parametrize("N", [1, 30])
def test_inference_mode(N):
    """States made in inference mode and outside of it, renewed in it."""
    from tarmac_b200 import ops
    from tarmac_b200.heads import DecayComm, rotation_table
    q, k, v = rows(2, N, 2, 16, F32)
    S = torch.randn(2, 2, 16, 16, device="cuda")
    want = ops.decay_attention(q, k, v, rates(2), S, return_state=True)
    with torch.inference_mode():
        for state in (S, S.clone()):
            own = state.clone()
            out, last = ops.decay_attention(q, k, v, rates(2), own, state_out=own)
            assert torch.equal(out, want[0]) and torch.equal(last, want[1])
        m = DecayComm(8, 2, 16).cuda()
        x = torch.randn(2, N, 8, device="cuda")
        cos, sin = rotation_table(torch.arange(N, device="cuda")[None], 16)
        state = m.empty_state(2)
        h, z = m.step(x, x, cos, sin, state)
        whole = m(x, x, cos, sin)
        for a, b in zip((h, z, state), whole):
            assert (a - b).abs().max() <= 1e-4 * b.abs().max()


@pytest.mark.parametrize("N,B,H,d,dtype", [
    (1, 2 ** 22, 4, 1, F32), (9, 2 ** 21, 4, 2, F32), (24, 2 ** 17, 3, 16, BF16),
    (12, 40000, 1, 72, BF16)])
def test_many_heads(N, B, H, d, dtype):
    """Up to 2^24 heads in a call: every head has its own rows' results, first and
    last ones against the 64-bit form (bounds as in test_decay_gpu: fp32 1e-5 of the
    sums of absolute terms; bf16 2^-8 of those and of the value)."""
    from tarmac_b200 import ops
    t = rows(B, N, H, d, dtype, 4)
    rate = rates(H)
    S = torch.randn(B, H, d, d, device="cuda")
    got = ops.decay_attention(*t[:3], rate, S, return_state=True)
    got = (*got, *ops.decay_attention_backward(*t[:3], rate, t[3], S, S))
    some = [0, 1, B // 2, B - 1]
    q, k, v, dout = (x[some].double().cpu() for x in t)
    s = S[some].double().cpu()
    args = (rate.cpu(), d ** -0.5)
    want = d64.decay_grads(q, k, v, *args, dout, s, None, s)
    mags = d64.decay_grads(q.abs(), k.abs(), v.abs(), *args, dout.abs(), s.abs(), None, s.abs())
    for i, (a, b, m) in enumerate(zip(got, want, mags)):
        state = i in (1, 5)
        tol = 1e-5 * m
        if dtype is BF16 and not state:
            tol = tol + 2 ** -8 * (m + b.abs())
        assert ((a[some].double().cpu() - b).abs() <= tol + 1e-30).all(), i


@pytest.mark.parametrize("N,dtype", [(3, F32), (100, BF16)])
def test_other_layouts_and_types(N, dtype):
    """A state that is a view, lengths of 64 bits, weights of the norms in bf16."""
    from tarmac_b200 import autograd as ag, ops
    q, k, v = rows(3, N, 2, 32, dtype)
    S = torch.randn(3, 2, 32, 32, device="cuda")
    lens = torch.tensor([N, 1, 2 ** 40], device="cuda")
    want = ops.decay_attention(q, k, v, rates(2), S, lens.clamp(max=N).int(), return_state=True)
    for state in (S.transpose(2, 3).contiguous().transpose(2, 3),
                  S.expand(2, -1, -1, -1, -1)[0], torch.stack([S, S], -1)[..., 0]):
        got = ops.decay_attention(q, k, v, rates(2), state, lens, return_state=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(ValueError, match="contiguous"):
        ops.decay_attention(q, k, v, rates(2), S, state_out=S.transpose(2, 3))
    x, y = (torch.randn(4, 7, 24, device="cuda").to(dtype) for _ in range(2))
    w = (1 + 0.1 * torch.randn(24, device="cuda")).bfloat16().requires_grad_()
    a = ag.residual_norm(x, y, w, w, None, w)
    b = ops.residual_norm(x, y, *(w.detach().float(),) * 2, None, w.detach().float())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    sum(t.float().sum() for t in a).backward()
    assert w.grad.dtype is BF16 and w.grad.isfinite().all()


def test_one_tensor_in_every_place():
    """x attends to itself, and is a block's stream and output at once."""
    from tarmac_b200 import autograd as ag, ops
    x, = rows(2, 50, 2, 32, F32, 1)
    x.requires_grad_()
    out = ag.decay_attention(x, x, x, rates(2))
    h, z = ag.residual_norm(x, x, None, None, x)
    g = torch.randn_like(x)
    dq, dk, dv, _ = ops.decay_attention_backward(x, x, x, rates(2), g)
    got, = torch.autograd.grad(out, x, g, retain_graph=True)
    assert (got - (dq + dk + dv)).abs().max() <= 1e-5 * got.abs().max()
    dx, dy, _, _, dgate, _ = ops.residual_norm_backward(x, x, None, None, x, None, g, g)
    got, = torch.autograd.grad((h, z), x, (g, g))
    assert (got - (dx + dy + dgate)).abs().max() <= 1e-5 * got.abs().max()


def test_streams_hand_on_their_results():
    """A call on one stream, its results read by a call on another after an event."""
    from tarmac_b200 import ops
    for N, d, dtype in ((1, 64, BF16), (300, 32, F32), (1300, 64, BF16)):
        q, k, v = rows(1, N, 2, d, dtype)
        S = torch.randn(1, 2, d, d, device="cuda")

        def twice(first, second):
            with torch.cuda.stream(first):
                out, last = ops.decay_attention(q, k, v, rates(2), S, return_state=True)
            second.wait_stream(first)
            with torch.cuda.stream(second):
                return [out, *ops.decay_attention(out, k, v, rates(2), last, return_state=True)]

        cur = torch.cuda.current_stream()
        want = twice(cur, cur)
        torch.cuda.synchronize()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        got = twice(a, b)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** 20])
@pytest.mark.parametrize("N,d,dtype", [(150, 64, BF16), (150, 72, BF16), (150, 32, F32), (60, 48, F32)])
def test_the_ends_of_the_scales(N, d, dtype, scale):
    """The largest and smallest scale of the gradients, with decays on both sides of
    2^-7 a row: the first state's gradient is the scale's alone, so that neither term
    hides the other (bounds as in test_many_heads)."""
    from tarmac_b200 import ops
    t = rows(2, N, 4, d, dtype, 4)
    rate = torch.tensor([-0.02, -4.84, -4.86, -7.0], device="cuda")
    S = torch.randn(2, 4, d, d, device="cuda")
    got = ops.decay_attention_backward(*t[:3], rate, t[3], S, S * scale, scale=scale)
    args = [x.double().cpu() for x in t]
    s = S.double().cpu()
    want = d64.decay_grads(*args[:3], rate.cpu(), scale, args[3], s, None, s * scale)[2:]
    mags = [x.abs() for x in args]
    mags = d64.decay_grads(*mags[:3], rate.cpu(), scale, mags[3], s.abs(), None, s.abs() * scale)[2:]
    for i, (a, b, m) in enumerate(zip(got, want, mags)):
        tol = 1e-5 * m
        if dtype is BF16 and i < 3:
            tol = tol + 2 ** -8 * (m + b.abs())
        assert ((a.double().cpu() - b).abs() <= tol).all(), i
