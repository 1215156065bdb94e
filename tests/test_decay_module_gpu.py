"""The block with a memory of fixed size on the GPU: refusals of the launchers,
a training step against a 64-bit module, stepping against reading at once."""

from __future__ import annotations

import copy

import pytest
import torch

import _decay64 as d64
import _heads64 as h64

pytestmark = pytest.mark.gpu


def bad(**kw):
    from tarmac_b200 import ops
    dev = "cuda"
    a = dict(q=torch.zeros(2, 3, 4, 16, device=dev), k=torch.zeros(2, 3, 2, 16, device=dev),
             log_decay=torch.zeros(4, device=dev))
    a["v"] = a["k"]
    a.update(kw)
    return ops.decay_attention(**a)


def test_refusals():
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    for kw in (dict(k=z(2, 3, 3, 16), v=z(2, 3, 3, 16)), dict(k=z(2, 4, 2, 16), v=z(2, 4, 2, 16)),
               dict(v=z(2, 3, 2, 8)), dict(q=z(2, 3, 64)), dict(log_decay=z(3)),
               dict(log_decay=torch.zeros(4)), dict(state=z(2, 4, 16, 8)),
               dict(state=torch.zeros(2, 4, 16, 16)), dict(lens=z(3, dtype=torch.int32)),
               dict(lens=torch.zeros(2, dtype=torch.int32)),
               dict(state_out=z(2, 4, 16, 32)[..., ::2])):
        with pytest.raises(ValueError):
            bad(**kw)
    for kw in (dict(k=z(2, 3, 2, 16).bfloat16()), dict(log_decay=z(4).double()),
               dict(state=z(2, 4, 16, 16).bfloat16()), dict(lens=z(2)),
               dict(q=z(2, 3, 4, 16).half(), k=z(2, 3, 2, 16).half(), v=z(2, 3, 2, 16).half())):
        with pytest.raises(TypeError):
            bad(**kw)
    room = z(3, 4, 16, 16)
    with pytest.raises(ValueError, match="apart"):
        bad(state=room[:2], state_out=room[1:])
    from tarmac_b200 import TarmacError, ops
    with pytest.raises(TarmacError):
        bad(q=z(2, 3, 4, 130), k=z(2, 3, 2, 130), v=z(2, 3, 2, 130))
    x = z(2, 3, 8)
    for args in ((x, z(2, 3, 9)), (x, x, z(9)), (x, x, None, z(2, 8)), (x, x, None, None, z(3, 8)),
                 (x, x, torch.zeros(8)), (x, x.cpu())):
        with pytest.raises(ValueError):
            ops.residual_norm(*args)
    with pytest.raises(TypeError):
        ops.residual_norm(x, x.bfloat16())
    with pytest.raises(TarmacError):
        ops.residual_norm(z(1, 8193), z(1, 8193))


def plain(m, x, z, cos, sin, state, lens):
    """DecayComm.forward in the type of its parameters, row by row."""
    d = m.head_dim
    parts = m.qkv(z).split([h * d for h in m.heads], -1)
    q, k, v = (t.unflatten(-1, (h, d)) for t, h in zip(parts, m.heads))
    q = h64.rotate(q, m.norm_q, cos, sin, m.eps, False)
    k = h64.rotate(k, m.norm_k, cos, sin, m.eps, False)
    out, state = d64.decay(q, k, v, m.log_decay, d ** -0.5, state, lens)
    return (*d64.norm(x, m.proj(out.flatten(2)), m.norm_post, m.norm_next, m.gate(z), m.scale,
                      m.eps), state)


@pytest.mark.parametrize("N,H,Hk,d", [(6, 4, 4, 16), (70, 4, 2, 24), (150, 2, 1, 64)])
def test_training_step(N, H, Hk, d):
    """Two blocks in a stack, fp32 against 64 bits: outputs, gradients of the
    parameters and of the first state within 5e-4 of the largest of each tensor
    (six library products of up to 450 terms, 2^-24 each, each followed by a
    norm, around operators that hold 1e-5)."""
    from tarmac_b200.heads import DecayComm, rotation_table
    torch.manual_seed(N)
    dim = 20
    m = torch.nn.ModuleList([DecayComm(dim, H, d, Hk) for _ in range(2)])
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.1 * torch.randn_like(p))
    ref = copy.deepcopy(m).double()
    x, t = torch.randn(3, N, dim), torch.randn(2, 3, N, dim)
    S, tS = torch.randn(3, H, d, d), torch.randn(3, H, d, d)
    cos, sin = rotation_table(torch.arange(N)[None], d)
    lens = torch.tensor([N, N - 1, N // 2])

    def run(blocks, f, cast):
        s0 = cast(S).requires_grad_(True)
        h = z = cast(x)
        state = s0
        for b in blocks:
            h, z, state = f(b, h, z, cast(cos), cast(sin), s0, lens.to(h.device))
        loss = (h * cast(t[0])).sum() + (z * cast(t[1])).sum() + (state * cast(tS)).sum()
        loss.backward()
        return [h, z, state, s0.grad, *(p.grad for p in blocks.parameters())]

    want = run(ref, plain, lambda a: a.double())
    got = run(m.cuda(), lambda b, *a: b(*a), lambda a: a.cuda())
    for a, b in zip(got, want):
        assert (a.double().cpu() - b).abs().max() <= 5e-4 * b.abs().max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_equal_one_pass(dtype):
    """Row by row over a kept state, and all rows at once. fp32 within 1e-4 of
    the largest; bf16 rows, rounded at a dozen places by 2^-8 each, 2^-3."""
    from tarmac_b200.heads import DecayComm, rotation_table
    torch.manual_seed(3)
    B, T, dim = 4, 40, 32
    m = DecayComm(dim, 4, 32, 2).cuda().to(dtype)
    m.log_decay = m.log_decay.float()
    x = torch.randn(B, T, dim, device="cuda", dtype=dtype)
    cos, sin = rotation_table(torch.arange(T, device="cuda")[None], 32)
    with torch.no_grad():
        want = m(x, x, cos, sin)
    S = m.empty_state(B)
    tol = 1e-4 if dtype is torch.float32 else 2 ** -3
    for t in range(T):
        row = x[:, t:t + 1]
        h, z = m.step(row, row, cos[:, t:t + 1], sin[:, t:t + 1], S)
        for a, b in ((h, want[0]), (z, want[1])):
            assert (a[:, 0].float() - b[:, t].float()).abs().max() <= tol * b.abs().max()
    assert (S - want[2]).abs().max() <= tol * want[2].abs().max()


def test_a_renewed_state_is_noticed():
    """A state that autograd saved and a later call renewed in place."""
    from tarmac_b200 import autograd, ops
    q, k, v = (torch.randn(2, 4, 2, 16, device="cuda", requires_grad=True) for _ in range(3))
    rate = torch.tensor([-0.1, -0.5], device="cuda")
    S = torch.randn(2, 2, 16, 16, device="cuda")
    out = autograd.decay_attention(q, k, v, rate, S)
    with torch.no_grad():
        ops.decay_attention(q, k, v, rate, S, state_out=S)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


def test_unused_outputs():
    """Only one of the outputs takes part in the loss."""
    from tarmac_b200 import autograd
    q, k, v = (torch.randn(2, 70, 2, 16, device="cuda", requires_grad=True) for _ in range(3))
    rate = torch.tensor([-0.1, -0.5], device="cuda")
    out, S = autograd.decay_attention(q, k, v, rate, return_state=True)
    a = torch.autograd.grad(S.sum(), (q, k, v), retain_graph=True)
    assert (a[0] == 0).all()
    b = torch.autograd.grad(out.sum(), (q, k, v), retain_graph=True)
    c = torch.autograd.grad(out.sum() + S.sum(), (q, k, v))
    for x, y, z in zip(a, b, c):  # two fp32 sums in another order
        assert (x + y - z).abs().max() <= 1e-5 * z.abs().max()
    x, y = (torch.randn(5, 24, device="cuda", requires_grad=True) for _ in range(2))
    h, z = autograd.residual_norm(x, y)
    gh, gz = torch.autograd.grad(h.sum(), x, retain_graph=True)[0], torch.autograd.grad(z.sum(), x)[0]
    assert torch.equal(gh, torch.ones_like(gh)) and gz.abs().max() > 0


def test_other_derivatives_are_refused():
    from torch.autograd import forward_ad
    from tarmac_b200 import autograd
    q = torch.randn(1, 4, 2, 16, device="cuda", requires_grad=True)
    rate = torch.zeros(2, device="cuda")
    out = autograd.decay_attention(q, q, q, rate)
    g, = torch.autograd.grad(out.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), q)
    x = q.detach()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: autograd.decay_attention(dual, x, x, rate),
                     lambda: autograd.residual_norm(dual, x)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()


def test_a_cast_block_reads_its_norms_weights_as_they_are():
    """bf16 rows, fp32 norms: the block's outputs are the operators' on the weights
    before the cast, to the bit, and their gradients come in fp32."""
    from tarmac_b200 import ops
    from tarmac_b200.heads import DecayComm, rotation_table
    torch.manual_seed(5)
    B, N, dim, d = 2, 40, 32, 16
    m = DecayComm(dim, 2, d).cuda()
    own = ("norm_q", "norm_k", "norm_post", "norm_next", "scale")
    with torch.no_grad():
        for n in own:
            getattr(m, n).add_(0.1 * torch.randn_like(getattr(m, n)))
    wq, wk, wo, wi, sc = (getattr(m, n).detach().clone() for n in own)
    m.bfloat16()
    x = torch.randn(B, N, dim, device="cuda", dtype=torch.bfloat16)
    cos, sin = rotation_table(torch.arange(N, device="cuda")[None], d)
    with torch.no_grad():
        q, k, v = (t.unflatten(-1, (2, d)) for t in m.qkv(x).split(2 * d, -1))
        q, k = ops.qk_norm_rotate(q, k, wq, wk, cos, sin, m.eps)
        out = ops.decay_attention(q, k, v, m.log_decay)
        want = ops.residual_norm(x, m.proj(out.flatten(2)), wo, wi, m.gate(x), sc, m.eps)
    h, z, _ = m(x, x, cos, sin)
    assert torch.equal(h, want[0]) and torch.equal(z, want[1])
    (h.float().sum() + z.float().square().sum()).backward()
    for n in own:
        g = getattr(m, n).grad
        assert g.dtype is torch.float32 and g.isfinite().all() and g.abs().max() > 0
    assert m.qkv.weight.grad.dtype is torch.bfloat16
