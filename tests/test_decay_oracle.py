"""The 64-bit forms that the GPU tests compare with: their gradients against
differences and against torch's autograd, and against closed forms."""

from __future__ import annotations

import pytest
import torch

import _decay64 as d64


def rnd(*shape):
    return torch.randn(*shape, dtype=torch.float64)


@pytest.mark.parametrize("Hk,lens", [(4, None), (2, [5, 3]), (1, [0, 5])])
def test_decay_gradients(Hk, lens):
    torch.manual_seed(Hk)
    B, N, H, d = 2, 5, 4, 3
    q, k, v = rnd(B, N, H, d), rnd(B, N, Hk, d), rnd(B, N, Hk, d)
    S, g, dS = rnd(B, H, d, d), rnd(B, N, H, d), rnd(B, H, d, d)
    rate = -torch.rand(H)
    lens = None if lens is None else torch.tensor(lens)
    leaves = [t.requires_grad_(True) for t in (q, k, v, S)]

    def f(q, k, v, S):
        return d64.decay(q, k, v, rate, 0.7, S, lens)

    assert torch.autograd.gradcheck(f, leaves)
    want = torch.autograd.grad(f(*leaves), leaves, (g, dS))
    with torch.no_grad():
        out, last = f(*leaves)
        got = d64.decay_grads(q, k, v, rate, 0.7, g, S, lens, dS)
    for a, b in zip(got, (out, last, *want)):
        assert (a - b).abs().max() <= 1e-12


def test_decay_is_masked_attention():
    """Without a state: weights l^(i-j) of the scores of a row's past."""
    torch.manual_seed(0)
    B, N, H, d = 2, 7, 3, 4
    q, k, v = rnd(B, N, H, d), rnd(B, N, H, d), rnd(B, N, H, d)
    rate = torch.tensor([0.0, -0.3, float("-inf")])
    i = torch.arange(N)
    gap = i[:, None] - i
    w = torch.exp(rate.double()[:, None, None] * gap.clamp_min(0))
    w = torch.where(gap > 0, w, (gap == 0).double())
    s = torch.einsum("bihd,bjhd->bhij", q, k) * w
    out, _ = d64.decay(q, k, v, rate, 0.5)
    assert (out - 0.5 * torch.einsum("bhij,bjhd->bihd", s, v)).abs().max() <= 1e-12


@pytest.mark.parametrize("gated", [False, True])
def test_norm_gradients(gated):
    torch.manual_seed(1)
    x, y, dh, dz = rnd(2, 3, 5), rnd(2, 3, 5), rnd(2, 3, 5), rnd(2, 3, 5)
    ws = [1 + 0.3 * rnd(5) for _ in range(3)]
    gate = rnd(2, 3, 5) if gated else None
    leaves = [t.requires_grad_(True) for t in (x, y, *ws, *([gate] if gated else []))]

    def f(x, y, wo, wi, sc, gate=None):
        return d64.norm(x, y, wo, wi, gate, sc, 1e-6)

    assert torch.autograd.gradcheck(f, leaves)
    want = torch.autograd.grad(f(*leaves), leaves, (dh, dz))
    with torch.no_grad():
        dx, dy, dwo, dwi, dg, dsc = d64.norm_grads(x, y, ws[0], ws[1], gate, ws[2], dh, dz, 1e-6)
    got = (dx, dy, dwo, dwi, dsc, *([dg] if gated else []))
    for a, b in zip(got, want):
        assert (a - b).abs().max() <= 1e-12
