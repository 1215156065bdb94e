"""The 64-bit forms that the multi-head GPU tests compare with: their gradient
formulas agree with differences of their forward forms. CPU only."""

from __future__ import annotations

import pytest
import torch

import _heads64 as h64

H = 1e-5


def slopes(f, x, n=6, seed=0):
    """Directional derivatives of f at x along n random directions."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(n):
        u = torch.randn(x.shape, generator=g, dtype=torch.float64)
        out.append((u, (f(x + H * u) - f(x - H * u)) / (2 * H)))
    return out


def agree(grad, f, x):
    # central differences in 64 bits: truncation H^2, rounding 1e-16 / H
    for u, s in slopes(f, x):
        got = (grad * u).sum()
        assert abs(got - s) <= 1e-6 * (1.0 + (grad * u).abs().sum())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,half", [(8, 4), (10, 3), (6, 0)])
def test_rotate_formula(d, half, interleaved):
    g = torch.Generator().manual_seed(d)
    x = torch.randn(2, 3, 4, d, generator=g, dtype=torch.float64)
    w = torch.randn(d, generator=g, dtype=torch.float64)
    dy = torch.randn(x.shape, generator=g, dtype=torch.float64)
    a = torch.randn(2, 3, half, generator=g, dtype=torch.float64)
    args = (a.cos(), a.sin(), 1e-6, interleaved)
    dx, dw = h64.rotate_grad(x, w, *args, dy)
    agree(dx, lambda t: (h64.rotate(t, w, *args) * dy).sum(), x)
    agree(dw, lambda t: (h64.rotate(x, t, *args) * dy).sum(), w)


@pytest.mark.parametrize("peers", ["all", "others", "past"])
def test_attention_formula(peers):
    g = torch.Generator().manual_seed(3)
    B, Nq, Nk, H_, Hk, d = 2, 5, 7, 4, 2, 6
    q = torch.randn(B, Nq, H_, d, generator=g, dtype=torch.float64)
    k, v = (torch.randn(B, Nk, Hk, d, generator=g, dtype=torch.float64) for _ in range(2))
    dout = torch.randn(q.shape, generator=g, dtype=torch.float64)
    seen = torch.rand(B, Nq, Nk, generator=g) < 0.7
    seen[0, 1] = False
    m = h64.mask(B, Nq, Nk, peers, torch.tensor([7, 4]), torch.tensor([1, 2]), seen)
    ref = h64.Attention(q, k, v, m, 0.4, dout)
    assert (ref.out[0, 1] == 0).all() and torch.isinf(ref.lse[0, :, 1]).all()

    def loss(q_, k_, v_):
        return (h64.Attention(q_, k_, v_, m, 0.4).out * dout).sum()

    agree(ref.dq, lambda t: loss(t, k, v), q)
    agree(ref.dk, lambda t: loss(q, t, v), k)
    agree(ref.dv, lambda t: loss(q, k, t), v)
