"""What the autograd form of attention with a decay asks of the operators: states
and their gradients only where the caller wants them. The kernels are replaced
by the 64-bit forms: host logic, CPU only."""

from __future__ import annotations

import pytest
import torch

import _decay64 as d64
from tarmac_b200 import autograd as tgrad

RATE = torch.tensor([-0.1, -0.5])


@pytest.fixture(autouse=True)
def asked(monkeypatch):
    """The calls, as (returns a state) and (gradient of the first state)."""
    calls = []

    def attention(q, k, v, rate, state=None, lens=None, scale=None, return_state=False):
        calls.append(return_state)
        res = d64.decay(q, k, v, rate, 0.5, state, lens)
        return res if return_state else res[0]

    def gradients(q, k, v, rate, dout, state=None, dstate=None, lens=None, scale=None,
                  need_dstate=True):
        calls.append(need_dstate)
        g = d64.decay_grads(q, k, v, rate, 0.5, dout, state, lens, dstate)[2:]
        return (*g[:3], g[3] if need_dstate and state is not None else None)

    monkeypatch.setattr(tgrad.ops, "decay_attention", attention)
    monkeypatch.setattr(tgrad.ops, "decay_attention_backward", gradients)
    return calls


def rows(grad=True):
    g = torch.Generator().manual_seed(0)
    t = [torch.randn(2, 5, 2, 3, generator=g, dtype=torch.float64) for _ in range(3)]
    S = torch.randn(2, 2, 3, 3, generator=g, dtype=torch.float64)
    return [x.requires_grad_(grad) for x in t], S


@pytest.mark.parametrize("want", [False, True])
def test_a_state_is_formed_where_it_is_returned(asked, want):
    t, S = rows()
    res = tgrad.decay_attention(*t, RATE, S, return_state=want)
    assert asked == [want] and isinstance(res, tuple) == want


@pytest.mark.parametrize("need", [False, True])
def test_the_first_states_gradient_where_it_is_needed(asked, need):
    t, S = rows()
    S.requires_grad_(need)
    out, last = tgrad.decay_attention(*t, RATE, S, return_state=True)
    (out.sum() + last.sum()).backward()
    assert asked == [True, need] and (S.grad is not None) == need
    assert all(x.grad is not None for x in t)


@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("returned", [False, True])
def test_gradients_against_differences(returned, state):
    t, S = rows()
    args = (*t, *([S.requires_grad_()] if state else []))

    def f(q, k, v, S=None):
        return tgrad.decay_attention(q, k, v, RATE, S, torch.tensor([5, 3]),
                                     return_state=returned)

    assert torch.autograd.gradcheck(f, args)


def test_only_the_state_takes_part():
    t, S = rows()
    out, last = tgrad.decay_attention(*t, RATE, S, return_state=True)
    last.sum().backward()
    assert (t[0].grad == 0).all() and t[1].grad.abs().max() > 0
