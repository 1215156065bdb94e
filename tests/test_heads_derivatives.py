"""Derivatives that the multi-head autograd functions do not have are refused,
not dropped. The kernels are replaced by torch forms: host logic, CPU only."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from tarmac_b200 import autograd as tgrad


@pytest.fixture(autouse=True)
def plain_kernels(monkeypatch):
    def attention(q, k, v, *how, return_lse=False):
        s = (q.transpose(1, 2) @ k.transpose(1, 2).transpose(-1, -2))
        out = (torch.softmax(s, -1) @ v.transpose(1, 2)).transpose(1, 2)
        return (out, torch.logsumexp(s, -1)) if return_lse else out

    def attention_grad(q, k, v, out, lse, dout, *how):
        with torch.enable_grad():
            t = [x.detach().requires_grad_() for x in (q, k, v)]
            return torch.autograd.grad(attention(*t), t, dout.detach())

    def rotate(q, k, *how):
        return tuple(x * torch.rsqrt(x.square().mean(-1, keepdim=True)) for x in (q, k))

    def rotate_grad(q, k, wq, wk, cos, sin, dq, dk, *how):
        with torch.enable_grad():
            t = [x.detach().requires_grad_() for x in (q, k)]
            return (*torch.autograd.grad(rotate(*t), t, (dq.detach(), dk.detach())), None, None)

    for name, f in (("head_attention", attention), ("head_attention_backward", attention_grad),
                    ("qk_norm_rotate", rotate), ("qk_norm_rotate_backward", rotate_grad)):
        monkeypatch.setattr(tgrad.ops, name, f)


def attend(x):
    return tgrad.head_attention(x, x, x)


def norm(x):
    return tgrad.qk_norm_rotate(x, x, None, None, torch.ones(1, 3, 0), torch.ones(1, 3, 0))[0]


@pytest.fixture
def x():
    return torch.randn(2, 3, 2, 4, generator=torch.Generator().manual_seed(0))


@pytest.mark.parametrize("f", [attend, norm])
def test_second_derivative_is_refused(f, x):
    x.requires_grad_()
    g, = torch.autograd.grad(f(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.square().sum().backward()


@pytest.mark.parametrize("f", [attend, norm])
def test_first_derivative_stays(f, x):
    x.requires_grad_()
    f(x).square().sum().backward()
    assert x.grad.shape == x.shape and x.grad.isfinite().all()


@pytest.mark.parametrize("f", [attend, norm])
def test_forward_mode_is_refused(f, x):
    with fwd.dual_level():
        with pytest.raises((NotImplementedError, RuntimeError)):
            f(fwd.make_dual(x, torch.ones_like(x)))
        assert f(x).shape == x.shape  # no tangent, nothing to refuse
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))
