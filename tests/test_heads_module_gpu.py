"""The multi-head block on the GPU: a training step against a 64-bit module,
stepping through a history against reading it at once, and both operators
replayed from a CUDA graph."""

from __future__ import annotations

import copy

import pytest
import torch

import _heads64 as h64

pytestmark = pytest.mark.gpu


def plain_block(m, x, cos, sin, mask):
    """HeadComm.forward in the type of its parameters, with dense matrices."""
    d, (H, Hk, _) = m.head_dim, m.heads
    parts = m.qkv(x).split([h * d for h in m.heads], -1)
    q, k, v = (t.unflatten(-1, (h, d)) for t, h in zip(parts, m.heads))
    q = h64.rotate(q, m.norm_q, cos, sin, m.eps, False)
    k = h64.rotate(k, m.norm_k, cos, sin, m.eps, False)
    kk, vv = (t.repeat_interleave(H // Hk, 2).transpose(1, 2) for t in (k, v))
    s = q.transpose(1, 2) @ kk.transpose(-1, -2) / d ** 0.5
    s = s.masked_fill(~mask[:, None], float("-inf"))
    blind = ~mask.any(-1)[:, None, :, None]
    p = torch.softmax(s.masked_fill(blind, 0.0), -1).masked_fill(blind, 0.0)
    return m.proj((p @ vv).transpose(1, 2).flatten(2))


@pytest.mark.parametrize("N,H,Hk,d,peers", [(6, 4, 4, 16, "others"), (70, 4, 2, 24, "past"),
                                            (150, 2, 1, 64, "others")])
def test_training_step(N, H, Hk, d, peers):
    """fp32 against 64 bits: outputs and parameter gradients within 2e-4 of the
    largest of each tensor (two library products of up to 450 terms, 2^-24
    each, around operators that hold 1e-5)."""
    from tarmac_b200.heads import HeadComm, rotation_table
    torch.manual_seed(N)
    m = HeadComm(20, H, d, Hk)
    with torch.no_grad():
        m.norm_q.add_(0.1 * torch.randn(d))
        m.norm_k.add_(0.1 * torch.randn(d))
    ref = copy.deepcopy(m).double()
    x, t = torch.randn(3, N, 20), torch.randn(3, N, H * d)
    pos = 10 * torch.rand(3, N, 2)
    cos, sin = rotation_table(pos, d // 4 * 4)
    seen = torch.rand(3, N, N) < 0.6
    seen[:, 2] = False
    lens = torch.tensor([N, N - 1, N // 2])
    mask = h64.mask(3, N, N, peers, lens, None, seen)
    want = plain_block(ref, x.double(), cos.double(), sin.double(), mask)
    (want * t.double()).sum().backward()
    m = m.cuda()
    got = m(x.cuda(), cos.cuda(), sin.cuda(), peers, seen.cuda(), lens.cuda())
    (got * t.cuda()).sum().backward()

    def near(a, b):
        assert (a.double().cpu() - b).abs().max() <= 2e-4 * b.abs().max()

    near(got.detach(), want.detach())
    for (name, a), b in zip(m.named_parameters(), ref.parameters()):
        near(a.grad, b.grad)


def test_steps_equal_one_pass():
    """Row by row over a history, and all rows at once under the past rule."""
    from tarmac_b200.heads import HeadComm, rotation_table
    torch.manual_seed(3)
    B, T, H, Hk, d = 4, 40, 4, 2, 32
    m = HeadComm(12, H, d, Hk).cuda()
    x = torch.randn(B, T, 12, device="cuda")
    cos, sin = rotation_table(torch.arange(T, device="cuda")[None], d)
    with torch.no_grad():
        want = m(x, cos, sin, "past")
    k, v = (torch.full((B, T + 3, Hk, d), float("nan"), device="cuda") for _ in range(2))
    n = torch.zeros(B, dtype=torch.int64, device="cuda")
    for t in range(T):
        got = m.step(x[:, t:t + 1], cos[:, t:t + 1], sin[:, t:t + 1], k, v, n)
        # two fp32 paths of one formula: library products of other shapes
        assert (got[:, 0] - want[:, t]).abs().max() <= 1e-4 * want.abs().max()
    assert (n == T).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_operators_in_a_graph(dtype):
    """A captured call replays to the same bits on new inputs."""
    from tarmac_b200 import ops
    torch.manual_seed(1)
    x = torch.randn(2, 200, 8 * 64, device="cuda").to(dtype)
    q, k, v = (t.unflatten(-1, (-1, 64)) for t in x.split([256, 128, 128], -1))
    a = torch.rand(1, 200, 32, device="cuda")
    cos, sin = a.cos(), a.sin()

    def run():
        qr, kr = ops.qk_norm_rotate(q, k, None, None, cos, sin)
        out, lse = ops.head_attention(qr, kr, v, "past", return_lse=True)
        grads = ops.head_attention_backward(qr, kr, v, out, lse, out, "past")
        back = ops.qk_norm_rotate_backward(q, k, None, None, cos, sin, *grads[:2])
        return [out, grads[2], *back[:2]]

    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = run()
    x.copy_(torch.randn_like(x))
    g.replay()
    for p, r in zip(held, run()):
        assert torch.equal(p, r)
