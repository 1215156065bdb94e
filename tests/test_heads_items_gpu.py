"""Multi-head attention calls in which a block of the persistent tensor-memory
kernels takes several units of work: the walk over them in alternating
direction and what a block carries from one to the next (barrier phases, ring
slots, the copies of S), with empty units between full ones. Each case asserts
the kernel that it is for, so that a change of the dispatch rules cannot empty
it. Tolerances are those of test_heads_gpu.py.

Also strides with the head axis outside the row axis."""

from __future__ import annotations

import random

import pytest
import torch

from test_heads_gpu import BF16, F32, attention_case, rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tarmac_b200 import ops
    return ops


CASES = [  # B, Nq, Nk, H, Hk, d, peers, share seen
    (310, 70, 70, 1, 1, 64, "others", None),    # one tile a unit, the second missing
    (211, 70, 70, 2, 1, 40, "past", 0.5),       # two heads of the same rows
    (161, 70, 70, 3, 1, 64, "all", 0.7),        # a missing tile in every other unit
    (163, 70, 650, 1, 1, 64, "past", None),     # six key tiles: the ring wraps
    (31, 300, 300, 4, 2, 128, "others", None),
    (83, 130, 260, 2, 2, 96, "past", None),
    (83, 200, 200, 4, 2, 24, "others", 0.6),
    (35, 300, 300, 4, 4, 64, "past", None),     # few heads: tiles in the outer order
]


@pytest.mark.parametrize("B,Nq,Nk,H,Hk,d,peers,seen", CASES)
def test_several_units_a_block(ops, B, Nq, Nk, H, Hk, d, peers, seen):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    fwd = ops.head_attention_plan(B, Nq, Nk, H, Hk, d, BF16, peers)
    bwd = ops.head_attention_plan(B, Nq, Nk, H, Hk, d, BF16, peers, backward=True)
    assert fwd["kernel"] == "head_fwd_tc" and bwd["kernel"] == "head_bwd_tc"
    for items in (fwd["items"], bwd["dq_items"], bwd["dkv_items"]):
        assert items > sms and items % sms
    rng = random.Random(B)
    lens = [rng.choice([0, 0, 1, Nk, Nk + 9, rng.randrange(Nk), rng.randrange(Nk)])
            for _ in range(B)]
    starts = [rng.choice([Nk - Nq, 0, -5, n - Nq, Nk // 2]) for n in lens]
    attention_case(ops, B, Nq, Nk, H, Hk, d, BF16, peers, lens=lens, starts=starts, seen=seen,
                   spoil=True)


@pytest.mark.parametrize("B,N,H,d,peers", [(170, 130, 2, 64, "past"), (90, 200, 3, 128, "all")])
def test_full_units(ops, B, N, H, d, peers):
    """Equal lengths, no empty unit."""
    attention_case(ops, B, N, N, H, H, d, BF16, peers)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,Nq,Nk,H,Hk,d,peers", [
    (3, 150, 150, 4, 2, 64, "past"), (2, 20, 20, 4, 4, 16, "others"),
    (2, 1, 1500, 8, 2, 128, "all"), (2, 40, 210, 2, 2, 80, "past"),
    (2, 201, 201, 6, 3, 32, "others")])
def test_heads_outside_rows(ops, B, Nq, Nk, H, Hk, d, peers, dtype):
    """[B, heads, N, d] memory seen as [B, N, heads, d]: the same bits as rows
    with their heads inside."""
    g = torch.Generator().manual_seed(d)
    near = [rows(g, B, n, (h,), d, dtype)[0] for n, h in
            ((Nq, H), (Nk, Hk), (Nk, Hk), (Nq, H))]
    far = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in near]
    assert far[0].stride(2) == Nq * d
    lens = torch.tensor([Nk, Nk // 2, 1][:B], dtype=torch.int32).cuda()
    res = []
    for q, k, v, dout in (near, far):
        out, lse = ops.head_attention(q, k, v, peers, lens, return_lse=True)
        if q is far[0]:
            out_in = out.transpose(1, 2).contiguous().transpose(1, 2)
        else:
            out_in = out
        res.append([out, lse, *ops.head_attention_backward(q, k, v, out_in, lse, dout, peers,
                                                           lens)])
    for a, b in zip(*res):
        assert torch.equal(a, b)
    cos, sin = torch.rand(2, 1, Nq, d // 4, generator=g).cuda()
    if Nq == Nk:
        for a, b in zip(ops.qk_norm_rotate(near[0], near[1], None, None, cos, sin),
                        ops.qk_norm_rotate(far[0], far[1], None, None, cos, sin)):
            assert torch.equal(a, b)
