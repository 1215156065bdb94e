"""Key lengths and first positions held in 64 bits, beyond what 32 bits hold:
lengths act like Nk (or 0), positions like ones past either end of the keys."""

from __future__ import annotations

import pytest
import torch

from test_heads_gpu import BF16, F32, rows

pytestmark = pytest.mark.gpu
BIG = [2 ** 31, 2 ** 32, 2 ** 32 + 3, 2 ** 40 + 1, 2 ** 63 - 1]


@pytest.fixture(scope="module")
def ops():
    from tarmac_b200 import ops
    return ops


def both(ops, q, k, v, dout, **how):
    out, lse = ops.head_attention(q, k, v, return_lse=True, **how)
    return [out, lse, *ops.head_attention_backward(q, k, v, out, lse, dout, **how)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,d", [(20, 16), (130, 64)])
def test_lengths_and_starts_of_64_bits(ops, N, d, dtype):
    g = torch.Generator().manual_seed(N)
    B = len(BIG)
    q, k, v = rows(g, B, N, (2, 1, 1), d, dtype)
    dout, = rows(g, B, N, (2,), d, dtype)
    big = torch.tensor(BIG, device="cuda")
    all_ = both(ops, q, k, v, dout)
    for a, b in zip(both(ops, q, k, v, dout, key_len=big), all_):
        assert torch.equal(a, b)
    for x in both(ops, q, k, v, dout, key_len=-big)[:1]:
        assert (x == 0).all()
    # from a position past all keys everything is past, and nothing is itself
    for peers in ("past", "others"):
        for a, b in zip(both(ops, q, k, v, dout, peers=peers, q_start=big), all_):
            assert torch.equal(a, b)
    for x in both(ops, q, k, v, dout, peers="past", q_start=-big)[:1]:
        assert (x == 0).all()
