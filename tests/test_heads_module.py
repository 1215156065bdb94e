"""Host side of the multi-head block: tables, shapes and refusals (CPU)."""

from __future__ import annotations

import math

import pytest
import torch

from tarmac_b200 import ops
from tarmac_b200.heads import HeadComm, rotation_table


def test_rotation_table_of_steps():
    cos, sin = rotation_table(torch.arange(5)[None], 8, base=100.0)
    assert cos.shape == sin.shape == (1, 5, 4) and cos.dtype == torch.float32
    for n in range(5):
        for i in range(4):
            a = n * 100.0 ** (-i / 4)
            assert abs(cos[0, n, i] - math.cos(a)) < 1e-6
            assert abs(sin[0, n, i] - math.sin(a)) < 1e-6


def test_rotation_table_of_places():
    pos = torch.tensor([[[1.0, -2.0], [0.5, 3.0]]])
    cos, _ = rotation_table(pos, 8)
    assert cos.shape == (1, 2, 4)
    assert torch.allclose(cos[..., 0], pos[..., 0].cos())
    assert torch.allclose(cos[..., 2], pos[..., 1].cos())


@pytest.mark.parametrize("pos,r", [(torch.zeros(2, 3), 3), (torch.zeros(2, 3, 2), 6),
                                   (torch.zeros(3), 4), (torch.zeros(2, 3), -2)])
def test_rotation_table_refuses(pos, r):
    with pytest.raises(ValueError):
        rotation_table(pos, r)


def test_block_shapes_and_refusals():
    with pytest.raises(ValueError):
        HeadComm(8, 6, 16, 4)
    m = HeadComm(8, 6, 16, 2)
    assert m.qkv.weight.shape == (10 * 16, 8) and m.proj.weight.shape == (96, 96)
    cos, sin = rotation_table(torch.arange(3)[None], 16)
    with pytest.raises(RuntimeError):  # there is no CPU implementation
        m(torch.zeros(1, 3, 8), cos, sin)
    with pytest.raises(RuntimeError):
        ops.pack_visibility(torch.ones(1, 2, 2, dtype=torch.bool))
