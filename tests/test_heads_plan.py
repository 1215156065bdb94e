"""Which kernels multi-head attention calls take, as the library reports it
(host-only)."""

from __future__ import annotations

import pytest
import torch

from tarmac_b200 import _lib, ops

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("args,dtype,want", [
    ((256, 6, 6, 4, 4, 16), F32, {"kernel": "head_fwd", "parts": 1}),
    ((2, 200, 200, 4, 2, 64), F32, {"kernel": "head_fwd", "parts": 1}),
    ((200, 70, 70, 2, 1, 40), BF16, {"kernel": "head_fwd_tc", "items": 200}),
    ((200, 64, 64, 2, 1, 40), BF16, {"kernel": "head_fwd", "parts": 1}),
    ((90, 192, 192, 4, 2, 24), BF16, {"kernel": "head_fwd", "parts": 1}),
    ((90, 193, 193, 4, 2, 24), BF16, {"kernel": "head_fwd_tc", "items": 360}),
    ((90, 193, 193, 4, 2, 20), BF16, {"kernel": "head_fwd", "parts": 1}),  # 40-byte rows
    ((160, 70, 70, 3, 1, 64), BF16, {"kernel": "head_fwd_tc", "items": 320}),
])
def test_forward(args, dtype, want):
    assert ops.head_attention_plan(*args, dtype) == want


def test_few_rows_split_the_keys():
    for dtype in (F32, BF16):
        plan = ops.head_attention_plan(1, 1, 4096, 4, 2, 64, dtype)
        assert plan["kernel"] == "head_fwd" and plan["parts"] == 16


@pytest.mark.parametrize("args,dtype,want", [
    ((200, 70, 70, 2, 1, 40), BF16, ("head_bwd_tc", 400, 200)),
    ((200, 70, 70, 2, 1, 40), F32, ("head_bwd", 600, 400)),
    ((4, 32, 300, 2, 2, 64), BF16, ("head_bwd", 8, 40)),
    ((4, 33, 300, 2, 2, 64), BF16, ("head_bwd_tc", 8, 24)),
    ((4, 192, 192, 2, 2, 32), BF16, ("head_bwd", 24, 24)),
    ((4, 193, 193, 2, 2, 32), BF16, ("head_bwd_tc", 16, 16)),
])
def test_backward(args, dtype, want):
    plan = ops.head_attention_plan(*args, dtype, "past", backward=True)
    assert (plan["kernel"], plan["dq_items"], plan["dkv_items"]) == want


def test_refuses_what_the_call_refuses():
    with pytest.raises(_lib.TarmacError):
        ops.head_attention_plan(2, 8, 8, 3, 2, 16)
    with pytest.raises(_lib.TarmacError):
        ops.head_attention_plan(2, 8, 8, 2, 2, 129)
