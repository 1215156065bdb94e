"""Which kernels calls of attention with a decay take, as the library reports it
(host-only)."""

from __future__ import annotations

import pytest
import torch

from tarmac_b200 import _lib, ops

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("args,dtype,kernel", [
    ((256, 1, 4, 4, 16), F32, "decay_step"),
    ((256, 8, 4, 4, 128), BF16, "decay_step"),
    ((256, 9, 4, 4, 16), F32, "decay_scan"),
    ((256, 23, 4, 4, 32), BF16, "decay_scan"),
    ((256, 24, 4, 4, 32), BF16, "decay_tc"),
    ((256, 15, 4, 4, 64), BF16, "decay_scan"),
    ((256, 16, 4, 4, 64), BF16, "decay_tc"),
    ((256, 24, 4, 4, 64), F32, "decay_scan"),
    ((256, 11, 4, 4, 72), BF16, "decay_scan"),
    ((256, 12, 4, 4, 72), BF16, "decay_tc"),
    ((256, 512, 4, 2, 16), BF16, "decay_tc"),
    ((256, 512, 4, 2, 8), BF16, "decay_scan"),
    ((256, 512, 4, 2, 20), BF16, "decay_scan"),  # 40-byte rows
])
def test_kernels(args, dtype, kernel):
    assert ops.decay_attention_plan(*args, dtype)["kernel"] == kernel


def test_gradients_of_few_rows_have_no_step():
    assert ops.decay_attention_plan(4, 3, 4, 4, 16, backward=True)["kernel"] == "decay_scan"


def test_few_heads_are_cut_in_segments():
    for dtype in (F32, BF16):
        plan = ops.decay_attention_plan(1, 8192, 4, 4, 64, dtype)
        assert plan["segments"] > 8 and plan["states"]
        plan = ops.decay_attention_plan(2048, 256, 4, 4, 64, dtype)
        assert plan["segments"] == 1 and not plan["states"]
    # the state after the last row comes from the segments' states
    assert ops.decay_attention_plan(2048, 256, 4, 4, 64, BF16, state=True)["states"]


def test_refuses_what_the_call_refuses():
    for args in ((2, 8, 3, 2, 16), (2, 8, 2, 2, 129), (-1, 8, 2, 2, 16)):
        with pytest.raises(_lib.TarmacError):
            ops.decay_attention_plan(*args)
