"""The multi-head cases of smoke() take the kernels that it names (host-only)."""

from __future__ import annotations

import torch

import __graft_entry__ as entry
from tarmac_b200 import ops


def test_smoke_reaches_both_kinds_of_kernels():
    took = {torch.float32: [], torch.bfloat16: []}
    for B, N, H, Hk, d in entry.HEAD_CASES:
        for dtype, kinds in took.items():
            kinds += [ops.head_attention_plan(B, N, N, H, Hk, d, dtype, "past", back)["kernel"]
                      for back in (False, True)]
    assert took[torch.bfloat16] == ["head_fwd", "head_bwd", "head_fwd_tc", "head_bwd_tc"]
    assert set(took[torch.float32]) == {"head_fwd", "head_bwd"}
