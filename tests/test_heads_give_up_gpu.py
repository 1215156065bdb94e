"""The tensor-memory attention kernels when one of their roles gives up, as it
does when a bounded wait runs out: the launch ends, the device stays usable,
and what comes back is NaN or right.

Test builds of the two kernels (TARMAC_GIVE_UP_AT in csrc/head_tc.cuh) let a
role give up at its block's second item, on the host's word; nothing is made to
hang. A call of fewer items than the GPU has SMs never gets there: it gives the
right values, bit for bit, as each item is computed by itself."""

from __future__ import annotations

import ctypes
import math
import subprocess
from ctypes import c_float, c_int, c_void_p
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

TESTS = Path(__file__).resolve().parent
PKG = TESTS.parent / "topk-tarmac_b200"
LOADER, WEIGHTS = 0, 1
B, N, H, D = 330, 130, 1, 64  # two row tiles: 330 forward items, 660 of each gradient kernel
FEW = 70                      # episodes with at most one item a block
HELD = 7.0                    # what the outputs hold before the call


def build(folder, role):
    from tarmac_build import NVCC_FLAGS, nvcc
    lib = folder / f"head_tc_{role}.so"
    csrc = PKG / "csrc"
    cmd = [nvcc(), *NVCC_FLAGS, "-I", str(csrc), "-DTARMAC_GIVE_UP_AT=1",
           f"-DTARMAC_GIVE_UP_ROLE={role}", "-shared", "-cudart", "static",
           str(TESTS / "native" / "head_tc_entry.cu"), str(csrc / "head_attn_tc.cu"),
           str(csrc / "head_bwd_tc.cu"), "-o", str(lib)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    so = ctypes.CDLL(str(lib))
    so.forward.argtypes = [c_void_p] * 5 + [c_int] * 4 + [c_float, c_void_p]
    so.backward.argtypes = [c_void_p] * 8 + [c_int] * 4 + [c_float, c_void_p]
    return so


@pytest.fixture(scope="module")
def builds(tmp_path_factory):
    import importlib.util
    import sys
    spec = importlib.util.spec_from_file_location("tarmac_build", PKG / "build.py")
    mod = importlib.util.module_from_spec(spec)
    sys.modules["tarmac_build"] = mod
    spec.loader.exec_module(mod)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert 2 * FEW <= sms < B
    made = {}

    def get(role):
        if role not in made:
            made[role] = build(tmp_path_factory.mktemp("give_up"), role)
        return made[role]
    return get


@pytest.fixture(scope="module")
def case():
    g = torch.Generator().manual_seed(11)
    return [torch.randn(B, N, H, D, generator=g).bfloat16().cuda() for _ in range(4)]


def held(*shape, dtype=torch.bfloat16):
    return torch.full(shape, HELD, device="cuda", dtype=dtype)


def forward(so, q, k, v):
    b = q.shape[0]
    out, lse = held(b, N, H, D), held(b, H, N, dtype=torch.float32)
    assert so.forward(*(t.data_ptr() for t in (q, k, v, out, lse)), b, N, H, D, D ** -0.5,
                      torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    return out, lse


def backward(so, q, k, v, dout, out, lse):
    b, rows = q.shape[0], -(-N // 128) * 128
    delta = torch.zeros(2, b, H, rows, device="cuda")
    delta[0] = -math.inf
    delta[0, :, :, :N] = -lse / math.log(2.0)
    delta[1, :, :, :N] = -(dout.float() * out.float()).sum(-1).transpose(1, 2)
    grads = [held(b, N, H, D) for _ in range(3)]
    assert so.backward(*(t.data_ptr() for t in (q, k, v, dout, delta, *grads)), b, N, H, D,
                       D ** -0.5, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    return grads


def by_parts(f, *ts):
    """f on a few episodes at a time, where no block has a second item."""
    parts = [f(*(t[i:i + FEW] for t in ts)) for i in range(0, B, FEW)]
    return [torch.cat(x) for x in zip(*parts)]


def nan_or_right(got, want):
    assert want.isfinite().all()
    assert (got.isnan() | (got == want)).all()


def still_right(so, case):
    """The device answers as before."""
    from tarmac_b200 import ops
    q, k, v = (t[:FEW] for t in case[:3])
    out, lse = forward(so, q, k, v)
    want, wlse = ops.head_attention(q, k, v, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)


def test_forward_loader(builds, case):
    """The loading thread gives up: every row is written, NaN or right."""
    so = builds(LOADER)
    want = by_parts(lambda *t: forward(so, *t), *case[:3])
    for a, b in zip(forward(so, *case[:3]), want):
        nan_or_right(a, b)
        assert a.isnan().any()  # it did give up
    still_right(so, case)


def test_backward_loader(builds, case):
    """The loading thread gives up: the launches end, and no product or copy
    that was in flight disturbs what runs behind them."""
    so = builds(LOADER)
    q, k, v, dout = case
    out, lse = by_parts(lambda *t: forward(so, *t), q, k, v)
    args = (q, k, v, dout, out, lse)
    want = by_parts(lambda *t: backward(so, *t), *args)
    got = backward(so, *args)
    assert any((a != b).any() for a, b in zip(got, want))  # it did give up
    still_right(so, case)
    for a, b in zip(by_parts(lambda *t: backward(so, *t), *args), want):
        assert torch.equal(a, b)


def test_forward_half_of_a_row(builds, case):
    """The warps of one half of each row's columns give up: the other half, with
    whom they share the row's maximum and sum, is not left with finite values."""
    so = builds(WEIGHTS)
    want = by_parts(lambda *t: forward(so, *t), *case[:3])
    for a, b in zip(forward(so, *case[:3]), want):
        nan_or_right(a, b)
        assert a.isnan().any()
    still_right(so, case)


@pytest.mark.parametrize("role", [LOADER, WEIGHTS])
def test_backward_rows(builds, case, role):
    """Every row of the gradients is written, also those of the items that a
    block had not reached when it gave up."""
    so = builds(role)
    q, k, v, dout = case
    out, lse = by_parts(lambda *t: forward(so, *t), q, k, v)
    args = (q, k, v, dout, out, lse)
    want = by_parts(lambda *t: backward(so, *t), *args)
    for a, b in zip(backward(so, *args), want):
        nan_or_right(a, b)
        assert a.isnan().any()
    still_right(so, case)
