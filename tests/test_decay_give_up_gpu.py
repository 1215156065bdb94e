"""The tensor-memory kernels of attention with a decay when one of their roles
gives up, as it does when a bounded wait runs out: the launch ends, the device
stays usable, and what comes back is NaN or right.

Test builds of the kernels (TARMAC_GIVE_UP_AT in csrc/head_tc.cuh) let a role
give up at its block's second unit, on the host's word; nothing is made to hang.
A call of fewer units than the GPU has SMs never gets there: it gives the right
values, bit for bit, as each unit is computed by itself."""

from __future__ import annotations

import ctypes
import subprocess
from ctypes import c_int, c_void_p
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

TESTS = Path(__file__).resolve().parent
PKG = TESTS.parent / "topk-tarmac_b200"
LOADER, WEIGHTS = 0, 1
B, N, FEW = 330, 200, 140  # episodes of one unit each; with at most one a block
HELD = 7.0                 # what the outputs hold before the call


@pytest.fixture(scope="module")
def builds(tmp_path_factory):
    import importlib.util
    spec = importlib.util.spec_from_file_location("tarmac_build", PKG / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert FEW <= torch.cuda.get_device_properties(0).multi_processor_count < B
    folder, csrc = tmp_path_factory.mktemp("give_up"), PKG / "csrc"
    procs = {}
    for role in (LOADER, WEIGHTS):
        lib = folder / f"decay_tc_{role}.so"
        cmd = [mod.nvcc(), *mod.NVCC_FLAGS, "-I", str(csrc), "-DTARMAC_GIVE_UP_AT=1",
               f"-DTARMAC_GIVE_UP_ROLE={role}", "-shared", "-cudart", "static",
               str(TESTS / "native" / "decay_tc_entry.cu"), str(csrc / "decay_tc.cu"),
               str(csrc / "head_attn_tc.cu"), "-o", str(lib)]
        procs[role] = lib, subprocess.Popen(cmd, stderr=subprocess.PIPE, text=True)
    made = {}
    for role, (lib, p) in procs.items():
        err = p.communicate()[1]
        assert p.returncode == 0, err
        made[role] = ctypes.CDLL(str(lib))
        made[role].rows.argtypes = [c_void_p] * 5 + [c_int] * 4 + [c_void_p]
        made[role].states.argtypes = [c_void_p] * 4 + [c_int] * 4 + [c_void_p]
    return made


def inputs(H, d):
    g = torch.Generator().manual_seed(d)
    q, k, v = (torch.randn(B, N, H, d, generator=g).bfloat16().cuda() for _ in range(3))
    return q, k, v, torch.linspace(-0.5, -0.01, H).cuda()


def rows(so, q, k, v, rate):
    out = torch.full_like(q, HELD)
    b, _, H, d = q.shape
    assert so.rows(*(t.data_ptr() for t in (q, k, v, rate, out)), b, N, H, d,
                   torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    return out


def states(so, k, v, rate):
    b, _, H, d = k.shape
    part = torch.full((b, H, d, d), HELD, device="cuda")
    assert so.states(*(t.data_ptr() for t in (k, v, rate, part)), b, N, H, d,
                     torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    return part


def by_parts(f, *ts):
    """f on few episodes at a time, where no block has a second unit."""
    return torch.cat([f(*(t[i:i + FEW] for t in ts)) for i in range(0, B, FEW)])


@pytest.mark.parametrize("role", [LOADER, WEIGHTS])
@pytest.mark.parametrize("H,d", [(2, 64), (1, 128)])
def test_rows(builds, H, d, role):
    so = builds[role]
    q, k, v, rate = inputs(H, d)
    want = by_parts(lambda *t: rows(so, *t, rate), q, k, v)
    got = rows(so, q, k, v, rate)
    assert want.isfinite().all()
    assert (got.isnan() | (got == want)).all()
    assert got.isnan().any()  # it did give up
    again = by_parts(lambda *t: rows(so, *t, rate), q, k, v)
    assert torch.equal(again, want)  # the device answers as before


@pytest.mark.parametrize("H,d", [(2, 64), (1, 128)])
def test_states(builds, H, d):
    so = builds[LOADER]
    _, k, v, rate = inputs(H, d)
    want = by_parts(lambda *t: states(so, *t, rate), k, v)
    got = states(so, k, v, rate)
    assert want.isfinite().all()
    assert (got.isnan() | (got == want)).all()
    assert got.isnan().any()
    assert torch.equal(by_parts(lambda *t: states(so, *t, rate), k, v), want)
