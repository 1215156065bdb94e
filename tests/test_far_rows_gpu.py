"""Operands whose episodes start beyond 2^31 elements of their tensor, and norms of wide
rows that a block takes many of: attention with a decay and the norms around a
block, in the kernels that form their addresses themselves and in those that
leave it to TMA."""

from __future__ import annotations

import pytest
import torch

import _decay64 as d64

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def far(tensors, dtype):
    """The tensors ([2, N, ..], each as wide) as views whose second episode starts
    beyond 2^31 elements."""
    size = tensors[0][0].numel()
    step = 2 ** 31 + len(tensors) * size
    big = torch.zeros(step + len(tensors) * size, device="cuda", dtype=dtype)
    views = []
    for i, t in enumerate(tensors):
        inner = t[0].contiguous().stride()
        view = big.as_strided(t.shape, (step, *inner), i * size)
        view.copy_(t)
        views.append(view)
    return views


@pytest.mark.parametrize("N,d,dtype,kernel", [
    (1, 64, F32, "decay_step"), (5, 40, BF16, "decay_step"), (20, 16, F32, "decay_scan"),
    (70, 48, F32, "decay_scan"), (70, 8, BF16, "decay_scan"), (150, 64, BF16, "decay_tc"),
    (150, 72, BF16, "decay_tc")])
def test_decay_attention(N, d, dtype, kernel):
    from tarmac_b200 import ops
    assert ops.decay_attention_plan(2, N, 1, 1, d, dtype, state=True)["kernel"] == kernel
    g = torch.Generator(device="cuda").manual_seed(N)
    t = [torch.randn(2, N, 1, d, generator=g, device="cuda").to(dtype) for _ in range(4)]
    S, dS = (torch.randn(2, 1, d, d, generator=g, device="cuda") for _ in range(2))
    rate = torch.tensor([-0.1], device="cuda")

    def run(q, k, v, dout):
        return [*ops.decay_attention(q, k, v, rate, S, return_state=True),
                *ops.decay_attention_backward(q, k, v, rate, dout, S, dS)]

    for a, b in zip(run(*far(t, dtype)), run(*t)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [200, 2048, 8192])
def test_residual_norm(D, dtype):
    from tarmac_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(D)
    t = [torch.randn(2, 9, D, generator=g, device="cuda").to(dtype) for _ in range(5)]
    w = [torch.randn(D, generator=g, device="cuda") for _ in range(3)]

    def run(x, y, gate, dh, dz):
        args = (x, y, w[0], w[1], gate, w[2])
        return [*ops.residual_norm(*args), *ops.residual_norm_backward(*args, dh, dz)]

    for a, b in zip(run(*far(t, dtype)), run(*t)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,gate,weights", [(4104, True, True), (8191, True, True),
                                            (8192, True, False), (8192, False, True)])
def test_wide_rows(D, gate, weights, dtype):
    """450 rows and more than one for every block. Tolerances as in
    test_residual_norm_gpu.check, whose forms and magnitudes these are: 1e-5 of the
    largest value (of a weight's gradient, of that and the number of rows), bf16
    2^-8 of the value for its rounding."""
    from tarmac_b200 import ops
    rows, eps = 450, 1e-6
    assert rows > torch.cuda.get_device_properties(0).multi_processor_count
    g = torch.Generator().manual_seed(D)
    x, y, s, dh, dz = (torch.randn(rows, D, generator=g).to(dtype) for _ in range(5))
    wo, wi, sc = (0.5 + 0.3 * torch.randn(D, generator=g) for _ in range(3))
    if not gate:
        s = None
    if not weights:
        wo = wi = sc = None
    gpu = [None if t is None else t.cuda() for t in (x, y, wo, wi, s, sc)]
    got = [*ops.residual_norm(*gpu, eps=eps),
           *ops.residual_norm_backward(*gpu, dh.cuda(), dz.cuda(), eps=eps)]
    plain = [None if t is None else t.double() for t in (x, y, wo, wi, s, sc)]
    want = [*d64.norm(*plain, eps), *d64.norm_grads(*plain, dh.double(), dz.double(), eps)]
    given = [True, True, True, True, weights, weights, gate, weights]
    for i, (a, b, there) in enumerate(zip(got, want, given)):
        assert (a is not None) == there
        if not there:
            continue
        weight = i in (4, 5, 7)
        b, err = b.abs(), (a.double().cpu() - b).abs()
        tol = 1e-5 * (b.max() + (rows if weight else 0.0))
        if dtype is BF16 and not weight:
            tol = tol + 2 ** -8 * b
        assert (err <= tol).all(), (i, (err - tol).max())
