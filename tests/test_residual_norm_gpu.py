"""The norms around a block on the GPU against the 64-bit form."""

from __future__ import annotations

import pytest
import torch

import _decay64 as d64

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
EPS = 1e-6
WEIGHTS = ("w_post", "w_pre", "scale")


def inputs(shape, dtype, gate=True, weights=WEIGHTS, seed=0):
    g = torch.Generator().manual_seed(seed + shape[-1])
    t = {n: torch.randn(*shape, generator=g).to(dtype) for n in ("x", "y", "gate", "dh", "dz")}
    if not gate:
        t["gate"] = None
    for n in WEIGHTS:
        w = 0.5 + 0.3 * torch.randn(shape[-1], generator=g)
        t[n] = w if n in weights else None
    return t


def dy_term(f, dh, dz):
    """max |ry c|, the larger term of dy: |c| <= |w_post e scale|."""
    ry = 1.0 / (f["y"].square().mean(-1, keepdim=True) + EPS).sqrt()
    plain = (f["x"], f["y"], f["w_post"], f["w_pre"], f["gate"], f["scale"])
    c = d64.norm_grads(*plain, dh, dz, EPS)[0]
    for w in ("w_post", "scale"):
        c = c if f[w] is None else c * f[w]
    return (ry * c).abs().max()


def check(t, dtype, wrap=lambda x: x):
    """fp32: a few dozen operations and sums in trees of at most 32 levels of
    a few terms, 2^-24 each of the sum of absolute terms: 1e-5 of the largest
    value. bf16: the same, rounded once (2^-8 of the value). The two terms of
    dy = ry (c - yn mean(c yn)) cancel where a row is one column, to eps / y^2
    of each; either is off by at most eight roundings (ry, yn: three; c: four;
    the product), so dy by 2 8 2^-24 of the larger, max |ry c|. 2^-126: fp32 has
    no smaller numbers in full precision (sigmoid(-200) is 2^-288)."""
    from tarmac_b200 import ops
    c = {n: None if x is None else x.cuda() for n, x in t.items()}
    rows = {n: None if c[n] is None else wrap(c[n]) for n in ("x", "y", "gate", "dh", "dz")}
    args = (rows["x"], rows["y"], c["w_post"], c["w_pre"], rows["gate"], c["scale"])
    got = [*ops.residual_norm(*args, eps=EPS),
           *ops.residual_norm_backward(*args, rows["dh"], rows["dz"], eps=EPS)]
    f = {n: None if x is None else x.double() for n, x in t.items()}
    zero = torch.zeros_like(f["x"])
    dh, dz = (zero if f[n] is None else f[n] for n in ("dh", "dz"))
    plain = (f["x"], f["y"], f["w_post"], f["w_pre"], f["gate"], f["scale"])
    want = [*d64.norm(*plain, EPS), *d64.norm_grads(*plain, dh, dz, EPS)]
    for i, (a, b) in enumerate(zip(got, want)):
        name = ("h", "z", "dx", "dy", "dw_post", "dw_pre", "dgate", "dscale")[i]
        given = {"dw_post": "w_post", "dw_pre": "w_pre", "dgate": "gate", "dscale": "scale"}
        if name in given and t[given[name]] is None:
            assert a is None
            continue
        weight = name in ("dw_post", "dw_pre", "dscale")
        assert a.dtype == (F32 if weight else dtype) and a.is_contiguous(), name
        err, b = (a.double().cpu() - b).abs(), b.abs()
        # a weight's gradient is a sum over all rows: relative to their number
        top = b.max() if not weight else b.max() + t["x"].numel() / t["x"].shape[-1]
        tol = 1e-5 * top + 2.0 ** -126
        if name == "dy":
            tol = tol + 2 ** -20 * dy_term(f, dh, dz)
        if dtype is BF16 and not weight:
            tol = tol + 2 ** -8 * b
        assert (err <= tol).all(), (name, (err - tol).max())
    return got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [1, 2, 3, 8, 12, 16, 17, 31, 64, 100, 250, 255, 256, 257, 264, 500,
                               1000, 2048, 2049, 4100, 8184, 8191, 8192])
def test_widths(D, dtype):
    check(inputs((3, 5, D), dtype), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 2, 7, 33, 1000, 5000])
@pytest.mark.parametrize("D", [8, 40, 200, 320])
def test_rows(rows, D, dtype):
    check(inputs((rows, D), dtype), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("weights", [(), ("w_post",), ("w_pre", "scale"), WEIGHTS])
def test_parts(weights, gate, dtype):
    check(inputs((2, 9, 72), dtype, gate, weights), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("none", ["dh", "dz"])
def test_one_gradient(none, dtype):
    t = inputs((4, 11, 96), dtype)
    t[none] = None
    check(t, dtype)


def rows_apart(t):
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 24, device=t.device, dtype=t.dtype)
    wide[..., 8:8 + t.shape[-1]] = t
    return wide[..., 8:8 + t.shape[-1]]


def swapped(t):
    return t.transpose(0, 1).contiguous().transpose(0, 1)


def off_grid(t):
    flat = torch.zeros(t.numel() + 1, device=t.device, dtype=t.dtype)
    flat[1:] = t.flatten()
    return flat[1:].view(t.shape)


def columns_apart(t):
    return t.transpose(1, 2).contiguous().transpose(1, 2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("wrap", [rows_apart, swapped, off_grid, columns_apart])
@pytest.mark.parametrize("D", [64, 272])
def test_layouts(D, wrap, dtype):
    check(inputs((6, 7, D), dtype), dtype, wrap)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_other_ranks(dtype):
    for shape in ((40,), (7, 40), (2, 3, 4, 40), (0, 3, 40)):
        t = inputs(shape, dtype)
        if 0 in shape:
            from tarmac_b200 import ops
            c = {n: x.cuda() for n, x in t.items()}
            args = (c["x"], c["y"], c["w_post"], c["w_pre"], c["gate"], c["scale"])
            assert ops.residual_norm(*args)[0].shape == shape
            grads = ops.residual_norm_backward(*args, c["dh"], c["dz"])
            assert all((grads[i] == 0).all() for i in (2, 3, 5))
        else:
            check(t, dtype)


def test_broadcast_gate():
    """One gate per episode for all of its rows (stride 0)."""
    t = inputs((3, 20, 64), BF16)
    t["gate"] = t["gate"][:, :1].expand(-1, 20, -1)
    check(t, BF16, lambda x: x)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [48, 768])
def test_same_bits_and_graph(D, dtype):
    from tarmac_b200 import ops
    c = {n: x.cuda() for n, x in inputs((300, D), dtype).items()}
    args = (c["x"], c["y"], c["w_post"], c["w_pre"], c["gate"], c["scale"])

    def run():
        return [*ops.residual_norm(*args), *ops.residual_norm_backward(*args, c["dh"], c["dz"])]

    first = run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = run()
    g.replay()
    for a, b in zip(held, first):
        assert torch.equal(a, b)
    c["x"].copy_(torch.randn_like(c["x"]))
    g.replay()
    for a, b in zip(held, run()):
        assert torch.equal(a, b)


def test_large_gates_and_zero_rows():
    """Gates of any size give 0 or 1; rows of zeros give the eps form."""
    t = inputs((2, 6, 32), F32)
    t["gate"][0] = 200.0
    t["gate"][1] = -200.0
    t["x"][:, 0] = 0.0
    t["y"][:, 1] = 0.0
    t["x"][:, 2] = t["y"][:, 2] = 0.0
    t["dz"][:, 0] = t["dz"][:, 2] = t["dz"][1] = 0.0
    t["dh"][:, 1:3] = 0.0
    t["dz"][:, 1] = 0.0
    check(t, F32)
