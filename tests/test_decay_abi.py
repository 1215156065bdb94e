"""Argument checks of attention with a decay and of the norms around a block, at
the C ABI and in the launchers. Nothing is launched and no GPU is needed."""

from __future__ import annotations

import pytest
import torch

from tarmac_b200 import _lib, autograd, ops
from tarmac_b200.heads import DecayComm, decay_slopes

FAKE = 1 << 20  # a non-null, 16-byte aligned address that is never touched


def _decay(backward, **kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE, dout=FAKE, strides=None, rate=FAKE, state=FAKE,
             last=FAKE, lens=None, B=2, N=8, H=4, Hk=2, d=16, dtype=_lib.F32, scale=0.25,
             dq=FAKE, dk=FAKE, dv=FAKE, first=FAKE, work=FAKE)
    a.update(kw)
    mid = (a["lens"], a["B"], a["N"], a["H"], a["Hk"], a["d"], a["dtype"], a["scale"])
    if backward:
        return _lib.lib().tarmac_decay_attention_backward(
            a["q"], a["k"], a["v"], a["dout"], a["strides"], a["rate"], a["state"], a["last"],
            *mid, a["dq"], a["dk"], a["dv"], a["first"], a["work"], None)
    return _lib.lib().tarmac_decay_attention(
        a["q"], a["k"], a["v"], a["out"], a["strides"], a["rate"], a["state"], a["last"], *mid,
        a["work"], None)


BOTH = [
    (dict(q=None), _lib.ERR_NULL), (dict(k=None), _lib.ERR_NULL), (dict(v=None), _lib.ERR_NULL),
    (dict(rate=None), _lib.ERR_NULL), (dict(dtype=2), _lib.ERR_DTYPE),
    (dict(d=0), _lib.ERR_SHAPE), (dict(d=129), _lib.ERR_SHAPE), (dict(B=-1), _lib.ERR_SHAPE),
    (dict(N=-1), _lib.ERR_SHAPE), (dict(scale=0.0), _lib.ERR_SHAPE),
    (dict(scale=float("nan")), _lib.ERR_SHAPE), (dict(scale=float("inf")), _lib.ERR_SHAPE),
    (dict(H=3), _lib.ERR_HEADS), (dict(Hk=0), _lib.ERR_HEADS),
    (dict(N=2 ** 29 + 1), _lib.ERR_N_TOO_LARGE), (dict(B=2 ** 23, H=4), _lib.ERR_N_TOO_LARGE),
    (dict(q=FAKE + 2), _lib.ERR_ALIGN), (dict(rate=FAKE + 2), _lib.ERR_ALIGN),
    (dict(state=FAKE + 1), _lib.ERR_ALIGN), (dict(last=FAKE + 2), _lib.ERR_ALIGN),
    (dict(lens=FAKE + 2), _lib.ERR_ALIGN), (dict(work=FAKE + 8), _lib.ERR_ALIGN),
    (dict(B=0), _lib.OK), (dict(B=0, N=0), _lib.OK),
    (dict(N=0, state=FAKE, last=FAKE, first=FAKE), _lib.OK),
]


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("kw,status", BOTH)
def test_decay_validation(kw, status, backward):
    assert _decay(backward, **kw) == status


def test_decay_own_checks():
    assert _decay(False, out=None) == _lib.ERR_NULL
    assert _decay(False, out=FAKE + 4) == _lib.ERR_ALIGN
    for name in ("dout", "dq", "dk", "dv"):
        assert _decay(True, **{name: None}) == _lib.ERR_NULL
    assert _decay(True, dk=FAKE + 4) == _lib.ERR_ALIGN
    assert _decay(True, work=None) == _lib.ERR_NULL          # shared heads are summed
    assert _decay(False, B=1, N=8192, work=None) == _lib.ERR_NULL  # segments
    fwd = _lib.lib().tarmac_decay_attention_workspace
    bwd = _lib.lib().tarmac_decay_attention_backward_workspace
    for dt in (_lib.F32, _lib.BF16):
        assert fwd(1, 8192, 4, 64, dt, 0) >= 2 * 4 * 64 * 64 * 4
        assert fwd(1, 1, 4, 64, dt, 1) == 0
        assert fwd(4096, 512, 4, 64, dt, 0) == 0
        assert fwd(0, 512, 4, 64, dt, 1) == 0
        assert bwd(4096, 512, 4, 4, 64, dt, 0) == 0
        assert bwd(4096, 512, 4, 2, 64, dt, 0) >= 4096 * 512 * 4 * 64 * 4
    assert fwd(2, 8, 4, 64, 7, 0) == 0


@pytest.mark.parametrize("scale,status", [
    (2.0 ** -60, _lib.OK), (2.0 ** 20, _lib.OK), (2.0 ** -61, _lib.ERR_SHAPE),
    (2.0 ** 21, _lib.ERR_SHAPE), (1e-40, _lib.ERR_SHAPE)])
def test_scales_of_the_gradients(scale, status):
    """Beyond these bounds powers of a decay or the state over the scale could leave
    fp32's range."""
    assert _decay(True, B=0, scale=scale) == status
    assert _decay(False, B=0, scale=scale) == _lib.OK


def _norm(backward, **kw):
    a = dict(x=FAKE, y=FAKE, gate=FAKE, dh=FAKE, dz=FAKE, w=None, B=2, N=3, D=64, dtype=_lib.F32,
             eps=1e-6, o=FAKE, o2=FAKE, dgate=FAKE, work=FAKE)
    a.update(kw)
    if backward:
        return _lib.lib().tarmac_residual_norm_backward(
            a["x"], a["y"], a["gate"], a["dh"], a["dz"], None, a["w"], None, None, a["B"], a["N"],
            a["D"], a["dtype"], a["eps"], a["o"], a["o2"], a["dgate"], None, None, None, a["work"],
            None)
    return _lib.lib().tarmac_residual_norm(
        a["x"], a["y"], a["gate"], None, a["w"], None, None, a["B"], a["N"], a["D"], a["dtype"],
        a["eps"], a["o"], a["o2"], None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("kw,status", [
    (dict(x=None), _lib.ERR_NULL), (dict(y=None), _lib.ERR_NULL), (dict(o2=None), _lib.ERR_NULL),
    (dict(dtype=7), _lib.ERR_DTYPE), (dict(D=0), _lib.ERR_SHAPE), (dict(D=8193), _lib.ERR_SHAPE),
    (dict(B=-1), _lib.ERR_SHAPE), (dict(eps=-1.0), _lib.ERR_SHAPE),
    (dict(eps=float("nan")), _lib.ERR_SHAPE), (dict(B=2 ** 20, N=2 ** 20), _lib.ERR_N_TOO_LARGE),
    (dict(x=FAKE + 1), _lib.ERR_ALIGN), (dict(gate=FAKE + 2), _lib.ERR_ALIGN),
    (dict(w=FAKE + 1), _lib.ERR_ALIGN), (dict(o=FAKE + 2), _lib.ERR_ALIGN), (dict(N=0), _lib.OK)])
def test_norm_validation(kw, status, backward):
    assert _norm(backward, **kw) == status


def test_norm_backward_own_checks():
    assert _norm(True, dgate=None) == _lib.ERR_NULL
    assert _norm(True, work=None) == _lib.ERR_NULL
    assert _norm(True, dz=FAKE + 2) == _lib.ERR_ALIGN
    assert _lib.lib().tarmac_residual_norm_workspace(2, 3, 64) >= 2 * 64 * 4
    assert _lib.lib().tarmac_residual_norm_workspace(0, 3, 64) == 0


def test_no_cpu_path():
    q, rate = torch.zeros(1, 2, 2, 8), torch.zeros(2)
    with pytest.raises(RuntimeError):
        ops.decay_attention(q, q, q, rate)
    with pytest.raises(RuntimeError):
        ops.decay_attention_backward(q, q, q, rate, q)
    with pytest.raises(RuntimeError):
        ops.residual_norm(q, q)
    with pytest.raises(RuntimeError):
        ops.residual_norm_backward(q, q, None, None, None, None, q, q)


def test_decays_have_no_gradient():
    q = torch.zeros(1, 2, 2, 8)
    with pytest.raises(ValueError, match="gradient"):
        autograd.decay_attention(q, q, q, torch.zeros(2, requires_grad=True))


def test_block_arguments():
    with pytest.raises(ValueError):
        DecayComm(8, 4, 8, 3)
    m = DecayComm(8, 4, 8, 2)
    assert m.empty_state(3).shape == (3, 4, 8, 8)
    assert "log_decay" in m.state_dict()
    assert (decay_slopes(8) < 0).all() and decay_slopes(8)[-1] == -1 / 256


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_cast_block_keeps_its_decays(dtype):
    m = DecayComm(24, 6, 16)
    want = decay_slopes(6)
    for step in (lambda: m.to(dtype), lambda: m.double(), lambda: m.to(dtype), lambda: m.float()):
        step()
        assert torch.equal(m.log_decay.float(), want)
    assert m.log_decay.dtype is torch.float32 and "log_decay" in m.state_dict()
    assert m.to(dtype).log_decay.dtype is torch.float32 and m.proj.weight.dtype is dtype


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_cast_block_keeps_its_norms_weights(dtype):
    """What the kernels read in fp32 is neither rounded nor cast call after call."""
    m = DecayComm(24, 6, 16)
    own = ("norm_q", "norm_k", "norm_post", "norm_next", "scale")
    torch.manual_seed(0)
    with torch.no_grad():
        for n in own:
            getattr(m, n).add_(0.1 * torch.randn_like(getattr(m, n)))
    want = {n: getattr(m, n).detach().clone() for n in own}
    params = dict(m.named_parameters())
    for p in m.parameters():
        p.grad = torch.ones_like(p)
    for step in (lambda: m.to(dtype), lambda: m.double(), lambda: m.to(dtype)):
        step()
        for n in own:
            w = getattr(m, n)
            assert w is params[n] and w.requires_grad
            assert w.dtype == w.grad.dtype == m.log_decay.dtype
            assert torch.equal(w.detach().float(), want[n])
        assert m.qkv.weight.dtype == m.qkv.weight.grad.dtype == m.gate.bias.dtype
    assert m.scale.dtype is torch.float32 and m.gate.weight.dtype is dtype


def test_room_for_a_state_renewed_in_place():
    """fp32 rows of 16 columns over several segments: each reads the state."""
    sizes = 3, 500, 2, 16, _lib.F32
    assert ops.decay_attention_plan(*sizes[:3], 1, 16, torch.float32)["segments"] > 1
    room = _lib.lib().tarmac_decay_attention_workspace
    assert room(*sizes, 1) >= room(*sizes, 0) + 3 * 2 * 16 * 16 * 4 > 0
