"""Argument checks of the multi-head entry points at the C ABI. Every call
fails validation or has no rows, so nothing is launched and no GPU is needed."""

from __future__ import annotations

import pytest

from tarmac_b200 import _lib

FAKE = 1 << 20  # a non-null, 16-byte aligned address that is never touched


def _attention(backward, **kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE, lse=FAKE, dout=FAKE, strides=None, key_len=None,
             q_start=None, bits=None, B=2, Nq=8, Nk=8, H=4, Hk=2, d=16, dtype=_lib.F32,
             peers=_lib.PEERS_ALL, scale=0.25, dq=FAKE, dk=FAKE, dv=FAKE, work=FAKE)
    a.update(kw)
    mid = (a["key_len"], a["q_start"], a["bits"], 0, a["B"], a["Nq"], a["Nk"], a["H"], a["Hk"],
           a["d"], a["dtype"], a["peers"], a["scale"])
    if backward:
        return _lib.lib().tarmac_head_attention_backward(
            a["q"], a["k"], a["v"], a["out"], a["lse"], a["dout"], a["strides"], *mid, a["dq"],
            a["dk"], a["dv"], a["work"], None)
    return _lib.lib().tarmac_head_attention(
        a["q"], a["k"], a["v"], a["out"], a["lse"], a["strides"], *mid, a["work"], None)


BOTH = [
    (dict(q=None), _lib.ERR_NULL),
    (dict(k=None), _lib.ERR_NULL),
    (dict(out=None), _lib.ERR_NULL),
    (dict(dtype=5), _lib.ERR_DTYPE),
    (dict(d=0), _lib.ERR_SHAPE),
    (dict(d=129), _lib.ERR_SHAPE),
    (dict(B=-1), _lib.ERR_SHAPE),
    (dict(scale=0.0), _lib.ERR_SHAPE),
    (dict(scale=float("inf")), _lib.ERR_SHAPE),
    (dict(scale=float("nan")), _lib.ERR_SHAPE),
    (dict(H=3), _lib.ERR_HEADS),
    (dict(Hk=0), _lib.ERR_HEADS),
    (dict(peers=3), _lib.ERR_MODE),
    (dict(Nk=2 ** 30 + 1), _lib.ERR_N_TOO_LARGE),
    (dict(q=FAKE + 2), _lib.ERR_ALIGN),
    (dict(key_len=FAKE + 1), _lib.ERR_ALIGN),
    (dict(work=FAKE + 8), _lib.ERR_ALIGN),
    (dict(B=0), _lib.OK),
]


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("kw,status", BOTH)
def test_attention_validation(kw, status, backward):
    assert _attention(backward, **kw) == status


def test_attention_own_checks():
    assert _attention(False, out=FAKE + 4) == _lib.ERR_ALIGN
    assert _attention(True, dk=FAKE + 4) == _lib.ERR_ALIGN
    assert _attention(True, lse=None) == _lib.ERR_NULL
    assert _attention(True, work=None) == _lib.ERR_NULL
    # one token over a long history splits the keys and needs its scratch
    assert _attention(False, B=1, Nq=1, Nk=4096, work=None) == _lib.ERR_NULL
    so = _lib.lib()
    assert so.tarmac_head_attention_workspace(1, 1, 4096, 4, 2, 16) > 0
    assert so.tarmac_head_attention_workspace(512, 512, 512, 4, 2, 16) == 0
    assert so.tarmac_head_attention_backward_workspace(2, 8, 4) >= 2 * 2 * 8 * 4 * 4


def _rotate(**kw):
    a = dict(q=FAKE, k=FAKE, qo=FAKE, ko=FAKE, wq=None, wk=None, cos=FAKE, sin=FAKE, B=2, N=3,
             H=4, Hk=2, d=16, r=16, dtype=_lib.BF16, eps=1e-6)
    a.update(kw)
    return _lib.lib().tarmac_qk_norm_rotate(
        a["q"], a["k"], a["qo"], a["ko"], None, a["wq"], a["wk"], a["cos"], a["sin"], 0, a["B"],
        a["N"], a["H"], a["Hk"], a["d"], a["r"], a["dtype"], a["eps"], 0, None)


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), _lib.ERR_NULL), (dict(ko=None), _lib.ERR_NULL), (dict(cos=None), _lib.ERR_NULL),
    (dict(dtype=3), _lib.ERR_DTYPE), (dict(d=130, r=2), _lib.ERR_SHAPE),
    (dict(r=3), _lib.ERR_HEADS), (dict(r=18), _lib.ERR_HEADS), (dict(H=0), _lib.ERR_HEADS),
    (dict(eps=-1.0), _lib.ERR_SHAPE), (dict(q=FAKE + 1), _lib.ERR_ALIGN),
    (dict(wq=FAKE + 2), _lib.ERR_ALIGN), (dict(N=0), _lib.OK)])
def test_rotate_validation(kw, status):
    assert _rotate(**kw) == status


def test_pack_validation():
    so = _lib.lib()
    assert so.tarmac_pack_visibility(None, 9, 3, 1, 3, 3, FAKE, None) == _lib.ERR_NULL
    assert so.tarmac_pack_visibility(FAKE, 9, 3, 1, -3, 3, FAKE, None) == _lib.ERR_SHAPE
    assert so.tarmac_pack_visibility(FAKE, 9, 3, 1, 3, 3, FAKE + 2, None) == _lib.ERR_ALIGN
    assert so.tarmac_pack_visibility(FAKE, 9, 3, 1, 3, 0, FAKE, None) == _lib.OK
    assert _lib.strerror(_lib.ERR_HEADS) != "unknown status"
