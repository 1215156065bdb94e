"""Host side of HeadComm.step: what it refuses before it touches the history
(CPU), and episodes without room left (GPU)."""

from __future__ import annotations

import pytest
import torch

from tarmac_b200.heads import HeadComm, rotation_table

B, ROOM, H, HK, D = 3, 5, 4, 2, 16


def inputs(device="cpu"):
    g = torch.Generator().manual_seed(0)
    cos, sin = rotation_table(torch.arange(ROOM + 3)[None], D)
    return dict(x=torch.randn(B, 1, 8, generator=g).to(device),
                cos=cos[:, :1].to(device), sin=sin[:, :1].to(device),
                past_k=torch.zeros(B, ROOM, HK, D, device=device),
                past_v=torch.zeros(B, ROOM, HK, D, device=device),
                past_len=torch.zeros(B, dtype=torch.int64, device=device))


@pytest.mark.parametrize("name,value,error", [
    ("x", torch.zeros(B, 2, 8), ValueError),  # one row at a time
    ("past_k", torch.zeros(B + 1, ROOM, HK, D), ValueError),
    ("past_k", torch.zeros(B, 0, HK, D), ValueError),
    ("past_k", torch.zeros(B, ROOM, H, D), ValueError),
    ("past_v", torch.zeros(B, ROOM + 1, HK, D), ValueError),
    ("past_len", torch.zeros(1, dtype=torch.int64), ValueError),
    ("past_len", torch.zeros(B), TypeError)])
def test_step_refuses(name, value, error):
    torch.manual_seed(0)
    m, a = HeadComm(8, H, D, HK), inputs()
    a[name] = value
    before = a["past_len"].clone()
    with pytest.raises(error):
        m.step(**a)
    assert torch.equal(a["past_len"], before)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_step_without_room(dtype):
    """An episode whose history is full gets NaN; the others, and the room
    behind the history, are not touched."""
    torch.manual_seed(0)
    m, a = HeadComm(8, H, D, HK).cuda(), inputs("cuda")
    store = torch.full((2, B, ROOM + 2, HK, D), 3.0, device="cuda")
    a["past_k"], a["past_v"] = store[0, :, 1:ROOM + 1], store[1, :, 1:ROOM + 1]
    a["past_len"] = torch.tensor([ROOM, 2, -1], device="cuda", dtype=dtype)
    y = m.step(**a)
    assert y[0].isnan().all() and y[2].isnan().all() and y[1].isfinite().all()
    assert a["past_len"].tolist() == [ROOM + 1, 3, 0]
    assert (store[:, :, 0] == 3.0).all() and (store[:, :, ROOM + 1] == 3.0).all()
    untouched = store[:, 1].clone()
    untouched[:, 3] = 3.0
    assert (untouched == 3.0).all()  # episode 1: its row 2 alone is new
    assert (store[:, 1, 3] != 3.0).any()
    a["past_len"].fill_(1)
    assert m.step(**a).isfinite().all()
