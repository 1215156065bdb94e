"""GPU: GraphedCall on calls that change their arguments: a state renewed in place, a
history that grows. Nothing may have happened to them before the first replay,
and every replay happens to them once."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def stream(T, B=3, H=2, d=16):
    g = torch.Generator().manual_seed(T)
    q, k, v = (torch.randn(B, T, H, d, generator=g).cuda() for _ in range(3))
    S = torch.randn(B, H, d, d, generator=g).cuda()
    return q, k, v, torch.tensor([-0.1, -0.5]).cuda(), S


def renew(q, k, v, rate, S):
    from tarmac_b200 import ops
    return ops.decay_attention(q, k, v, rate, S, state_out=S)[0]


def rows(t, *ts):
    return [x[:, t:t + 1].contiguous() for x in ts]


@pytest.mark.parametrize("zeros", [False, True])
def test_a_state_starts_and_steps_as_direct_calls(zeros):
    """The same bits as direct calls; `zeros`: an example that leaves its state as
    it was."""
    from tarmac_b200.graphs import GraphedCall
    q, k, v, rate, S = stream(4)
    want_S, want = S.clone(), []
    for t in range(4):
        want.append(renew(*rows(t, q, k, v), rate, want_S))
    first = [torch.zeros_like(x) if zeros else x for x in rows(0, q, k, v)]
    mine = torch.zeros_like(S) if zeros else S.clone()
    before = mine.clone()
    step = GraphedCall(renew, *first, rate, mine)
    assert torch.equal(mine, before)
    mine.copy_(S)
    for t in range(4):
        assert torch.equal(step(*rows(t, q, k, v), rate, mine), want[t])
    assert torch.equal(mine, want_S)


@pytest.mark.parametrize("zeros", [False, True])
def test_another_state_is_renewed_itself(zeros):
    from tarmac_b200.graphs import GraphedCall
    q, k, v, rate, S = stream(2)
    example = torch.zeros_like(S)
    first = [torch.zeros_like(x) if zeros else x for x in rows(0, q, k, v)]
    step = GraphedCall(renew, *first, rate, example)
    assert (example == 0).all()
    for state in (S.clone(), 2 * S):
        want = state.clone()
        out = renew(*rows(1, q, k, v), rate, want)
        assert torch.equal(step(*rows(1, q, k, v), rate, state), out)
        assert torch.equal(state, want)


def test_a_replay_is_noticed_by_autograd():
    from tarmac_b200 import autograd
    from tarmac_b200.graphs import GraphedCall
    q, k, v, rate, S = stream(3)
    step = GraphedCall(renew, *rows(0, q, k, v), rate, S)
    leaves = [x.requires_grad_() for x in rows(1, q, k, v)]
    out = autograd.decay_attention(*leaves, rate, S)
    step(*rows(2, q, k, v), rate, S)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


def test_a_call_that_changes_nothing_leaves_its_arguments_alone():
    from tarmac_b200 import ops
    from tarmac_b200.graphs import GraphedCall
    q, k, v, rate, _ = stream(5)
    versions = [t._version for t in (q, k, v, rate)]
    step = GraphedCall(ops.decay_attention, q, k, v, rate)
    assert torch.equal(step(q, k, v, rate), ops.decay_attention(q, k, v, rate))
    assert versions == [t._version for t in (q, k, v, rate)]


def test_blocks():
    """One new row of either block, in a loop: outputs and what is kept as from
    direct calls."""
    from tarmac_b200.graphs import GraphedCall
    from tarmac_b200.heads import DecayComm, HeadComm, rotation_table
    torch.manual_seed(0)
    B, T, dim = 3, 4, 24
    x = torch.randn(B, T, dim, device="cuda")
    cos, sin = rotation_table(torch.arange(T, device="cuda")[None], 16)
    m = DecayComm(dim, 2, 16).cuda()
    S, want_S = m.empty_state(B), m.empty_state(B)
    step = None
    for t in range(T):
        a, c, s = rows(t, x, cos, sin)
        h, z = m.step(a, a, c, s, want_S)
        if step is None:
            step = GraphedCall(m.step, a.clone(), a.clone(), c, s, S)
            assert (S == 0).all()
        got = step(a, a, c, s, S)
        assert torch.equal(got[0], h) and torch.equal(got[1], z) and torch.equal(S, want_S)
    m = HeadComm(dim, 2, 16).cuda()
    kept = [torch.zeros(B, T, 2, 16, device="cuda") for _ in range(4)]
    n, want_n = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))
    step = None
    for t in range(T):
        a, c, s = rows(t, x, cos, sin)
        y = m.step(a, c, s, kept[0], kept[1], want_n)
        if step is None:
            step = GraphedCall(m.step, a, c, s, kept[2], kept[3], n)
            assert (n == 0).all() and (kept[2] == 0).all()
        got = step(a, c, s, kept[2], kept[3], n)
        assert torch.equal(got, y) and torch.equal(n, want_n)
    assert torch.equal(kept[0], kept[2]) and torch.equal(kept[1], kept[3])


def test_no_room_for_copies(monkeypatch):
    """Arguments that the device cannot hold twice are kept in host memory."""
    from tarmac_b200 import graphs
    q, k, v, rate, S = stream(4)

    class Full(torch.Tensor):
        def clone(self, *a, **kw):
            raise torch.OutOfMemoryError("no room")

    monkeypatch.setattr(torch.Tensor, "clone", Full.clone)
    mine, want_S = S + 0, S + 0
    step = graphs.GraphedCall(renew, *rows(0, q, k, v), rate, mine)
    monkeypatch.undo()
    assert torch.equal(mine, want_S)
    assert torch.equal(step(*rows(1, q, k, v), rate, mine), renew(*rows(1, q, k, v), rate, want_S))
    assert torch.equal(mine, want_S)


def test_arguments_of_other_types():
    """Whatever a function takes: masks, complex numbers, scalars, views, NaN."""
    from tarmac_b200.graphs import GraphedCall
    x = torch.full((4, 6), float("nan"), device="cuda")
    mask = torch.tensor([True, False, True, True], device="cuda")
    z = torch.randn(3, dtype=torch.complex64, device="cuda").conj()
    one = torch.ones((), device="cuda", dtype=torch.float64)
    wide = torch.randn(1, 6, device="cuda").expand(4, 6)
    args = (x.t(), mask, z, one, wide)
    versions = [t._version for t in args]

    def fn(x, mask, z, one, wide):
        return mask[:, None] * wide * one, z * 2, x.isnan().sum()

    step = GraphedCall(fn, *args)
    for a, b in zip(step(*args), fn(*args)):
        assert torch.equal(a, b)
    assert versions == [t._version for t in args]


def test_garbage_graphs_do_not_end_a_capture():
    """A graph in a reference cycle that nobody holds is released before the capture,
    not by a collection in it."""
    import gc
    from tarmac_b200 import ops
    from tarmac_b200.graphs import GraphedCall
    x = torch.randn(4, 8, 16, device="cuda")
    gc.collect()
    gc.disable()
    try:
        old = [GraphedCall(ops.dense_attention, x, x, x)]
        old.append(old)
        del old

        def fn(x):
            if torch.cuda.is_current_stream_capturing():
                gc.collect()
            return ops.dense_attention(x, x, x)

        step = GraphedCall(fn, x)
    finally:
        gc.enable()
    assert torch.equal(step(x), ops.dense_attention(x, x, x))
