"""GPU parity of the multi-head operators (csrc/head_*.cu) against their plain
64-bit forms (tests/_heads64.py, whose gradients test_heads_oracle.py pins to
differences).

Tolerances, element by element, from the roundings of each path:

* rotate: fp32 arithmetic on rows of d columns, a handful of roundings and a
  sum of d squares: (d / 8 + 16) 2^-24 of the row's largest value; bf16 adds
  its output rounding, 2^-8 of the value (8 significant bits: the unit
  roundoff is 2^-8). Weight gradients: a sum of n terms in fp32, split over lanes:
  (n / 64 + 64) 2^-24 of the sum of magnitudes at most.
* attention, fp32: a score's products drop below 2^-22 and its chains of d / 8
  chopped sums lose 2^-23 each, of S = max scale sum |q k|; weights carry that
  twice (numerator and sum) and the sums over N keys (N / 32 + 16) 2^-22:
  eps = 2 (d / 8 + 8) 2^-23 S + (N / 32 + 16) 2^-22, relative to the sums of
  magnitudes that make up each output.
* attention, bf16: the weights and dS are rounded (2^-8), outputs too (2^-8),
  and D takes the rounded out (2^-8), each of its own magnitudes, plus the fp32
  eps.
"""

from __future__ import annotations

import pytest
import torch

import _heads64 as h64

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from tarmac_b200 import ops
    return ops


def near(got, want, bound):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (
        f"{int(bad.sum())} of {bad.numel()} off; worst {((got - want).abs() / bound)[bad].max()} "
        f"times the bound")


def rows(g, B, N, heads, d, dtype, shift=0):
    """Column blocks of one [B, N, sum(heads) d + shift] tensor, moved by
    `shift` elements off its rows' starts, as [B, N, h, d] views on the GPU."""
    x = torch.randn(B, N, sum(heads) * d + shift, generator=g).to(dtype).cuda()
    return [p.unflatten(-1, (h, d)) for p, h in
            zip(x[..., shift:].split([h * d for h in heads], -1), heads)]


def wide(*ts):
    return [None if t is None else t.detach().double().cpu() for t in ts]


# ---------------------------------------------------------------------------
# rotate
# ---------------------------------------------------------------------------

ROTATE = [  # B, N, H, Hk, d, r, interleaved, own table, shift
    (3, 5, 4, 4, 16, 16, False, True, 0),
    (2, 33, 6, 2, 40, 24, True, True, 0),
    (2, 9, 3, 1, 40, 24, False, False, 0),
    (1, 1, 1, 1, 2, 2, False, False, 0),
    (2, 7, 5, 3, 1, 0, False, False, 0),
    (2, 7, 5, 3, 33, 6, True, True, 0),
    (2, 7, 5, 3, 127, 126, False, True, 0),
    (2, 6, 9, 2, 128, 128, False, True, 0),
    (2, 6, 2, 9, 128, 64, True, False, 0),
    (2, 6, 4, 2, 64, 32, False, True, 3),
    (2, 6, 4, 2, 80, 80, False, True, 4),
    (700, 6, 4, 4, 16, 16, False, True, 0),
    # rows that fill their lanes, over several row tiles of a block
    (3, 50, 4, 2, 64, 32, False, False, 0),
    (2, 301, 6, 2, 64, 64, True, True, 0),
    (2, 45, 2, 6, 128, 128, False, False, 0),
    (3, 131, 2, 4, 128, 64, False, True, 0),
    (5, 70, 8, 4, 32, 16, True, True, 0),
    (1, 260, 2, 2, 32, 32, False, True, 0),
    (2, 150, 4, 6, 48, 16, False, True, 0),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,N,H,Hk,d,r,inter,own,shift", ROTATE)
def test_rotate(ops, B, N, H, Hk, d, r, inter, own, shift, dtype):
    g = torch.Generator().manual_seed(B * 1000 + d)
    q, k = rows(g, B, N, (H, Hk), d, dtype, shift)
    q, k = q * 3.0 if shift == 0 else q, k  # a scaled, contiguous query too
    wq, wk = (1 + 0.3 * torch.randn(d, generator=g) for _ in range(2))
    a = 7 * torch.randn(B if own else 1, N, r // 2, generator=g)
    cos, sin = a.cos(), a.sin()
    dq, dk = rows(g, B, N, (H, Hk), d, dtype, shift)
    gpu = [t.cuda() for t in (wq, wk, cos, sin)]
    eps = 1e-6
    out = ops.qk_norm_rotate(q, k, *gpu, eps, inter)
    grad = ops.qk_norm_rotate_backward(q, k, *gpu, dq, dk, eps, inter)
    again = ops.qk_norm_rotate_backward(q, k, *gpu, dq, dk, eps, inter)
    for x, y in zip(grad, again):
        assert torch.equal(x, y)  # a fixed order of sums
    cos, sin = cos.double(), sin.double()
    u = (d / 8 + 16) * 2.0 ** -24
    for x, w, y, gy, dx, dw in ((q, wq, out[0], dq, grad[0], grad[2]),
                                (k, wk, out[1], dk, grad[1], grad[3])):
        x, w, gy = wide(x, w, gy)
        want = h64.rotate(x, w, cos, sin, eps, inter)
        rnd = 2.0 ** -8 if dtype == BF16 else 0.0
        near(y, want, u * want.abs().amax(-1, keepdim=True) * 2 + rnd * want.abs() + 1e-30)
        wdx, wdw = h64.rotate_grad(x, w, cos, sin, eps, inter, gy)
        s = 1.0 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        mag = s * (gy.abs().amax(-1, keepdim=True) * w.abs().max() * 2 *
                   (1 + x.abs().amax(-1, keepdim=True) ** 2 * s * s))
        near(dx, wdx, u * mag + rnd * wdx.abs() + 1e-30)
        n = x.shape[0] * x.shape[1] * x.shape[2]
        total = (2 * gy.abs().amax(-1, keepdim=True) * (x * s).abs()).sum((0, 1, 2))
        near(dw, wdw, (n / 64 + 64) * 2.0 ** -24 * total + 1e-30)


def test_rotate_without_weights(ops):
    g = torch.Generator().manual_seed(1)
    q, k = rows(g, 2, 4, (3, 2), 24, F32)
    cos, sin = torch.ones(1, 4, 12).cuda(), torch.zeros(1, 4, 12).cuda()
    one = torch.ones(24).cuda()
    for x, y in zip(ops.qk_norm_rotate(q, k, None, None, cos, sin),
                    ops.qk_norm_rotate(q, k, one, one, cos, sin)):
        assert torch.equal(x, y)
    dq, dk, dwq, dwk = ops.qk_norm_rotate_backward(q, k, None, one, cos, sin, q, k)
    assert dwq is None and dwk.shape == (24,)


def test_rotate_zero_rows_and_values(ops):
    q = torch.zeros(2, 3, 2, 16).cuda()
    cos, sin = torch.ones(1, 3, 8).cuda(), torch.zeros(1, 3, 8).cuda()
    for t in ops.qk_norm_rotate(q, q, None, None, cos, sin):
        assert (t == 0).all()
    e = torch.empty(0, 3, 2, 16).cuda()
    w = torch.ones(16).cuda()
    dq, dk, dwq, dwk = ops.qk_norm_rotate_backward(e, e, w, w, cos, sin, e, e)
    assert dq.shape == e.shape and (dwq == 0).all() and (dwk == 0).all()
    assert ops.qk_norm_rotate(e, e, w, w, cos, sin)[0].shape == e.shape


def test_rotate_many_rows(ops):
    """Rows times lanes per row past 32 bits: a row of width 1 keeps its sign
    (x / sqrt(x^2) with eps 0), forward and in the weight's gradient."""
    N = 2 ** 27 + 300
    q = torch.ones(1, N, 1, 1, dtype=BF16, device="cuda")
    q[0, -200:] = -2.0
    q[0, 7] = -3.0
    none = torch.empty(1, N, 0, device="cuda")
    oq, ok = ops.qk_norm_rotate(q, q, None, None, none, none, eps=0.0)
    assert torch.equal(oq, q.sign()) and torch.equal(ok, oq)
    del ok, oq
    w = torch.ones(1, device="cuda")
    g = torch.zeros_like(q)
    g[0, -1000:] = 1.0  # 800 rows of +1, 200 of -1, each to 2^-21
    dq, dk, dwq, dwk = ops.qk_norm_rotate_backward(q, q, w, w, none, none, g, g, eps=0.0)
    assert abs(dwq.item() - 600) < 1e-2 and abs(dwk.item() - 600) < 1e-2
    assert dq.abs().max() < 2.0 ** -20 and dk.abs().max() < 2.0 ** -20  # lengths do not matter


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def attention_case(ops, B, Nq, Nk, H, Hk, d, dtype, peers="all", lens=None, starts=None,
                   seen=None, shift=0, seed=0, spoil=False, scale=None, shared_mask=False,
                   size=1.0, broadcast=False):
    g = torch.Generator().manual_seed(seed + 31 * Nq + Nk + d)
    if Nq == Nk:
        q, k, v = rows(g, B, Nq, (H, Hk, Hk), d, dtype, shift)
    else:
        q, = rows(g, B, Nq, (H,), d, dtype, shift)
        k, v = rows(g, B, Nk, (Hk, Hk), d, dtype, shift)
    if size != 1.0:
        q = q * size
    dout, = rows(g, B, Nq, (H,), d, dtype, shift)
    if broadcast:  # one history for all episodes, one gradient for all rows
        k, v = (t[:1].expand(B, -1, -1, -1) for t in (k, v))
        dout = dout[:1, :1].expand(B, Nq, -1, -1)
    key_len = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    q_start = None if starts is None else torch.tensor(starts, dtype=torch.int32)
    visible = None
    if seen is not None:
        visible = torch.rand(1 if shared_mask else B, Nq, Nk, generator=g) < seen
        visible[:, ::5] = False
    if spoil:  # what lies beyond key_len is never read
        for b, n in enumerate(lens):
            k[b, max(0, n):] = float("nan")
            v[b, max(0, n):] = float("inf")
    how = dict(peers=peers, key_len=None if key_len is None else key_len.cuda(),
               q_start=None if q_start is None else q_start.cuda(),
               visible=None if visible is None else visible.cuda(), scale=scale)
    out, lse = ops.head_attention(q, k, v, return_lse=True, **how)
    grads = ops.head_attention_backward(q, k, v, out, lse, dout, **how)
    out2, lse2 = ops.head_attention(q, k, v, return_lse=True, **how)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    for a, b in zip(grads, ops.head_attention_backward(q, k, v, out, lse, dout, **how)):
        assert torch.equal(a, b)  # no order left to chance
    m = h64.mask(B, Nq, Nk, peers, key_len, q_start, visible)
    qd, kd, vd, gd = wide(q, k, v, dout)
    kd, vd = kd.nan_to_num(0, 0, 0), vd.nan_to_num(0, 0, 0)
    ref = h64.Attention(qd, kd, vd, m, 1 / d ** 0.5 if scale is None else scale, gd)
    top = float(ref.abs_scores.max()) if ref.abs_scores.numel() else 0.0
    eps = 2 * (d / 8 + 8) * 2.0 ** -23 * top + (max(Nk, Nq * (H // Hk)) / 32 + 16) * 2.0 ** -22
    rnd = 2.0 ** -8 if dtype == BF16 else 0.0
    tiny = 1e-30
    near(out, ref.out, eps * ref.out_mag + rnd * (ref.out_mag + ref.out.abs()) + tiny)
    dead = torch.isinf(ref.lse)
    assert torch.equal(torch.isinf(lse.cpu()), dead)
    near(lse[~dead.cuda()], ref.lse[~dead], eps * (1 + top) + 2.0 ** -22 * ref.lse[~dead].abs())
    near(grads[0], ref.dq, eps * ref.dq_mag + rnd * (ref.dq_rnd + ref.dq.abs()) + tiny)
    near(grads[1], ref.dk, eps * ref.dk_mag + rnd * (ref.dk_rnd + ref.dk.abs()) + tiny)
    near(grads[2], ref.dv, eps * ref.dv_mag + rnd * (ref.dv_mag + ref.dv.abs()) + tiny)
    return out, lse, grads


SHAPES = [  # B, Nq, Nk, H, Hk, d
    (3, 6, 6, 4, 4, 16),
    (2, 1, 1, 2, 1, 32),
    (2, 65, 65, 4, 2, 64),
    (1, 130, 130, 6, 3, 80),
    (1, 200, 200, 2, 2, 128),
    (2, 3, 150, 8, 2, 64),
    (2, 150, 3, 3, 3, 24),
    (2, 70, 90, 5, 1, 96),
    (2, 33, 70, 4, 2, 64),
    (1, 300, 3, 3, 3, 64),
    (2, 200, 200, 4, 2, 16),
    (1, 210, 40, 2, 1, 24),
    (1, 40, 210, 2, 2, 8),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("peers", ["all", "others", "past"])
@pytest.mark.parametrize("B,Nq,Nk,H,Hk,d", SHAPES)
def test_attention_peers(ops, B, Nq, Nk, H, Hk, d, peers, dtype):
    attention_case(ops, B, Nq, Nk, H, Hk, d, dtype, peers)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("peers", ["all", "others", "past"])
@pytest.mark.parametrize("Nq,Nk,d", [(40, 40, 16), (129, 129, 64), (5, 300, 32), (257, 257, 128)])
def test_attention_lengths_and_sight(ops, Nq, Nk, d, peers, dtype):
    """Lengths of zero, one and beyond Nk, starts before the first key and
    past the last, rows that see nothing."""
    attention_case(ops, 5, Nq, Nk, 4, 2, d, dtype, peers, lens=[0, 1, Nk, Nk + 9, Nk // 2],
                   starts=[0, -3, Nk - 1, 1 - Nq, Nk // 3], seen=0.5, spoil=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [1, 3, 8, 17, 40, 72, 100, 127])
def test_attention_widths(ops, d, dtype):
    attention_case(ops, 2, 67, 67, 2, 1, d, dtype, "others")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [1, 2, 4, 8])
def test_attention_off_the_grid(ops, shift, dtype):
    """Rows that start off the 16-byte grid, a mask shared by all episodes."""
    attention_case(ops, 2, 70, 70, 4, 2, 64, dtype, "past", seen=0.6, shift=shift,
                   shared_mask=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,Nq,Nk,H,Hk,d,lens", [
    (1, 1, 3000, 4, 1, 64, None), (2, 2, 2049, 6, 2, 128, [2049, 700]),
    (3, 1, 5000, 8, 8, 16, [1, 0, 4999]), (1, 40, 1500, 2, 2, 32, None)])
def test_attention_long_history(ops, B, Nq, Nk, H, Hk, d, lens, dtype):
    """Few rows: the key axis is split and joined."""
    if Nq * H // Hk <= 64:
        assert ops._attention_work(B, Nq, Nk, H, Hk, d) > 0
    attention_case(ops, B, Nq, Nk, H, Hk, d, dtype, "past", lens=lens, seen=0.8,
                   starts=None if lens is None else [n - Nq for n in lens])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_broadcast_inputs(ops, dtype):
    attention_case(ops, 3, 150, 150, 4, 2, 64, dtype, "others", broadcast=True)
    attention_case(ops, 3, 2, 700, 4, 2, 128, dtype, "all", broadcast=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_large_scores(ops, dtype):
    """Scores far apart: the running maximum moves and old sums shrink to
    nothing."""
    attention_case(ops, 2, 200, 200, 2, 2, 64, dtype, "all", scale=2.0, size=4.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,N,H,Hk,d,peers,lens,seen", [
    (1, 700, 2, 2, 64, "past", None, None),
    (2, 513, 4, 1, 128, "others", [513, 259], None),
    (1, 640, 2, 1, 64, "all", None, 0.5),
    (2, 385, 3, 3, 96, "past", [385, 128], 0.4),
    (3, 512, 2, 2, 32, "others", None, 0.9)])
def test_attention_many_tiles(ops, B, N, H, Hk, d, peers, lens, seen, dtype):
    attention_case(ops, B, N, N, H, Hk, d, dtype, peers, lens=lens, seen=seen)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_gradient_by_parts(ops, dtype):
    """out and lse of the whole softmax with a part of its keys: that part's
    share of the gradients."""
    B, N, H, Hk, d, cut = 2, 200, 4, 2, 64, 72
    g = torch.Generator().manual_seed(5)
    q, k, v = rows(g, B, N, (H, Hk, Hk), d, dtype)
    dout, = rows(g, B, N, (H,), d, dtype)
    out, lse = ops.head_attention(q, k, v, "past", return_lse=True)
    parts = []
    for a, b in ((0, cut), (cut, N)):
        first = torch.full((B,), -a, dtype=torch.int32, device="cuda")
        parts.append(wide(*ops.head_attention_backward(
            q, k[:, a:b], v[:, a:b], out, lse, dout, "past", q_start=first)))
    qd, kd, vd, gd = wide(q, k, v, dout)
    ref = h64.Attention(qd, kd, vd, h64.mask(B, N, N, "past", None, None, None), d ** -0.5, gd)
    eps = 2 * (d / 8 + 8) * 2.0 ** -23 * float(ref.abs_scores.max()) \
        + (N * (H // Hk) / 32 + 16) * 2.0 ** -22
    rnd = 2.0 ** -8 if dtype == BF16 else 0.0
    # a part's dq is at most dq_mag, and is rounded by itself
    near(parts[0][0] + parts[1][0], ref.dq, eps * ref.dq_mag + rnd * (ref.dq_rnd + ref.dq_mag))
    near(torch.cat([x[1] for x in parts], 1), ref.dk,
         eps * ref.dk_mag + rnd * (ref.dk_rnd + ref.dk.abs()))
    near(torch.cat([x[2] for x in parts], 1), ref.dv,
         eps * ref.dv_mag + rnd * (ref.dv_mag + ref.dv.abs()))


def test_attention_empty_sizes(ops):
    def t(*s):
        return torch.zeros(*s, device="cuda")
    out, lse = ops.head_attention(t(2, 3, 4, 16), t(2, 0, 2, 16), t(2, 0, 2, 16), return_lse=True)
    assert (out == 0).all() and torch.isinf(lse).all()
    dq, dk, dv = ops.head_attention_backward(t(2, 3, 4, 16), t(2, 0, 2, 16), t(2, 0, 2, 16), out,
                                             lse, out)
    assert (dq == 0).all() and dk.numel() == 0
    out, lse = ops.head_attention(t(2, 0, 4, 16), t(2, 3, 2, 16), t(2, 3, 2, 16), return_lse=True)
    dq, dk, dv = ops.head_attention_backward(t(2, 0, 4, 16), t(2, 3, 2, 16), t(2, 3, 2, 16), out,
                                             lse, out)
    assert out.numel() == 0 and (dk == 0).all() and (dv == 0).all()
    assert ops.head_attention(t(0, 3, 4, 16), t(0, 3, 2, 16), t(0, 3, 2, 16)).numel() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_gradient_against_differences(ops, dtype):
    """Slopes of the kernel's own fp32 forward pass along random directions.
    Step h: truncation about h^2 of the slope's scale, rounding 2^-20 / h of
    the loss's: both below 2 % of |g| |u| / sqrt(n) at h = 1/32."""
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(2, 50, 2, 32, generator=g).cuda() for _ in range(3))
    dout = torch.randn(2, 50, 2, 32, generator=g).cuda()
    t = [x.to(dtype) for x in (q, k, v, dout)]
    out, lse = ops.head_attention(*t[:3], "past", return_lse=True)
    grads = ops.head_attention_backward(*t[:3], out, lse, t[3], "past")
    base = [x.float() for x in t[:3]]
    h = 1.0 / 32

    def loss(x):
        return float((ops.head_attention(*x, "past").double() * t[3].double()).sum())

    for i in range(3):
        u = torch.randn(base[i].shape, generator=g).cuda()
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + h * u, base[i] - h * u
        slope = (loss(up) - loss(dn)) / (2 * h)
        gi = grads[i].double()
        size = float(gi.norm() * u.double().norm()) / gi.numel() ** 0.5
        assert abs(slope - float((gi * u.double()).sum())) <= 0.02 * size * 3


def test_attention_offsets_past_32_bits(ops):
    """Episodes more than 2^31 elements apart."""
    N, H, d, far = 70, 2, 64, 2 ** 31 + 64
    room = torch.empty(far + N * 3 * H * d, dtype=BF16, device="cuda")
    x = room.as_strided((2, N, 3 * H * d), (far, 3 * H * d, 1))
    g = torch.Generator().manual_seed(2)
    small = torch.randn(2, N, 3 * H * d, generator=g).to(BF16).cuda()
    x.copy_(small)
    big = [p.unflatten(-1, (H, d)) for p in x.chunk(3, -1)]
    ref = [p.unflatten(-1, (H, d)) for p in small.chunk(3, -1)]
    out, lse = ops.head_attention(*big, "others", return_lse=True)
    want, wlse = ops.head_attention(*ref, "others", return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    for a, b in zip(ops.head_attention_backward(*big, out, lse, want, "others"),
                    ops.head_attention_backward(*ref, want, wlse, want, "others")):
        assert torch.equal(a, b)
    cos, sin = torch.rand(2, 2, N, d // 2, generator=g).cuda()
    for a, b in zip(ops.qk_norm_rotate(big[0], big[1], None, None, cos, sin),
                    ops.qk_norm_rotate(ref[0], ref[1], None, None, cos, sin)):
        assert torch.equal(a, b)


def test_operators_on_another_stream(ops):
    g = torch.Generator().manual_seed(9)
    q, k, v = rows(g, 2, 130, (4, 2, 2), 64, BF16)
    seen = (torch.rand(2, 130, 130, generator=g) < 0.5).cuda()
    want, wlse = ops.head_attention(q, k, v, visible=seen, return_lse=True)
    wgrad = ops.head_attention_backward(q, k, v, want, wlse, want, visible=seen)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out, lse = ops.head_attention(q, k, v, visible=seen, return_lse=True)
        grad = ops.head_attention_backward(q, k, v, out, lse, out, visible=seen)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    for a, b in zip(grad, wgrad):
        assert torch.equal(a, b)


@pytest.mark.parametrize("B,Nq,Nk,shift", [(2, 5, 64, 0), (1, 33, 100, 0), (3, 7, 1, 0),
                                           (2, 4, 96, 5), (1, 3, 4111, 1)])
def test_pack_visibility(ops, B, Nq, Nk, shift):
    g = torch.Generator().manual_seed(Nk)
    seen = (torch.rand(B, Nq, Nk + shift, generator=g) < 0.5).cuda()[..., shift:]
    words = ops.pack_visibility(seen).cpu().long() & 0xffffffff
    assert words.shape == (B, Nq, (Nk + 31) // 32)
    j = torch.arange(Nk)
    assert torch.equal((words[..., j // 32] >> (j % 32)) & 1 == 1, seen.cpu())


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------

def test_refusals(ops):
    def t(*s, **kw):
        return torch.zeros(*s, device="cuda", **kw)
    q, k = t(2, 5, 4, 16), t(2, 5, 2, 16)
    cos = t(1, 5, 8)
    with pytest.raises(RuntimeError):
        ops.head_attention(q.cpu(), k.cpu(), k.cpu())
    with pytest.raises(TypeError):
        ops.head_attention(q.half(), k.half(), k.half())
    with pytest.raises(TypeError):
        ops.head_attention(q, k.bfloat16(), k)
    with pytest.raises(ValueError):
        ops.head_attention(q, k, t(2, 6, 2, 16))
    with pytest.raises(ValueError):
        ops.head_attention(q, t(2, 5, 3, 16), t(2, 5, 3, 16))
    with pytest.raises(ValueError):
        ops.head_attention(q, k, k, peers="left")
    with pytest.raises(ValueError):
        ops.head_attention(q, k, k, key_len=t(3, dtype=torch.int32))
    with pytest.raises(TypeError):
        ops.head_attention(q, k, k, key_len=t(2))
    with pytest.raises(ValueError):
        ops.head_attention(q, k, k, visible=t(2, 5, 6, dtype=torch.bool))
    with pytest.raises(TypeError):
        ops.head_attention(q, k, k, visible=t(2, 5, 1))
    with pytest.raises(ValueError):
        ops.head_attention(q, k, k, visible=torch.zeros(2, 5, 5, dtype=torch.bool))
    wide_ = t(2, 5, 4, 129)
    with pytest.raises(RuntimeError, match="outside the supported range"):
        ops.head_attention(wide_, wide_, wide_)
    with pytest.raises(RuntimeError, match="outside the supported range"):
        ops.head_attention(q, k, k, scale=-1.0)
    out, lse = ops.head_attention(q, k, k, return_lse=True)
    with pytest.raises(ValueError):
        ops.head_attention_backward(q, k, k, out, lse[:, :3], out)
    with pytest.raises(ValueError):
        ops.head_attention_backward(q, k, k, out, lse, out[:, :4])
    with pytest.raises(ValueError):
        ops.qk_norm_rotate(q, k, t(15), None, cos, cos)
    with pytest.raises(ValueError):
        ops.qk_norm_rotate(q, k, None, None, t(1, 4, 8), t(1, 4, 8))
    with pytest.raises(ValueError):
        ops.qk_norm_rotate(q, k, None, None, t(1, 5, 9), t(1, 5, 9))
    with pytest.raises(TypeError):
        ops.qk_norm_rotate(q, k, None, None, cos.double(), cos.double())
    with pytest.raises(ValueError):
        ops.qk_norm_rotate(q, t(2, 4, 2, 16), None, None, cos, cos)
    with pytest.raises(TypeError):
        ops.pack_visibility(t(2, 5, 5))
