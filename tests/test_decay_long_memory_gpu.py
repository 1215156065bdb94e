"""Attention with a decay whose heads keep thousands of rows: a decay rounded to
fp32 and applied again and again must not add its rounding up.

Heads keep about T rows and read T rows. A factor off by e in each of T / n
places is off by e m at an age of m places, and the state by 0.43 T / n e of its
norm (the root mean square of an age under weights exp(-a / T) over [0, T]). The
rates are those around -1 / T whose l^n is farthest from an fp32 number,
e close to 2^-25. What remains is the rounding of the sums: one of the state a
place leaves sqrt(0.34 T / n) of at most 2^-24 / sqrt(3) (a uniform rounding's root
mean square, at the mantissa where it is largest) of the norm."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def closed(k, v, rate, start=None, scale=1.0):
    """l^N start + scale sum_t l^(N - 1 - t) k_t v_t^T in float64, [B, H, d, d]."""
    N, H, d = k.shape[1], rate.shape[0], k.shape[3]
    age = torch.arange(N - 1, -1, -1, device=k.device, dtype=torch.float64)[:, None]
    w = torch.exp(rate.double() * age)[None, :, :, None] * scale  # [1, N, H, 1]
    heads = []
    for h in range(H):
        a, b = (t[:, :, h * t.shape[2] // H].double() for t in (k, v))
        heads.append((a * w[:, :, h]).transpose(1, 2) @ b)
    S = torch.stack(heads, 1)
    if start is not None:
        S = S + torch.exp(rate.double() * N)[:, None, None] * start.double()
    return S


def first_state(q, dout, rate, dstate, scale):
    """The gradient of the state before the first row: l R_0."""
    lam = torch.exp(rate.double())[:, None, None]
    return lam * closed(q.flip(1), dout.flip(1), rate, dstate / lam, scale)


def off(got, want):
    """The largest distance of a head, of its norm."""
    return ((got.double() - want).flatten(2).norm(dim=2) / want.flatten(2).norm(dim=2)).max()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 8])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
def test_steps_in_place(d, rows, dtype):
    """600 rows in calls of one or eight over a state renewed in place. A row
    rounds the state twice: sqrt(2 0.34 600) 2^-24 / sqrt(3) = 7e-7, bound 1e-6; a
    decay off in every row would leave 0.43 600 2^-25 = 7.7e-6."""
    from tarmac_b200 import ops
    B, T = 3, 600
    keep = torch.tensor([532.0, 516.0, 585.0, 483.0, 522.0, 716.0])
    rate, H = (-1.0 / keep).cuda(), 6
    g = torch.Generator(device="cuda").manual_seed(d + rows)
    q, k, v = (torch.randn(B, T, H, d, generator=g, device="cuda").to(dtype) for _ in range(3))
    S = torch.randn(B, H, d, d, generator=g, device="cuda")
    want = closed(k, v, rate, S)
    for t in range(0, T, rows):
        ops.decay_attention(*(x[:, t:t + rows] for x in (q, k, v)), rate, S, state_out=S)
    assert off(S, want) <= 1e-6


def both_states(B, N, H, Hk, d, dtype, keep, kernel, segments, tol, expand):
    """The state after the last row and the gradient of the first."""
    from tarmac_b200 import ops
    for backward in (False, True):
        plan = ops.decay_attention_plan(B, N, H, Hk, d, dtype, state=True, backward=backward)
        assert plan["kernel"] == kernel
        assert segments[0] <= plan["segments"] <= segments[1]
    rate = (-1.0 / torch.tensor(keep)).cuda()
    g = torch.Generator(device="cuda").manual_seed(N + d)
    b = 1 if expand else B
    q, k, v, dout = (torch.randn(b, N, h, d, generator=g, device="cuda").to(dtype)
                     .expand(B, -1, -1, -1) for h in (H, Hk, Hk, H))
    S, dS = (torch.randn(b, H, d, d, generator=g, device="cuda").expand(B, -1, -1, -1)
             for _ in range(2))
    last = ops.decay_attention(q, k, v, rate, S, return_state=True)[1]
    first = ops.decay_attention_backward(q, k, v, rate, dout, S, dS)[3]
    some = [0, B - 1] if B > 1 else [0]
    q, k, v, dout, S, dS = (t[some] for t in (q, k, v, dout, S, dS))
    assert off(last[some], closed(k, v, rate, S)) <= tol
    assert off(first[some], first_state(q, dout, rate, dS, d ** -0.5)) <= tol


@pytest.mark.parametrize("B,d", [(1480, 8), (592, 24), (222, 40), (74, 72)])
def test_one_walk(B, d):
    """fp32 rows one after the other, 16384 of them. One rounding of the state a
    row: sqrt(0.34 16384) 2^-24 / sqrt(3) = 2.6e-6, 16 rows by themselves 2.4e-7:
    bound 3e-6. Off once in 16 rows: 0.43 1024 2^-25 = 1.3e-5."""
    both_states(B, 16384, 2, 2, d, F32, [16384.0, 15794.0], "decay_scan", (1, 1), 3e-6, True)


@pytest.mark.parametrize("H,d,keep", [
    (8, 16, [57737.0, 66781.0, 63963.0, 71565.0, 72941.0, 58589.0, 65536.0, 60000.0]),
    (1, 40, [66781.0])])
def test_many_segments(H, d, keep):
    """fp32 rows in 683 segments of 96 or 820 of 80. A segment's rows: weights off
    by up to 96 2^-25 / 2, as a random walk sqrt(96) 2^-24 / sqrt(3) = 3.4e-7; a rounding
    where segments are joined: sqrt(0.34 820) 2^-24 / sqrt(3) = 5.7e-7; bound 1.5e-6. Off
    in every segment: 0.43 683 2^-25 = 8.7e-6."""
    both_states(1, 65536, H, H, d, F32, keep, "decay_scan", (600, 900), 1.5e-6, False)


@pytest.mark.parametrize("B,N,H,Hk,d,keep", [
    (37, 65536, 8, 8, 16, [66780.0, 76152.0, 57800.0, 77396.0, 55900.0, 71496.0, 65536.0, 60000.0]),
    (18, 32768, 8, 1, 72, [33390.0, 38076.0, 28900.0, 38698.0, 27950.0, 35748.0, 32768.0, 30000.0])])
def test_many_chunks(B, N, H, Hk, d, keep):
    """bf16 rows, chunks of 128 on the tensor memory. A weight is off by 2^-22 (the
    exponential) and no more for what follows; a chunk's product sums 24 steps,
    truncated: 24 2^-23 2/3 of it, 1.9e-6, all toward zero; a rounding of the state a
    chunk: sqrt(0.34 512) 2^-24 / sqrt(3) = 4.6e-7: bound 2.6e-6. Off in every chunk by
    2^-25: 0.43 512 2^-25 = 6.6e-6, by the exponential's 2^-22 eight times that."""
    both_states(B, N, H, Hk, d, BF16, keep, "decay_tc", (1, 1), 2.6e-6, False)
