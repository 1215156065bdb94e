"""Plain 64-bit forms of the multi-head operators, for the tests: the
definitions of include/tarmac_b200.h written out with dense matrices."""

from __future__ import annotations

import torch


def rotate(x, w, cos, sin, eps, interleaved):
    """Head norm and rotation of x [B, N, h, d] (float64)."""
    z = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        z = z * w
    half = cos.shape[-1]
    if half == 0:
        return z
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cos[:, :, None], sin[:, :, None]
    y = z.clone()
    y[..., a] = z[..., a] * c - z[..., b] * s
    y[..., b] = z[..., a] * s + z[..., b] * c
    return y


def rotate_grad(x, w, cos, sin, eps, interleaved, dy):
    """(dx, dw) by the formula: dz = R^T dy, dx = s (g - x s^2 mean(g x))."""
    s = 1.0 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    half = cos.shape[-1]
    dz = dy.clone()
    if half:
        i = torch.arange(half)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, sn = cos[:, :, None], sin[:, :, None]
        dz[..., a] = dy[..., a] * c + dy[..., b] * sn
        dz[..., b] = dy[..., b] * c - dy[..., a] * sn
    dw = (dz * x * s).sum((0, 1, 2))
    g = dz if w is None else dz * w
    return s * (g - x * s * s * (g * x).mean(-1, keepdim=True)), dw


def mask(B, Nq, Nk, peers, key_len=None, q_start=None, visible=None):
    """[B, Nq, Nk] truth values."""
    j = torch.arange(Nk)[None, None]
    start = torch.full((B,), Nk - Nq) if q_start is None else q_start.long()
    pos = start[:, None, None] + torch.arange(Nq)[None, :, None]
    m = torch.ones(B, Nq, Nk, dtype=torch.bool)
    if peers == "others":
        m &= j != pos
    elif peers == "past":
        m &= j <= pos
    if key_len is not None:
        m &= j < key_len.long()[:, None, None]
    if visible is not None:
        m &= visible
    return m


class Attention:
    """out, lse and, given dout, the gradients; float64, [B, N, h, d]."""

    def __init__(self, q, k, v, m, scale, dout=None):
        B, Nq, H, d = q.shape
        G = H // k.shape[2]
        kk = k.repeat_interleave(G, 2).permute(0, 2, 1, 3)
        vv = v.repeat_interleave(G, 2).permute(0, 2, 1, 3)
        qq = q.permute(0, 2, 1, 3)
        m = m[:, None]
        kk = torch.where(m.any(2)[..., None], kk, 0.0)  # keys nobody sees
        vv = torch.where(m.any(2)[..., None], vv, 0.0)
        s = (qq @ kk.transpose(-1, -2) * scale).masked_fill(~m, float("-inf"))
        self.lse = torch.logsumexp(s, -1) if s.shape[-1] else torch.full(
            s.shape[:-1], float("-inf"), dtype=s.dtype)
        p = torch.exp(s - self.lse.clamp_min(-1e300)[..., None])
        self.p, self.abs_scores = p, qq.abs() @ kk.abs().transpose(-1, -2) * scale
        o = p @ vv
        self.out = o.permute(0, 2, 1, 3)
        self.out_mag = (p @ vv.abs()).permute(0, 2, 1, 3)
        if dout is None:
            return
        g = dout.permute(0, 2, 1, 3)

        def shared(x):  # sum over the query heads of a key head
            return x.unflatten(1, (-1, G)).sum(2).permute(0, 2, 1, 3)

        D = (g * o).sum(-1, keepdim=True)
        ds = p * (g @ vv.transpose(-1, -2) - D)
        self.dq = (ds @ kk * scale).permute(0, 2, 1, 3)
        self.dk = shared(ds.transpose(-1, -2) @ qq * scale)
        self.dv = shared(p.transpose(-1, -2) @ g)
        # magnitudes that roundings are relative to
        ds_mag = p * (g.abs() @ vv.abs().transpose(-1, -2) +
                      (g.abs() * o.abs()).sum(-1, keepdim=True))
        # what a bf16 path rounds: dS itself, and out inside D
        ds_rnd = ds.abs() + p * (g.abs() * o.abs()).sum(-1, keepdim=True)

        def spread(x):
            return ((x @ kk.abs() * scale).permute(0, 2, 1, 3),
                    shared(x.transpose(-1, -2) @ qq.abs() * scale))

        self.dq_mag, self.dk_mag = spread(ds_mag)
        self.dq_rnd, self.dk_rnd = spread(ds_rnd)
        self.dv_mag = shared(p.transpose(-1, -2) @ g.abs())
