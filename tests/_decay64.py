"""Plain 64-bit forms of attention with a decay for each head and of the norms
around a block, for the tests: the definitions of include/tarmac_b200.h, row by
row and differentiable."""

from __future__ import annotations

import torch


def share(x, H):
    """Heads [.., Hk, ..] of dimension 2 repeated to H."""
    return x if x.shape[2] == H else x.repeat_interleave(H // x.shape[2], 2)


def decay(q, k, v, log_decay, scale, state=None, lens=None):
    """(out, state) of float64 tensors; padding is replaced before it is used."""
    B, N, H, d = q.shape
    if lens is None:
        lens = torch.full((B,), N)
    live = torch.arange(N) < lens.long().clamp(0, N)[:, None]
    q, k, v = (torch.where(live[:, :, None, None], t, 0.0) for t in (q, k, v))
    k, v = share(k, H), share(v, H)
    lam = torch.exp(log_decay.double())[:, None, None]
    S = torch.zeros(B, H, d, d, dtype=torch.float64) if state is None else state
    outs = []
    for t in range(N):
        new = lam * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        S = torch.where(live[:, t, None, None, None], new, S)
        outs.append(scale * (q[:, t, :, :, None] * S).sum(-2))
    out = torch.stack(outs, 1) if N else torch.zeros(B, 0, H, d, dtype=torch.float64)
    return torch.where(live[:, :, None, None], out, 0.0), S


def decay_grads(q, k, v, log_decay, scale, dout, state=None, lens=None, dstate=None):
    """(out, state, dq, dk, dv, dS): the formula's, backwards row by row."""
    B, N, H, d = q.shape
    Hk = k.shape[2]
    if lens is None:
        lens = torch.full((B,), N)
    live = torch.arange(N) < lens.long().clamp(0, N)[:, None]
    q, k, v, dout = (torch.where(live[:, :, None, None], t, 0.0) for t in (q, k, v, dout))
    kk, vv = share(k, H), share(v, H)
    lam = torch.exp(log_decay.double())[:, None, None]
    S = torch.zeros(B, H, d, d, dtype=torch.float64) if state is None else state
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    for t in range(N):
        new = lam * S + kk[:, t, :, :, None] * vv[:, t, :, None, :]
        S = torch.where(live[:, t, None, None, None], new, S)
        out[:, t] = scale * (q[:, t, :, :, None] * S).sum(-2)
        dq[:, t] = scale * (dout[:, t, :, None, :] * S).sum(-1)
    R = torch.zeros_like(S) if dstate is None else dstate
    dk, dv = torch.zeros_like(kk), torch.zeros_like(vv)
    for t in range(N - 1, -1, -1):
        R = R + scale * q[:, t, :, :, None] * dout[:, t, :, None, :]
        dk[:, t] = (R * vv[:, t, :, None, :]).sum(-1)
        dv[:, t] = (R * kk[:, t, :, :, None]).sum(-2)
        R = torch.where(live[:, t, None, None, None], lam * R, R)
    m = live[:, :, None, None]
    dk, dv = (x.unflatten(2, (Hk, H // Hk)).sum(3) for x in (dk, dv))
    return (torch.where(m, out, 0.0), S, torch.where(m, dq, 0.0), torch.where(m, dk, 0.0),
            torch.where(m, dv, 0.0), R)


def norm(x, y, w_post, w_pre, gate, scale, eps):
    """(h, z), float64."""
    u = y / (y.square().mean(-1, keepdim=True) + eps).sqrt()
    if w_post is not None:
        u = u * w_post
    if gate is not None:
        u = u * torch.sigmoid(gate)
    if scale is not None:
        u = u * scale
    h = x + u
    z = h / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    return h, z if w_pre is None else z * w_pre


def norm_grads(x, y, w_post, w_pre, gate, scale, dh, dz, eps):
    """(dx, dy, dw_post, dw_pre, dgate, dscale) by the formula."""
    one = torch.ones(x.shape[-1], dtype=torch.float64)
    wo, wi, sc = (one if w is None else w for w in (w_post, w_pre, scale))
    s = torch.ones_like(x) if gate is None else torch.sigmoid(gate)
    ry = 1.0 / (y.square().mean(-1, keepdim=True) + eps).sqrt()
    yn = y * ry
    u = yn * wo
    h = x + sc * s * u
    rh = 1.0 / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    hn = h * rh
    a = dz * wi
    e = dh + rh * (a - hn * (a * hn).mean(-1, keepdim=True))
    b = e * sc * s
    def rows(t):  # sum over all rows
        return t.reshape(-1, t.shape[-1]).sum(0)

    c = wo * b
    dy = ry * (c - yn * (c * yn).mean(-1, keepdim=True))
    return (e, dy, rows(b * yn), rows(dz * hn), e * sc * u * s * (1 - s), rows(e * s * u))
