"""Communication blocks of several heads: query/key/value projection, head
norms with the position rotation, attention, output projection.

The single-head module (``src.agents.mappo.AttentionComm``) lets every agent
read every other one. This block is for agents with wider messages and a
limited field of view (``visible``), in episodes of unequal size
(``key_len``), or for one agent that reads its own past, step by step
(:meth:`HeadComm.step`). :class:`DecayComm` reads its past through a memory of
fixed size instead, whose cost does not grow with the history, and can be
stacked. They have no counterpart in the reference.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import autograd as tgrad
from . import ops


def rotation_table(pos: torch.Tensor, r: int, base: float = 10000.0):
    """(cos, sin) of the r / 2 angles of each row, fp32 [Bt, N, r / 2], from
    positions [Bt, N] (time steps) or [Bt, N, 2] (places: the first half of
    the angles turns with x, the second with y). Angle i of m turns by
    ``position * base ** (-i / m)``."""
    if r < 0 or r % 2:
        raise ValueError(f"r must be even and not negative; got {r}")
    if pos.dim() == 3 and pos.shape[-1] == 2:
        if r % 4:
            raise ValueError(f"r must be a multiple of 4 for places; got {r}")
        axes = pos.unbind(-1)
    elif pos.dim() == 2:
        axes = (pos,)
    else:
        raise ValueError(f"pos must be [B, N] or [B, N, 2]; got {tuple(pos.shape)}")
    m = r // 2 // len(axes)
    freq = base ** (-torch.arange(m, device=pos.device, dtype=torch.float32) / max(m, 1))
    angle = torch.cat([a.float()[..., None] * freq for a in axes], -1)
    return angle.cos(), angle.sin()


class HeadComm(nn.Module):
    """(B, N, in_dim) -> (B, N, n_heads * head_dim)."""

    def __init__(self, in_dim: int, n_heads: int, head_dim: int,
                 n_kv_heads: int | None = None, eps: float = 1e-6) -> None:
        super().__init__()
        n_kv_heads = n_heads if n_kv_heads is None else n_kv_heads
        if n_kv_heads < 1 or n_heads % n_kv_heads:
            raise ValueError("n_heads must be a multiple of n_kv_heads")
        self.heads = (n_heads, n_kv_heads, n_kv_heads)
        self.head_dim, self.eps = head_dim, eps
        self.qkv = nn.Linear(in_dim, sum(self.heads) * head_dim)
        self.norm_q = nn.Parameter(torch.ones(head_dim))
        self.norm_k = nn.Parameter(torch.ones(head_dim))
        self.proj = nn.Linear(n_heads * head_dim, n_heads * head_dim)

    def _qkv(self, x, cos, sin):
        """Normed, rotated queries and keys, and values: views of one product."""
        d = self.head_dim
        parts = self.qkv(x).split([h * d for h in self.heads], -1)
        q, k, v = (t.unflatten(-1, (h, d)) for t, h in zip(parts, self.heads))
        q, k = tgrad.qk_norm_rotate(q, k, self.norm_q, self.norm_k, cos, sin, self.eps)
        return q, k, v

    def forward(self, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                peers: str = "others", visible: torch.Tensor | None = None,
                key_len: torch.Tensor | None = None) -> torch.Tensor:
        """Messages of a whole set at once. ``cos``, ``sin``: the rows' table
        (:func:`rotation_table`); the masks are those of
        :func:`ops.head_attention`. An agent that sees nobody gets the output
        projection's bias."""
        q, k, v = self._qkv(x, cos, sin)
        out = tgrad.head_attention(q, k, v, peers, key_len, None, visible)
        return self.proj(out.flatten(2))

    @torch.no_grad()
    def step(self, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
             past_k: torch.Tensor, past_v: torch.Tensor,
             past_len: torch.Tensor) -> torch.Tensor:
        """One new row per episode, x [B, 1, in_dim], over each one's past.
        ``past_k``, ``past_v`` [B, room, n_kv_heads, head_dim] hold the first
        ``past_len`` (int32 or int64 [B]) rows; the new keys and values are
        written behind them and ``past_len`` grows by one, in place. The caller
        keeps ``past_len`` below the room: an episode that has none left (or a
        negative length) gets NaN, and its last (or first) row is lost."""
        B, shape = x.shape[0], tuple(past_k.shape)
        if x.dim() != 3 or x.shape[1] != 1:
            raise ValueError(f"x must be [B, 1, in_dim]; got {tuple(x.shape)}")
        if len(shape) != 4 or shape[0] != B or shape[1] < 1 \
                or shape[2:] != (self.heads[1], self.head_dim) or past_v.shape != shape:
            raise ValueError(
                f"past_k and past_v must share one [{B}, room, {self.heads[1]}, "
                f"{self.head_dim}] shape; got {shape}, {tuple(past_v.shape)}")
        if tuple(past_len.shape) != (B,):
            raise ValueError(f"past_len must be [{B}]; got {tuple(past_len.shape)}")
        if past_len.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"past_len must be int32 or int64; got {past_len.dtype}")
        q, k, v = self._qkv(x, cos, sin)
        if q.dtype is not past_k.dtype:
            q, k, v = (t.to(past_k.dtype) for t in (q, k, v))
        n = past_len.view(B, 1, 1, 1)
        at = n.clamp(0, shape[1] - 1)  # never written out of range
        lost = at != n
        row = at.long().expand(k.shape)
        past_k.scatter_(1, row, k)
        past_v.scatter_(1, row, v)
        past_len += 1
        out = ops.head_attention(q, past_k, past_v, "all",
                                 key_len=past_len.to(torch.int32))
        out.masked_fill_(lost, float("nan"))
        return self.proj(out.flatten(2).to(x.dtype))


def decay_slopes(n_heads: int) -> torch.Tensor:
    """log of each head's decay, fp32 [n_heads]: -2 ** (-8 h / n_heads), from
    about half a row's memory to 256 rows'."""
    h = torch.arange(1, n_heads + 1, dtype=torch.float32)
    return -(2.0 ** (-8.0 * h / n_heads))


class DecayComm(nn.Module):
    """One block of a stack over a stream of rows (B, N, dim): attention with a
    decay for each head on the normed rows z, projected, normed, gated and
    added to the stream x, whose norm is the next block's z."""

    def __init__(self, dim: int, n_heads: int, head_dim: int,
                 n_kv_heads: int | None = None, eps: float = 1e-6) -> None:
        super().__init__()
        n_kv_heads = n_heads if n_kv_heads is None else n_kv_heads
        if n_kv_heads < 1 or n_heads % n_kv_heads:
            raise ValueError("n_heads must be a multiple of n_kv_heads")
        self.heads = (n_heads, n_kv_heads, n_kv_heads)
        self.head_dim, self.eps = head_dim, eps
        self.qkv = nn.Linear(dim, sum(self.heads) * head_dim)
        self.gate = nn.Linear(dim, dim)
        self.proj = nn.Linear(n_heads * head_dim, dim)
        self.norm_q = nn.Parameter(torch.ones(head_dim))
        self.norm_k = nn.Parameter(torch.ones(head_dim))
        self.norm_post = nn.Parameter(torch.ones(dim))
        self.norm_next = nn.Parameter(torch.ones(dim))
        self.scale = nn.Parameter(torch.ones(dim))
        self.register_buffer("log_decay", decay_slopes(n_heads))

    def _apply(self, fn, recurse=True):
        """A cast to a shorter type is for the products: the decays, the norms'
        weights and the scale, which the kernels read in fp32, stay in it."""
        own = [t for p in self._parameters.values() for t in (p, p.grad)]
        own += self._buffers.values()

        def keep(t):
            new = fn(t)
            if new.dtype != t.dtype and new.element_size() < 4 \
                    and any(t is o for o in own):
                new = t.to(new.device, torch.float32)
            return new

        return super()._apply(keep, recurse)

    def empty_state(self, B: int) -> torch.Tensor:
        """The state before any row, fp32 [B, n_heads, head_dim, head_dim]."""
        return torch.zeros(B, self.heads[0], self.head_dim, self.head_dim,
                           device=self.log_decay.device)

    def _qkv(self, z, cos, sin):
        d = self.head_dim
        parts = self.qkv(z).split([h * d for h in self.heads], -1)
        q, k, v = (t.unflatten(-1, (h, d)) for t, h in zip(parts, self.heads))
        q, k = tgrad.qk_norm_rotate(q, k, self.norm_q, self.norm_k, cos, sin, self.eps)
        return q, k, v

    def _join(self, x, z, out):
        return tgrad.residual_norm(x, self.proj(out.flatten(2)), self.norm_post,
                                   self.norm_next, self.gate(z), self.scale, self.eps)

    def forward(self, x: torch.Tensor, z: torch.Tensor, cos: torch.Tensor,
                sin: torch.Tensor, state: torch.Tensor | None = None,
                lens: torch.Tensor | None = None):
        """The rows of whole episodes at once, from ``state`` (zero when None).
        z: the normed rows, the block's input (the first block's may be x
        itself); ``cos``, ``sin``: the rows' table (:func:`rotation_table`);
        rows from ``lens`` on are padding. Returns the stream, its norm and the
        state after the last row."""
        q, k, v = self._qkv(z, cos, sin)
        out, state = tgrad.decay_attention(q, k, v, self.log_decay, state, lens,
                                           return_state=True)
        return (*self._join(x, z, out), state)

    @torch.no_grad()
    def step(self, x: torch.Tensor, z: torch.Tensor, cos: torch.Tensor,
             sin: torch.Tensor, state: torch.Tensor):
        """One new row per episode (N = 1, or a few), ``state`` renewed in
        place. Returns the stream and its norm."""
        q, k, v = self._qkv(z, cos, sin)
        out, _ = ops.decay_attention(q, k, v, self.log_decay, state, state_out=state)
        return self._join(x, z, out)
