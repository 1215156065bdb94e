"""Differentiable attention-core operations (torch.autograd.Function).

Forward runs the sm_100a kernels of :mod:`tarmac_b200.ops`; backward runs the
gradient kernels (csrc/backward.cu; csrc/head_*.cu for the multi-head
operators) through the same C ABI. The single-head ones give the
gradients autograd forms through the reference's eager path
(src/agents/mappo.py:192-231 topk_gather, 265-292 zorder_k, 361-373 dense):
the peer selection itself carries no gradient. Gradients come back in the
dtype of q.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops


class DenseAttention(torch.autograd.Function):
    """softmax(q k^T * scale, diagonal excluded) v."""

    @staticmethod
    def forward(ctx, q, k, v, scale=None):
        out = ops.dense_attention(q, k, v, scale)
        ctx.save_for_backward(q, k, v, out)
        ctx.scale = scale
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out = ctx.saved_tensors
        dq, dk, dv = ops.dense_attention_backward(q, k, v, out, dout, ctx.scale)
        t = q.dtype
        return dq.to(t), dk.to(t), dv.to(t), None


class TopkAttention(torch.autograd.Function):
    """Fused score-then-select top-k attention (k <= 8; "argmax" keeps the
    lowest index on a tie, "sort" the highest)."""

    @staticmethod
    def forward(ctx, q, k, v, topk, mode="argmax", scale=None):
        if topk > ops.STREAM_MAX_K or mode == "threshold":
            raise NotImplementedError(
                "gradients of top-k attention need k <= 8 and the argmax or "
                "sort tie rule (the retained set must be a list of k peers)")
        out, idx = ops.topk_attention(q, k, v, topk, mode, scale,
                                      return_indices=True)
        ctx.save_for_backward(q, k, v, idx)
        ctx.scale = scale
        ctx.mark_non_differentiable(idx)
        return out, idx

    @staticmethod
    def backward(ctx, dout, _didx):
        q, k, v, idx = ctx.saved_tensors
        dq, dk, dv = ops.gather_attention_backward(q, k, v, dout, idx,
                                                   ctx.scale)
        t = q.dtype
        return dq.to(t), dk.to(t), dv.to(t), None, None, None


class PrescoreAttention(torch.autograd.Function):
    """Attention over the given peers idx ([B, N, kk])."""

    @staticmethod
    def forward(ctx, q, k, v, idx, scale=None):
        out = ops.prescore_attention(q, k, v, idx, scale)
        ctx.save_for_backward(q, k, v, idx)
        ctx.scale = scale
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, idx = ctx.saved_tensors
        dq, dk, dv = ops.gather_attention_backward(q, k, v, dout, idx,
                                                   ctx.scale)
        t = q.dtype
        return dq.to(t), dk.to(t), dv.to(t), None, None


class MortonPrescoreAttention(torch.autograd.Function):
    """Fused Z-order window selection + attention over the selected peers."""

    @staticmethod
    def forward(ctx, q, k, v, pos, topk, bits=10, scale=None):
        out, idx = ops.morton_prescore_attention(q, k, v, pos, topk, bits,
                                                 scale, return_indices=True)
        ctx.save_for_backward(q, k, v, idx)
        ctx.scale = scale
        ctx.mark_non_differentiable(idx)
        return out, idx

    @staticmethod
    def backward(ctx, dout, _didx):
        q, k, v, idx = ctx.saved_tensors
        dq, dk, dv = ops.gather_attention_backward(q, k, v, dout, idx,
                                                   ctx.scale)
        t = q.dtype
        return dq.to(t), dk.to(t), dv.to(t), None, None, None, None


class QkNormRotate(torch.autograd.Function):
    """Head norms and position rotation (:func:`ops.qk_norm_rotate`). The
    tables carry no gradient. First derivatives in reverse mode only: a second
    derivative or a forward-mode tangent is refused."""

    @staticmethod
    def forward(ctx, q, k, wq, wk, cos, sin, eps=1e-6, interleaved=False):
        ctx.save_for_backward(q, k, wq, wk, cos, sin)
        ctx.how = (eps, interleaved)
        return ops.qk_norm_rotate(q, k, wq, wk, cos, sin, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, wq, wk, cos, sin = ctx.saved_tensors
        dq, dk, dwq, dwk = ops.qk_norm_rotate_backward(
            q, k, wq, wk, cos, sin, dq_out, dk_out, *ctx.how)
        if wq is not None:
            dwq = dwq.to(wq.dtype)
        if wk is not None:
            dwk = dwk.to(wk.dtype)
        return dq, dk, dwq, dwk, None, None, None, None


class HeadAttention(torch.autograd.Function):
    """Masked attention with heads (:func:`ops.head_attention`); ``visible``
    is None or the words of :func:`ops.pack_visibility`. First derivatives in
    reverse mode only, as :class:`QkNormRotate`."""

    @staticmethod
    def forward(ctx, q, k, v, peers="all", key_len=None, q_start=None,
                visible=None, scale=None):
        out, lse = ops.head_attention(q, k, v, peers, key_len, q_start,
                                      visible, scale, return_lse=True)
        ctx.save_for_backward(q, k, v, out, lse, key_len, q_start, visible)
        ctx.how = (peers, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, key_len, q_start, visible = ctx.saved_tensors
        peers, scale = ctx.how
        dq, dk, dv = ops.head_attention_backward(
            q, k, v, out, lse, dout, peers, key_len, q_start, visible, scale)
        return dq, dk, dv, None, None, None, None, None


class DecayAttention(torch.autograd.Function):
    """Attention with a decay for each head (:func:`ops.decay_attention`), with
    the state after the last row where ``return_state`` asks for it. The decays
    carry no gradient. First derivatives in reverse mode only, as
    :class:`QkNormRotate`."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, state=None, lens=None, scale=None,
                return_state=True):
        ctx.save_for_backward(q, k, v, log_decay, state, lens)
        ctx.scale = scale
        ctx.set_materialize_grads(False)  # an unused state costs nothing
        return ops.decay_attention(q, k, v, log_decay, state, lens, scale,
                                   return_state=return_state)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dstate=None):
        q, k, v, log_decay, state, lens = ctx.saved_tensors
        if dout is None:
            dout = torch.zeros_like(q)
        dq, dk, dv, first = ops.decay_attention_backward(
            q, k, v, log_decay, dout, state, dstate, lens, ctx.scale,
            need_dstate=ctx.needs_input_grad[4])
        return dq, dk, dv, None, first, None, None, None


class ResidualNorm(torch.autograd.Function):
    """The norms around a block with its gate and residual scale
    (:func:`ops.residual_norm`). First derivatives in reverse mode only, as
    :class:`QkNormRotate`."""

    @staticmethod
    def forward(ctx, x, y, w_post=None, w_pre=None, gate=None, scale=None,
                eps=1e-6):
        ctx.save_for_backward(x, y, w_post, w_pre, gate, scale)
        ctx.eps = eps
        ctx.set_materialize_grads(False)  # an unused z costs nothing
        return ops.residual_norm(x, y, w_post, w_pre, gate, scale, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dz):
        x, y, w_post, w_pre, gate, scale = ctx.saved_tensors
        dx, dy, dwo, dwi, dgate, dsc = ops.residual_norm_backward(
            x, y, w_post, w_pre, gate, scale, dh, dz, ctx.eps)
        dwo, dwi, dsc = (g if g is None else g.to(w.dtype)
                         for g, w in ((dwo, w_post), (dwi, w_pre), (dsc, scale)))
        return dx, dy, dwo, dwi, dgate, dsc, None


def _needs_grad(*ts) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in ts)


# The functions below take the differentiable form only when autograd will
# need it; otherwise they call the forward kernels directly (same results).

def dense_attention(q, k, v, scale=None):
    if _needs_grad(q, k, v):
        return DenseAttention.apply(q, k, v, scale)
    return ops.dense_attention(q, k, v, scale)


def _has_tangent(*ts) -> bool:
    """Does one of these carry a forward-mode tangent? The function's apply
    then refuses it; the plain call would drop it."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(
        forward_ad.unpack_dual(t).tangent is not None for t in ts)


def topk_attention(q, k, v, topk, mode="argmax", scale=None):
    if _needs_grad(q, k, v):
        return TopkAttention.apply(q, k, v, topk, mode, scale)[0]
    return ops.topk_attention(q, k, v, topk, mode, scale)


def prescore_attention(q, k, v, idx, scale=None):
    if _needs_grad(q, k, v):
        return PrescoreAttention.apply(q, k, v, idx, scale)
    return ops.prescore_attention(q, k, v, idx, scale)


def morton_prescore_attention(q, k, v, pos, topk, bits=10, scale=None):
    if _needs_grad(q, k, v):
        return MortonPrescoreAttention.apply(q, k, v, pos, topk, bits,
                                             scale)[0]
    return ops.morton_prescore_attention(q, k, v, pos, topk, bits, scale)


def qk_norm_rotate(q, k, wq, wk, cos, sin, eps=1e-6, interleaved=False):
    ts = [t for t in (q, k, wq, wk) if t is not None]
    if _needs_grad(*ts) or _has_tangent(*ts):
        return QkNormRotate.apply(q, k, wq, wk, cos, sin, eps, interleaved)
    return ops.qk_norm_rotate(q, k, wq, wk, cos, sin, eps, interleaved)


def head_attention(q, k, v, peers="all", key_len=None, q_start=None,
                   visible=None, scale=None):
    if _needs_grad(q, k, v) or _has_tangent(q, k, v):
        if visible is not None and visible.dtype == torch.bool:
            visible = ops.pack_visibility(visible)  # once for both directions
        return HeadAttention.apply(q, k, v, peers, key_len, q_start, visible,
                                   scale)
    return ops.head_attention(q, k, v, peers, key_len, q_start, visible, scale)


def decay_attention(q, k, v, log_decay, state=None, lens=None, scale=None,
                    return_state=False):
    if torch.is_grad_enabled() and log_decay.requires_grad:
        raise ValueError("log_decay has no gradient: pass a tensor that does "
                         "not require one")
    ts = [t for t in (q, k, v, log_decay, state) if t is not None]
    if _needs_grad(*ts) or _has_tangent(*ts):
        return DecayAttention.apply(q, k, v, log_decay, state, lens, scale,
                                    return_state)
    return ops.decay_attention(q, k, v, log_decay, state, lens, scale,
                               return_state)


def residual_norm(x, y, w_post=None, w_pre=None, gate=None, scale=None, eps=1e-6):
    ts = [t for t in (x, y, w_post, w_pre, gate, scale) if t is not None]
    if _needs_grad(*ts) or _has_tangent(*ts):
        return ResidualNorm.apply(x, y, w_post, w_pre, gate, scale, eps)
    return ops.residual_norm(x, y, w_post, w_pre, gate, scale, eps)
