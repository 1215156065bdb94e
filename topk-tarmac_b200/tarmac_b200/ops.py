"""Torch-facing launchers over the C ABI.

Each function takes CUDA tensors, checks them, allocates the output
(``torch.empty_like`` / ``torch.empty``; the C ABI itself never allocates) and
launches on the current stream of the tensors' device. Q, K, V are ``[B, N, d]`` fp32 or bf16 tensors
with a unit innermost stride; other strides (e.g. the ``qkv.chunk(3, -1)``
views of the comm module) are passed through without a copy. Nothing here
computes on the CPU: a CPU tensor or a missing library is an error.

The semantics are those of the reference's eager path
(src/kernels/fused_topk_attention.py:390-402): scores q.k * scale with the
diagonal excluded, softmax over the retained peers, weighted sum of V rows.
"""

from __future__ import annotations

import contextlib
import functools
import struct

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_MODES = {"argmax": _lib.SELECT_ARGMAX, "threshold": _lib.SELECT_THRESHOLD,
          "sort": _lib.SELECT_SORT}

RESIDENT_MAX_N = 1024
STREAM_MAX_K = 8
MORTON_MAX_N = 4096


def default_scale(d: int) -> float:
    """1/sqrt(d), as the reference kernels pass it (fused_topk_attention.py:327)."""
    return 1.0 / (d ** 0.5)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# the raw current-stream handle without building a Stream object (falls back
# to the public call on a torch without the accessor)
_RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_SAME_DEVICE = contextlib.nullcontext()


def _index(dev: torch.device) -> int:
    """The device's ordinal (a bare "cuda" device means the current one)."""
    return torch.cuda.current_device() if dev.index is None else dev.index


def _stream(dev: torch.device) -> int:
    if _RAW_STREAM is not None:
        return _RAW_STREAM(_index(dev))
    return torch.cuda.current_stream(dev).cuda_stream


def _on(dev: torch.device):
    """Device context for a launch: the library launches on the current
    device, so switch only when the tensors live on another one."""
    if dev.index is None or dev.index == torch.cuda.current_device():
        return _SAME_DEVICE
    return torch.cuda.device(dev)


def _unit_inner(t: torch.Tensor) -> torch.Tensor:
    return t if (t.shape[-1] == 1 or t.stride(-1) == 1) else t.contiguous()


def _check_qkv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor):
    if q.dim() != 3 or k.shape != q.shape or v.shape != q.shape:
        raise ValueError(f"q, k, v must share one [B, N, d] shape; got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise RuntimeError("tarmac_b200 kernels need CUDA tensors (there is no "
                           "CPU implementation)")
    if not (q.device == k.device == v.device):
        raise ValueError("q, k, v must be on one device")
    if not (q.dtype == k.dtype == v.dtype) or q.dtype not in _DTYPES:
        raise TypeError(f"q, k, v must all be float32 or bfloat16; got "
                        f"{q.dtype}, {k.dtype}, {v.dtype}")
    return _unit_inner(q), _unit_inner(k), _unit_inner(v)


def _strides(q, k, v, o) -> bytes:
    """Batch and row strides of q, k, v, o as the int64[8] the C ABI reads.
    A bytes object passes as a pointer to its buffer and lives as long as
    the call's arguments; packing costs well under the eight-element ctypes
    array it replaces (host cost per call matters for small problems)."""
    sq, sk, sv, so = q.stride(), k.stride(), v.stride(), o.stride()
    return _PACK8(sq[0], sq[1], sk[0], sk[1], sv[0], sv[1], so[0], so[1])


_PACK8 = struct.Struct("=8q").pack
_CONTIG = torch.contiguous_format


def _empty_as(q: torch.Tensor) -> torch.Tensor:
    """A contiguous output of q's shape, dtype and device."""
    return torch.empty_like(q, memory_format=_CONTIG)


def _scale(d: int, scale: float | None) -> float:
    return default_scale(d) if scale is None else float(scale)


def dense_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    scale: float | None = None) -> torch.Tensor:
    """softmax(q k^T * scale, diagonal excluded) v."""
    q, k, v = _check_qkv(q, k, v)
    B, N, d = q.shape
    out = _empty_as(q)
    if N < 2:
        return out.fill_(float("nan"))
    strides = _strides(q, k, v, out)
    with _on(q.device):
        _lib.call("tarmac_dense_attention", _ptr(q), _ptr(k), _ptr(v),
                  _ptr(out), strides, B, N, d,
                  _DTYPES[q.dtype], _scale(d, scale), _stream(q.device))
    return out


def topk_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                   topk: int, mode: str = "argmax", scale: float | None = None,
                   return_indices: bool = False):
    """Fused score-then-select top-k attention.

    ``mode``: ``"argmax"`` (lowest index wins a tie at the k-th score),
    ``"sort"`` (highest index wins) or ``"threshold"`` (every tied peer kept).
    ``topk`` must already lie in [1, N-1]. With ``return_indices`` also returns
    the retained peers, int32 ``[B, N, topk]`` in rank order (k <= 8,
    argmax/sort only).
    """
    q, k, v = _check_qkv(q, k, v)
    B, N, d = q.shape
    if mode not in _MODES:
        raise ValueError(f"unknown selection mode {mode!r}")
    out = _empty_as(q)
    idx = (torch.empty((B, N, topk), device=q.device, dtype=torch.int32)
           if return_indices else None)
    strides = _strides(q, k, v, out)
    with _on(q.device):
        _lib.call("tarmac_topk_attention", _ptr(q), _ptr(k), _ptr(v),
                  _ptr(out), strides, B, N, d,
                  _DTYPES[q.dtype], _scale(d, scale), int(topk), _MODES[mode],
                  _ptr(idx), _stream(q.device))
    return (out, idx) if return_indices else out


def streaming_topk_attention(q: torch.Tensor, k: torch.Tensor,
                             v: torch.Tensor, topk: int,
                             scale: float | None = None,
                             return_indices: bool = False):
    """Exact top-k (k <= 8, lowest index wins a tie) with keys streamed
    through shared memory; no cap on N."""
    q, k, v = _check_qkv(q, k, v)
    B, N, d = q.shape
    out = _empty_as(q)
    idx = (torch.empty((B, N, topk), device=q.device, dtype=torch.int32)
           if return_indices else None)
    strides = _strides(q, k, v, out)
    with _on(q.device):
        _lib.call("tarmac_streaming_topk_attention", _ptr(q), _ptr(k), _ptr(v),
                  _ptr(out), strides, B, N, d,
                  _DTYPES[q.dtype], _scale(d, scale), int(topk), _ptr(idx),
                  _stream(q.device))
    return (out, idx) if return_indices else out


def prescore_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       idx: torch.Tensor,
                       scale: float | None = None) -> torch.Tensor:
    """Attention over the peers named by ``idx`` ([B, N, kk], int64 or int32).
    Rows naming a peer outside [0, N) come back as NaN."""
    q, k, v = _check_qkv(q, k, v)
    B, N, d = q.shape
    if idx.dim() != 3 or tuple(idx.shape[:2]) != (B, N):
        raise ValueError(f"idx must be [B, N, kk]; got {tuple(idx.shape)}")
    if idx.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"idx must be int64 or int32; got {idx.dtype}")
    if idx.device != q.device:
        raise ValueError("idx must be on the device of q")
    idx = idx.contiguous()
    kk = idx.shape[-1]
    out = _empty_as(q)
    if kk == 0:
        return out.fill_(float("nan"))
    strides = _strides(q, k, v, out)
    with _on(q.device):
        _lib.call("tarmac_prescore_attention", _ptr(q), _ptr(k), _ptr(v),
                  _ptr(out), strides, _ptr(idx),
                  int(idx.dtype == torch.int64), kk, B, N, d,
                  _DTYPES[q.dtype], _scale(d, scale), _stream(q.device))
    return out


def _check_pos(pos: torch.Tensor) -> torch.Tensor:
    if pos.dim() != 3 or pos.shape[-1] != 2:
        raise ValueError(f"pos must be [B, N, 2]; got {tuple(pos.shape)}")
    if not pos.is_cuda:
        raise RuntimeError("tarmac_b200 kernels need CUDA tensors")
    if pos.dtype != torch.float32:
        raise TypeError(f"pos must be float32; got {pos.dtype}")
    return pos.contiguous()


def morton_code(pos: torch.Tensor, bits: int = 10) -> torch.Tensor:
    """Per-episode Morton codes, int64 [B, N]."""
    pos = _check_pos(pos)
    B, N, _ = pos.shape
    out = torch.empty((B, N), device=pos.device, dtype=torch.int64)
    with _on(pos.device):
        _lib.call("tarmac_morton_code", _ptr(pos), B, N, int(bits), _ptr(out),
                  _stream(pos.device))
    return out


def morton_select(pos: torch.Tensor, k: int, bits: int = 10) -> torch.Tensor:
    """Z-order window peers, int64 [B, N, k] (stable order on equal codes)."""
    pos = _check_pos(pos)
    B, N, _ = pos.shape
    out = torch.empty((B, N, k), device=pos.device, dtype=torch.int64)
    with _on(pos.device):
        _lib.call("tarmac_morton_select", _ptr(pos), B, N, int(k), int(bits),
                  _ptr(out), _stream(pos.device))
    return out


def morton_prescore_attention(q: torch.Tensor, k: torch.Tensor,
                              v: torch.Tensor, pos: torch.Tensor, topk: int,
                              bits: int = 10, scale: float | None = None,
                              return_indices: bool = False):
    """Fused Z-order selection + attention over the selected peers."""
    q, k, v = _check_qkv(q, k, v)
    pos = _check_pos(pos)
    B, N, d = q.shape
    if tuple(pos.shape[:2]) != (B, N):
        raise ValueError("pos must be [B, N, 2] matching q")
    out = _empty_as(q)
    idx = (torch.empty((B, N, topk), device=q.device, dtype=torch.int64)
           if return_indices else None)
    strides = _strides(q, k, v, out)
    with _on(q.device):
        _lib.call("tarmac_morton_prescore_attention", _ptr(q), _ptr(k),
                  _ptr(v), _ptr(out), strides, _ptr(pos),
                  B, N, d, _DTYPES[q.dtype], _scale(d, scale), int(topk),
                  int(bits), _ptr(idx), _stream(q.device))
    return (out, idx) if return_indices else out


# ---------------------------------------------------------------------------
# gradients (training path)
# ---------------------------------------------------------------------------

def _strides_n(*ts) -> bytes:
    vals = []
    for t in ts:
        st = t.stride()
        vals += [st[0], st[1]]
    return struct.pack(f"={len(vals)}q", *vals)


def gather_attention_backward(q: torch.Tensor, k: torch.Tensor,
                              v: torch.Tensor, dout: torch.Tensor,
                              idx: torch.Tensor, scale: float | None = None):
    """Gradients (dq, dk, dv), fp32 [B, N, d], of attention over the fixed
    peer set ``idx`` ([B, N, kk], int32 or int64): the peers a top-k call
    retained, the Morton window, or given indices. The selection carries no
    gradient. dk and dv accumulate with atomic adds (summation order not
    fixed)."""
    q, k, v = _check_qkv(q, k, v)
    dout = _unit_inner(dout)
    B, N, d = q.shape
    if dout.shape != q.shape or dout.device != q.device:
        raise ValueError("dout must match q's shape and device")
    if dout.dtype != q.dtype:
        dout = dout.to(q.dtype)
    if idx.dim() != 3 or tuple(idx.shape[:2]) != (B, N):
        raise ValueError(f"idx must be [B, N, kk]; got {tuple(idx.shape)}")
    if idx.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"idx must be int64 or int32; got {idx.dtype}")
    idx = idx.contiguous()
    dq = torch.empty((B, N, d), device=q.device, dtype=torch.float32)
    dk = torch.empty_like(dq)
    dv = torch.empty_like(dq)
    strides = _strides_n(q, k, v, dout)
    with _on(q.device):
        _lib.call("tarmac_gather_attention_backward", _ptr(q), _ptr(k),
                  _ptr(v), _ptr(dout), strides, _ptr(idx),
                  int(idx.dtype == torch.int64), idx.shape[-1], B, N, d,
                  _DTYPES[q.dtype], _scale(d, scale), _ptr(dq), _ptr(dk),
                  _ptr(dv), _stream(q.device))
    return dq, dk, dv


def dense_attention_backward(q: torch.Tensor, k: torch.Tensor,
                             v: torch.Tensor, out: torch.Tensor,
                             dout: torch.Tensor, scale: float | None = None):
    """Gradients (dq, dk, dv), fp32 [B, N, d], of dense masked-diagonal
    attention given its forward output ``out``. P is recomputed, not stored;
    deterministic."""
    q, k, v = _check_qkv(q, k, v)
    out, dout = _unit_inner(out), _unit_inner(dout)
    B, N, d = q.shape
    for t, name in ((out, "out"), (dout, "dout")):
        if t.shape != q.shape or t.device != q.device:
            raise ValueError(f"{name} must match q's shape and device")
    out = out.to(q.dtype)
    dout = dout.to(q.dtype)
    dq = torch.empty((B, N, d), device=q.device, dtype=torch.float32)
    dk = torch.empty_like(dq)
    dv = torch.empty_like(dq)
    work = torch.empty((2, B, N), device=q.device, dtype=torch.float32)
    strides = _strides_n(q, k, v, out, dout)
    with _on(q.device):
        _lib.call("tarmac_dense_attention_backward", _ptr(q), _ptr(k), _ptr(v),
                  _ptr(out), _ptr(dout), strides, B, N, d,
                  _DTYPES[q.dtype], _scale(d, scale), _ptr(dq), _ptr(dk),
                  _ptr(dv), _ptr(work), _stream(q.device))
    return dq, dk, dv


# ---------------------------------------------------------------------------
# positional and random selectors
# ---------------------------------------------------------------------------

SELECT_MAX_N = 8192
SELECT_MAX_K = 32


def knn_select(pos: torch.Tensor, k: int) -> torch.Tensor:
    """Exact k nearest peers (self excluded), int64 [B, N, k], by increasing
    (distance, index)."""
    pos = _check_pos(pos)
    B, N, _ = pos.shape
    out = torch.empty((B, N, k), device=pos.device, dtype=torch.int64)
    with _on(pos.device):
        _lib.call("tarmac_knn_select", _ptr(pos), B, N, int(k), _ptr(out),
                  _stream(pos.device))
    return out


def grid_knn_select(pos: torch.Tensor, k: int) -> torch.Tensor:
    """k nearest among the 3 x 3 grid cells around each agent (the reference's
    grid sizing and per-cell capacity), int64 [B, N, k]."""
    pos = _check_pos(pos)
    B, N, _ = pos.shape
    out = torch.empty((B, N, k), device=pos.device, dtype=torch.int64)
    with _on(pos.device):
        _lib.call("tarmac_grid_knn_select", _ptr(pos), B, N, int(k),
                  _ptr(out), _stream(pos.device))
    return out


def random_select(B: int, N: int, k: int, device,
                  generator: torch.Generator | None = None) -> torch.Tensor:
    """k distinct peers per agent, uniform over the k-subsets of the other
    N - 1 agents, int64 [B, N, k]. The Philox key is drawn from ``generator``
    (torch's default CPU generator when None), so torch.manual_seed fixes
    the selection."""
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("tarmac_b200 kernels need a CUDA device")
    seed, offset = (int(x) for x in torch.randint(
        0, 2 ** 62, (2,), generator=generator))
    out = torch.empty((B, N, k), device=device, dtype=torch.int64)
    with _on(device):
        _lib.call("tarmac_random_select", int(B), int(N), int(k), seed,
                  offset, _ptr(out), _stream(device))
    return out


# ---------------------------------------------------------------------------
# the whole communication module (inference)
# ---------------------------------------------------------------------------

def comm_forward(x: torch.Tensor, w_qkv: torch.Tensor, b_qkv: torch.Tensor,
                 w_proj: torch.Tensor, b_proj: torch.Tensor,
                 topk: int) -> torch.Tensor:
    """gelu(attention(split(x W_qkv^T + b_qkv))) W_proj^T + b_proj in one
    kernel: dense attention for ``topk == 0``, else top-k (k <= 8, lowest
    index on a tie). fp32, inference only (no autograd)."""
    ts = (x, w_qkv, b_qkv, w_proj, b_proj)
    if not x.is_cuda:
        raise RuntimeError("tarmac_b200 kernels need CUDA tensors")
    if any(t.device != x.device for t in ts[1:]):
        raise ValueError("x and the comm weights must be on one device")
    if x.dim() != 3:
        raise ValueError(f"x must be [B, N, in_dim]; got {tuple(x.shape)}")
    x, w_qkv, b_qkv, w_proj, b_proj = (
        t if t.dtype == torch.float32 and t.is_contiguous()
        else t.contiguous().float() for t in ts)
    B, N, D = x.shape
    m = w_proj.shape[0]
    if w_qkv.shape != (3 * m, D) or b_qkv.shape != (3 * m,) or \
            w_proj.shape != (m, m) or b_proj.shape != (m,):
        raise ValueError("weights must be qkv [3m, in_dim], [3m] and proj "
                         "[m, m], [m]")
    out = torch.empty((B, N, m), device=x.device, dtype=torch.float32)
    with _on(x.device):
        _lib.call("tarmac_comm_forward", _ptr(x), _ptr(w_qkv), _ptr(b_qkv),
                  _ptr(w_proj), _ptr(b_proj), B, N, D, m, int(topk),
                  _ptr(out), _stream(x.device))
    return out


# ---------------------------------------------------------------------------
# multi-head operators
# ---------------------------------------------------------------------------

_PEERS = {"all": _lib.PEERS_ALL, "others": _lib.PEERS_OTHERS,
          "past": _lib.PEERS_PAST}
_PACK6 = struct.Struct("=6q").pack
_PACK9 = struct.Struct("=9q").pack
_PACK12 = struct.Struct("=12q").pack
_PACK15 = struct.Struct("=15q").pack


def _check_heads(named: dict, like: torch.Tensor) -> None:
    """Every tensor 4-D, of one supported dtype, on the CUDA device of ``like``."""
    if not like.is_cuda:
        raise RuntimeError("tarmac_b200 kernels need CUDA tensors (there is no "
                           "CPU implementation)")
    if like.dtype not in _DTYPES:
        raise TypeError(f"tensors must be float32 or bfloat16; got {like.dtype}")
    for name, t in named.items():
        if t.dim() != 4:
            raise ValueError(f"{name} must be [B, N, heads, d]; got {tuple(t.shape)}")
        if t.device != like.device:
            raise ValueError(f"{name} must be on the device of the queries")
        if t.dtype != like.dtype:
            raise TypeError(f"{name} must have the queries' dtype {like.dtype}; "
                            f"got {t.dtype}")


def _norm_weight(w, name: str, d: int, dev) -> torch.Tensor | None:
    if w is None:
        return None
    if tuple(w.shape) != (d,):
        raise ValueError(f"{name} must be [{d}]; got {tuple(w.shape)}")
    if w.device != dev:
        raise ValueError(f"{name} must be on the device of the queries")
    return w if w.dtype == torch.float32 and w.is_contiguous() \
        else w.float().contiguous()


def _check_rotate(q, k, wq, wk, cos, sin):
    _check_heads({"q": q, "k": k}, q)
    B, N, H, d = q.shape
    if k.shape[0] != B or k.shape[1] != N or k.shape[3] != d:
        raise ValueError(f"k must be [{B}, {N}, heads, {d}]; got {tuple(k.shape)}")
    wq, wk = _norm_weight(wq, "wq", d, q.device), _norm_weight(wk, "wk", d, q.device)
    if cos.shape != sin.shape or cos.dim() != 3 or cos.shape[0] not in (1, B) \
            or cos.shape[1] != N or 2 * cos.shape[2] > d:
        raise ValueError(f"cos and sin must be [1 or {B}, {N}, r / 2] with "
                         f"r <= {d}; got {tuple(cos.shape)}, {tuple(sin.shape)}")
    for t in (cos, sin):
        if t.device != q.device:
            raise ValueError("cos and sin must be on the device of the queries")
        if t.dtype != torch.float32:
            raise TypeError(f"cos and sin must be float32; got {t.dtype}")
    return (_unit_inner(q), _unit_inner(k), wq, wk, cos.contiguous(),
            sin.contiguous())


def _rotate_ready(q, k, wq, wk, cos, sin) -> bool:
    """Whether the arguments can be passed on as they are. Cheap: a call on a
    few rows is bound by its host work, so the checks that name a fault
    (:func:`_check_rotate`) run only when this one fails."""
    qs, ks, cs = q.shape, k.shape, cos.shape
    if len(qs) != 4 or len(ks) != 4 or len(cs) != 3 or sin.shape != cs:
        return False
    B, N, _, d = qs
    t, dev = q.dtype, q.get_device()
    f32 = torch.float32
    return (t in _DTYPES and k.dtype is t and cos.dtype is f32 and sin.dtype is f32
            and dev >= 0 and k.get_device() == dev and cos.get_device() == dev
            and sin.get_device() == dev and ks[0] == B and ks[1] == N and ks[3] == d
            and (cs[0] == 1 or cs[0] == B) and cs[1] == N and 2 * cs[2] <= d
            and q.stride(3) == 1 and k.stride(3) == 1
            and cos.is_contiguous() and sin.is_contiguous()
            and (wq is None or (wq.dtype is f32 and wq.shape == (d,)
                                and wq.get_device() == dev and wq.stride(0) == 1))
            and (wk is None or (wk.dtype is f32 and wk.shape == (d,)
                                and wk.get_device() == dev and wk.stride(0) == 1)))


def _launch(dev: int, name: str, *args) -> None:
    """Call an entry point on the current stream of CUDA device ``dev`` (the
    stream is the last argument of every entry point)."""
    if dev == _GET_DEVICE():
        _lib.call(name, *args, _stream_of(dev))
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, _stream_of(dev))


_GET_DEVICE = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _stream_of(dev: int) -> int:
    if _RAW_STREAM is not None:
        return _RAW_STREAM(dev)
    return torch.cuda.current_stream(dev).cuda_stream


def _table_stride(cos: torch.Tensor, B: int) -> int:
    """Elements between two episodes' tables (0: one table for all)."""
    return cos.shape[1] * cos.shape[2] if cos.shape[0] == B and B > 1 else 0


def qk_norm_rotate(q: torch.Tensor, k: torch.Tensor,
                   wq: torch.Tensor | None, wk: torch.Tensor | None,
                   cos: torch.Tensor, sin: torch.Tensor, eps: float = 1e-6,
                   interleaved: bool = False):
    """Norm every head of q ([B, N, H, d]) and k ([B, N, Hk, d]) by its root
    mean square, scale by ``wq`` / ``wk`` ([d], None for ones) and rotate the
    first r columns by the rows' angles, in one pass. ``cos``, ``sin``: fp32
    [1 or B, N, r / 2]; column pairs are (i, i + r / 2), or (2i, 2i + 1) with
    ``interleaved``. Returns contiguous (q', k') in the inputs' dtype. The
    single-token form is N = 1 with the token's row of the table."""
    if not _rotate_ready(q, k, wq, wk, cos, sin):
        q, k, wq, wk, cos, sin = _check_rotate(q, k, wq, wk, cos, sin)
    B, N, H, d = q.shape
    qo, ko = _empty_as(q), _empty_as(k)
    _launch(q.get_device(), "tarmac_qk_norm_rotate", q.data_ptr(),
            k.data_ptr(), qo.data_ptr(), ko.data_ptr(),
            _PACK6(*q.stride()[:3], *k.stride()[:3]), _ptr(wq), _ptr(wk),
            cos.data_ptr(), sin.data_ptr(), _table_stride(cos, B), B, N, H,
            k.shape[2], d, 2 * cos.shape[2], _DTYPES[q.dtype], eps,
            int(interleaved))
    return qo, ko


def qk_norm_rotate_backward(q: torch.Tensor, k: torch.Tensor,
                            wq: torch.Tensor | None, wk: torch.Tensor | None,
                            cos: torch.Tensor, sin: torch.Tensor,
                            dq_out: torch.Tensor, dk_out: torch.Tensor,
                            eps: float = 1e-6, interleaved: bool = False):
    """Gradients of :func:`qk_norm_rotate` for its inputs and the gradients of
    its outputs: (dq, dk) in the inputs' dtype and (dwq, dwk) fp32 [d] (None
    where there is no weight). Deterministic."""
    if not _rotate_ready(q, k, wq, wk, cos, sin):
        q, k, wq, wk, cos, sin = _check_rotate(q, k, wq, wk, cos, sin)
    gq, gk = _gradient(dq_out, q, "dq_out"), _gradient(dk_out, k, "dk_out")
    B, N, H, d = q.shape
    dq, dk = _empty_as(q), _empty_as(k)
    work = torch.empty(_rotate_work(B, N, H, k.shape[2], d) // 4,
                       device=q.device, dtype=torch.float32)
    dwq, dwk = torch.empty((2, d), device=q.device, dtype=torch.float32)
    dwq = None if wq is None else dwq
    dwk = None if wk is None else dwk
    _launch(q.get_device(), "tarmac_qk_norm_rotate_backward", q.data_ptr(),
            k.data_ptr(), gq.data_ptr(), gk.data_ptr(),
            _PACK12(*q.stride()[:3], *k.stride()[:3], *gq.stride()[:3],
                    *gk.stride()[:3]),
            _ptr(wq), _ptr(wk), cos.data_ptr(), sin.data_ptr(),
            _table_stride(cos, B), B, N, H, k.shape[2], d, 2 * cos.shape[2],
            _DTYPES[q.dtype], eps, int(interleaved), dq.data_ptr(),
            dk.data_ptr(), _ptr(dwq), _ptr(dwk), work.data_ptr())
    return dq, dk, dwq, dwk


def _gradient(g: torch.Tensor, like: torch.Tensor, name: str) -> torch.Tensor:
    """``g`` checked against the tensor it belongs to, with unit inner stride."""
    if g.shape != like.shape:
        raise ValueError(f"{name} must have the shape {tuple(like.shape)}; got "
                         f"{tuple(g.shape)}")
    if g.dtype is not like.dtype or g.get_device() != like.get_device():
        _check_heads({name: g}, like)
    return g if g.stride(3) == 1 else _unit_inner(g)


@functools.lru_cache(maxsize=1024)
def _rotate_work(B, N, H, Hk, d) -> int:
    return _lib.lib().tarmac_qk_norm_rotate_workspace(B, N, H, Hk, d)


def pack_visibility(visible: torch.Tensor) -> torch.Tensor:
    """Truth values [1 or B, Nq, Nk] to the words the attention kernels read:
    int32 [1 or B, Nq, ceil(Nk / 32)], 32 keys each, lowest key in the lowest
    bit. A program that uses one mask in several calls packs it once."""
    if visible.dim() != 3:
        raise ValueError(f"visible must be [B, Nq, Nk]; got {tuple(visible.shape)}")
    if visible.dtype != torch.bool:
        raise TypeError(f"visible must be bool; got {visible.dtype}")
    if not visible.is_cuda:
        raise RuntimeError("tarmac_b200 kernels need CUDA tensors")
    visible = _unit_inner(visible)
    B, Nq, Nk = visible.shape
    bits = torch.empty((B, Nq, (Nk + 31) // 32), device=visible.device,
                       dtype=torch.int32)
    with _on(visible.device):
        _lib.call("tarmac_pack_visibility", _ptr(visible), visible.stride(0),
                  visible.stride(1), B, Nq, Nk, _ptr(bits),
                  _stream(visible.device))
    return bits


def _check_attention(q, k, v, peers, key_len, q_start, visible):
    """Checked q, k, v, lengths, starts and visibility words."""
    _check_heads({"q": q, "k": k, "v": v}, q)
    B, Nq, H, d = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != d:
        raise ValueError(f"k and v must share one [{B}, Nk, heads, {d}] shape; "
                         f"got {tuple(k.shape)}, {tuple(v.shape)}")
    Nk, Hk = k.shape[1], k.shape[2]
    if Hk < 1 or H % Hk:
        raise ValueError(f"the query heads ({H}) must be a multiple of the key "
                         f"heads ({Hk})")
    if peers not in _PEERS:
        raise ValueError(f"peers must be 'all', 'others' or 'past'; got {peers!r}")
    ints = []
    for name, t in (("key_len", key_len), ("q_start", q_start)):
        if t is not None:
            if tuple(t.shape) != (B,):
                raise ValueError(f"{name} must be [{B}]; got {tuple(t.shape)}")
            if t.dtype not in (torch.int32, torch.int64):
                raise TypeError(f"{name} must be int32 or int64; got {t.dtype}")
            if t.device != q.device:
                raise ValueError(f"{name} must be on the device of the queries")
            if t.dtype is torch.int64:  # beyond 32 bits they act like the bounds
                t = t.clamp(-2 ** 31, 2 ** 31 - 1)
            t = t.to(torch.int32).contiguous()
        ints.append(t)
    if visible is not None:
        if visible.device != q.device:
            raise ValueError("visible must be on the device of the queries")
        words = (Nk + 31) // 32
        wide = Nk if visible.dtype == torch.bool else words
        if visible.dim() != 3 or visible.shape[0] not in (1, B) \
                or tuple(visible.shape[1:]) != (Nq, wide):
            raise ValueError(
                f"visible must be bool [1 or {B}, {Nq}, {Nk}] or its words "
                f"int32 [1 or {B}, {Nq}, {words}]; got {tuple(visible.shape)}")
        if visible.dtype == torch.bool:
            visible = pack_visibility(visible)
        elif visible.dtype != torch.int32:
            raise TypeError(f"visible must be bool or int32; got {visible.dtype}")
        visible = visible.contiguous()
    return _unit_inner(q), _unit_inner(k), _unit_inner(v), *ints, visible


def _attention_ready(q, k, v, peers, key_len, q_start) -> bool:
    """As :func:`_rotate_ready`, for calls without a visibility mask."""
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or v.shape != ks or peers not in _PEERS:
        return False
    t, dev = q.dtype, q.get_device()
    if not (t in _DTYPES and k.dtype is t and v.dtype is t and dev >= 0
            and k.get_device() == dev and v.get_device() == dev
            and ks[0] == qs[0] and ks[3] == qs[3] and ks[2] > 0
            and qs[2] % ks[2] == 0 and q.stride(3) == 1 and k.stride(3) == 1
            and v.stride(3) == 1):
        return False
    for x in (key_len, q_start):
        if x is not None and not (
                x.dtype is torch.int32 and x.shape == (qs[0],)
                and x.get_device() == dev and x.is_contiguous()):
            return False
    return True


def _bits_stride(bits: torch.Tensor | None) -> int:
    """Words between two episodes' masks (0: one mask for all)."""
    if bits is None or bits.shape[0] == 1:
        return 0
    return bits.shape[1] * bits.shape[2]


@functools.lru_cache(maxsize=1024)
def _attention_work(B, Nq, Nk, H, Hk, d) -> int:
    return _lib.lib().tarmac_head_attention_workspace(B, Nq, Nk, H, Hk, d)


@functools.lru_cache(maxsize=1024)
def _attention_backward_work(B, Nq, H) -> int:
    return _lib.lib().tarmac_head_attention_backward_workspace(B, Nq, H)


def head_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                   peers: str = "all", key_len: torch.Tensor | None = None,
                   q_start: torch.Tensor | None = None,
                   visible: torch.Tensor | None = None,
                   scale: float | None = None, return_lse: bool = False):
    """Masked attention with heads: q [B, Nq, H, d], k and v [B, Nk, Hk, d]
    with H a multiple of Hk; returns out [B, Nq, H, d] (and lse, fp32
    [B, H, Nq]).

    Row i stands at position ``q_start[b] + i`` (default ``Nk - Nq + i``) and
    sees key j when ``j < key_len[b]``, ``peers`` allows it ("all"; "others":
    not its own position; "past": positions up to its own) and
    ``visible[b, i, j]`` holds (bool [1 or B, Nq, Nk], or the words of
    :func:`pack_visibility`). A row that sees nothing gets 0 (lse -inf). Keys
    and values from ``key_len`` on are never used, whatever they hold; those
    before it must be finite, masked or not (a weight of zero times a NaN is a
    NaN). One token over a long history is Nq = 1: the key axis is then split
    over the GPU."""
    if visible is None and _attention_ready(q, k, v, peers, key_len, q_start):
        bits = None
    else:
        q, k, v, key_len, q_start, bits = _check_attention(
            q, k, v, peers, key_len, q_start, visible)
    B, Nq, H, d = q.shape
    _, Nk, Hk, _ = k.shape
    dev = q.get_device()
    out = _empty_as(q)
    lse = (torch.empty((B, H, Nq), device=q.device, dtype=torch.float32)
           if return_lse else None)
    nbytes = _attention_work(B, Nq, Nk, H, Hk, d)
    work = (torch.empty(nbytes, device=q.device, dtype=torch.uint8)
            if nbytes else None)
    _launch(dev, "tarmac_head_attention", q.data_ptr(), k.data_ptr(),
            v.data_ptr(), out.data_ptr(), _ptr(lse),
            _PACK9(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3]),
            _ptr(key_len), _ptr(q_start), _ptr(bits), _bits_stride(bits), B,
            Nq, Nk, H, Hk, d, _DTYPES[q.dtype], _PEERS[peers],
            _scale(d, scale), _ptr(work))
    return (out, lse) if return_lse else out


def head_attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                            out: torch.Tensor, lse: torch.Tensor,
                            dout: torch.Tensor, peers: str = "all",
                            key_len: torch.Tensor | None = None,
                            q_start: torch.Tensor | None = None,
                            visible: torch.Tensor | None = None,
                            scale: float | None = None):
    """Gradients (dq, dk, dv) of :func:`head_attention` in the inputs' dtype,
    given its ``out`` and ``lse`` and the gradient of out. The probabilities
    are recomputed; shared key heads are summed over their query heads;
    deterministic."""
    if visible is None and _attention_ready(q, k, v, peers, key_len, q_start):
        bits = None
    else:
        q, k, v, key_len, q_start, bits = _check_attention(
            q, k, v, peers, key_len, q_start, visible)
    B, Nq, H, d = q.shape
    _, Nk, Hk, _ = k.shape
    out, dout = _gradient(out, q, "out"), _gradient(dout, q, "dout")
    if lse.shape != (B, H, Nq) or lse.dtype is not torch.float32 \
            or lse.get_device() != q.get_device():
        raise ValueError(f"lse must be float32 [{B}, {H}, {Nq}] on the device "
                         "of the queries")
    lse = lse.contiguous()
    dq, dk, dv = _empty_as(q), _empty_as(k), _empty_as(v)
    work = torch.empty(_attention_backward_work(B, Nq, H), device=q.device,
                       dtype=torch.uint8)
    _launch(q.get_device(), "tarmac_head_attention_backward", q.data_ptr(),
            k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
            dout.data_ptr(),
            _PACK15(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
                    *out.stride()[:3], *dout.stride()[:3]),
            _ptr(key_len), _ptr(q_start), _ptr(bits), _bits_stride(bits), B,
            Nq, Nk, H, Hk, d, _DTYPES[q.dtype], _PEERS[peers],
            _scale(d, scale), dq.data_ptr(),
            dk.data_ptr(), dv.data_ptr(), work.data_ptr())
    return dq, dk, dv


def head_attention_plan(B: int, Nq: int, Nk: int, H: int, Hk: int, d: int,
                        dtype: torch.dtype = torch.float32, peers: str = "all",
                        backward: bool = False) -> dict:
    """The kernels a contiguous :func:`head_attention` call (or its gradients)
    with these shapes takes, e.g. {"kernel": "head_fwd_tc", "items": 240}.
    Host-only (no GPU needed); raises :class:`TarmacError` for arguments the
    call itself would reject."""
    import ctypes
    import json
    buf = ctypes.create_string_buffer(128)
    _lib.call("tarmac_head_attention_plan", int(backward), None, B, Nq, Nk, H,
              Hk, d, _DTYPES[dtype], _PEERS[peers], buf, len(buf))
    return json.loads(buf.value.decode())


# ---------------------------------------------------------------------------
# a memory of fixed size: attention with a decay for each head
# ---------------------------------------------------------------------------

def _check_state(t, name: str, q: torch.Tensor) -> torch.Tensor | None:
    """A state tensor, fp32 [B, H, d, d], contiguous."""
    if t is None:
        return None
    B, _, H, d = q.shape
    if t.dtype is torch.float32 and t.shape == (B, H, d, d) \
            and t.get_device() == q.get_device() and t.is_contiguous():
        return t
    if tuple(t.shape) != (B, H, d, d):
        raise ValueError(f"{name} must be [{B}, {H}, {d}, {d}]; got {tuple(t.shape)}")
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32; got {t.dtype}")
    if t.device != q.device:
        raise ValueError(f"{name} must be on the device of the queries")
    return t.contiguous()


def _check_decay(q, k, v, log_decay, lens):
    """Checked q, k, v, decays and lengths."""
    _check_heads({"q": q, "k": k, "v": v}, q)
    B, N, H, d = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[1] != N or k.shape[3] != d:
        raise ValueError(f"k and v must share one [{B}, {N}, heads, {d}] shape; "
                         f"got {tuple(k.shape)}, {tuple(v.shape)}")
    Hk = k.shape[2]
    if Hk < 1 or H % Hk:
        raise ValueError(f"the query heads ({H}) must be a multiple of the key "
                         f"heads ({Hk})")
    if tuple(log_decay.shape) != (H,):
        raise ValueError(f"log_decay must be [{H}]; got {tuple(log_decay.shape)}")
    if log_decay.dtype != torch.float32:
        raise TypeError(f"log_decay must be float32; got {log_decay.dtype}")
    if log_decay.device != q.device:
        raise ValueError("log_decay must be on the device of the queries")
    if lens is not None:
        if tuple(lens.shape) != (B,):
            raise ValueError(f"lens must be [{B}]; got {tuple(lens.shape)}")
        if lens.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"lens must be int32 or int64; got {lens.dtype}")
        if lens.device != q.device:
            raise ValueError("lens must be on the device of the queries")
        if lens.dtype is torch.int64:  # beyond 32 bits they act like the bounds
            lens = lens.clamp(-2 ** 31, 2 ** 31 - 1)
        lens = lens.to(torch.int32).contiguous()
    return (_unit_inner(q), _unit_inner(k), _unit_inner(v), log_decay.contiguous(),
            lens)


def _decay_ready(q, k, v, log_decay, lens) -> bool:
    """As :func:`_rotate_ready`."""
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or v.shape != ks:
        return False
    t, dev = q.dtype, q.get_device()
    return (t in _DTYPES and k.dtype is t and v.dtype is t and dev >= 0
            and k.get_device() == dev and v.get_device() == dev
            and ks[0] == qs[0] and ks[1] == qs[1] and ks[3] == qs[3] and ks[2] > 0
            and qs[2] % ks[2] == 0 and q.stride(3) == 1 and k.stride(3) == 1
            and v.stride(3) == 1 and log_decay.dtype is torch.float32
            and log_decay.shape == (qs[2],) and log_decay.get_device() == dev
            and log_decay.is_contiguous()
            and (lens is None or (lens.dtype is torch.int32
                                  and lens.shape == (qs[0],)
                                  and lens.get_device() == dev
                                  and lens.is_contiguous())))


@functools.lru_cache(maxsize=1024)
def _decay_work(*sizes) -> int:
    return _lib.lib().tarmac_decay_attention_workspace(*sizes)


@functools.lru_cache(maxsize=1024)
def _decay_backward_work(*sizes) -> int:
    return _lib.lib().tarmac_decay_attention_backward_workspace(*sizes)


def _scratch(nbytes: int, dev: torch.device) -> torch.Tensor | None:
    return torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    log_decay: torch.Tensor, state: torch.Tensor | None = None,
                    lens: torch.Tensor | None = None, scale: float | None = None,
                    return_state: bool = False,
                    state_out: torch.Tensor | None = None):
    """Attention with a decay for each head, a memory of fixed size: q
    [B, N, H, d], k and v [B, N, Hk, d] with H a multiple of Hk. For the rows
    of an episode in order, with l = exp(log_decay[h]) (fp32 [H], at most 0),

        S = l S + k v^T,   out = scale S^T q   (scale: default d ** -0.5).

    ``state`` (fp32 [B, H, d, d], by the columns of k, then of v) is S before
    the first row, zero when None. Returns out [B, N, H, d], or (out, S after
    the last row) with ``return_state`` or a ``state_out`` to write it to: a
    contiguous tensor like ``state`` and apart from all inputs, or ``state``
    itself, renewed in place. Rows from ``lens`` [B] on are padding, whatever
    they hold: they get 0 and leave S alone; those before must be finite (a
    head's infinity may reach any of its rows as a NaN). One new row over a
    kept state is N = 1; a state renewed call after call does not gather the
    rounding of its decay."""
    if not _decay_ready(q, k, v, log_decay, lens):
        q, k, v, log_decay, lens = _check_decay(q, k, v, log_decay, lens)
    start = _check_state(state, "state", q)
    if state_out is not None:
        if _check_state(state_out, "state_out", q) is not state_out:
            raise ValueError("state_out must be contiguous")
        if state is not None and state_out is not state \
                and _overlap(state_out, start):
            raise ValueError("state_out must be state itself or apart from it")
    B, N, H, d = q.shape
    out = _empty_as(q)
    if state_out is not None:  # a graph that saved what it holds now has to know
        torch.autograd.graph.increment_version(state_out)
    if return_state and state_out is None:
        state_out = torch.empty((B, H, d, d), device=q.device, dtype=torch.float32)
    work = _scratch(_decay_work(B, N, H, d, _DTYPES[q.dtype], int(state_out is not None)),
                    q.device)
    _launch(q.get_device(), "tarmac_decay_attention", q.data_ptr(), k.data_ptr(),
            v.data_ptr(), out.data_ptr(),
            _PACK9(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3]),
            log_decay.data_ptr(), _ptr(start), _ptr(state_out), _ptr(lens), B, N,
            H, k.shape[2], d, _DTYPES[q.dtype], _scale(d, scale), _ptr(work))
    return out if state_out is None else (out, state_out)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Do two contiguous tensors share memory without being the same?"""
    a0, b0 = a.data_ptr(), b.data_ptr()
    return a0 != b0 and a0 < b0 + 4 * b.numel() and b0 < a0 + 4 * a.numel()


def decay_attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                             log_decay: torch.Tensor, dout: torch.Tensor,
                             state: torch.Tensor | None = None,
                             dstate: torch.Tensor | None = None,
                             lens: torch.Tensor | None = None,
                             scale: float | None = None,
                             need_dstate: bool = True):
    """Gradients (dq, dk, dv, dS) of :func:`decay_attention`, given those of out
    (``dout``) and of the state that it returned (``dstate``, or None). dS, of
    the state before the first row, is None where ``state`` is, or without
    ``need_dstate``. Shared key heads are summed over their query heads; padding
    gets zeros; the decays have no gradient; ``scale`` is from 2 ** -60 to 2 ** 20.
    Deterministic."""
    if not _decay_ready(q, k, v, log_decay, lens):
        q, k, v, log_decay, lens = _check_decay(q, k, v, log_decay, lens)
    dout = _gradient(dout, q, "dout")
    start, dstate = _check_state(state, "state", q), _check_state(dstate, "dstate", q)
    B, N, H, d = q.shape
    Hk = k.shape[2]
    dq, dk, dv = _empty_as(q), _empty_as(k), _empty_as(v)
    first = torch.empty_like(start) if need_dstate and start is not None else None
    work = _scratch(_decay_backward_work(B, N, H, Hk, d, _DTYPES[q.dtype],
                                         int(first is not None)), q.device)
    _launch(q.get_device(), "tarmac_decay_attention_backward", q.data_ptr(),
            k.data_ptr(), v.data_ptr(), dout.data_ptr(),
            _PACK12(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
                    *dout.stride()[:3]),
            log_decay.data_ptr(), _ptr(start), _ptr(dstate), _ptr(lens), B, N, H,
            Hk, d, _DTYPES[q.dtype], _scale(d, scale), dq.data_ptr(),
            dk.data_ptr(), dv.data_ptr(), _ptr(first), _ptr(work))
    return dq, dk, dv, first


def decay_attention_plan(B: int, N: int, H: int, Hk: int, d: int,
                         dtype: torch.dtype = torch.float32, state: bool = False,
                         backward: bool = False) -> dict:
    """The kernels a contiguous :func:`decay_attention` call (or its gradients)
    with these shapes takes, e.g. {"kernel": "decay_tc", "segments": 4, "states":
    True}; ``state``: with a state returned (a gradient of the one given).
    Host-only (no GPU needed); raises :class:`TarmacError` for arguments the
    call itself would reject."""
    import ctypes
    import json
    buf = ctypes.create_string_buffer(128)
    _lib.call("tarmac_decay_attention_plan", int(backward), None, B, N, H, Hk, d,
              _DTYPES[dtype], int(state), buf, len(buf))
    return json.loads(buf.value.decode())


# ---------------------------------------------------------------------------
# the norms around a block
# ---------------------------------------------------------------------------

_PACK10 = struct.Struct("=10q").pack


def _norm_rows(t: torch.Tensor) -> torch.Tensor:
    """[B, N, D] view (a copy where the strides allow none) with unit inner
    stride. Leading dimensions that are evenly spaced become one."""
    t = _unit_inner(t)
    if t.dim() == 3:
        return t
    if t.dim() < 3:
        return t.reshape((1,) * (3 - t.dim()) + tuple(t.shape))
    return t.flatten(0, -3)


def _check_norm(x, named: dict, weights: dict):
    """The rows as [B, N, D] and the weights, checked."""
    if not x.is_cuda:
        raise RuntimeError("tarmac_b200 kernels need CUDA tensors (there is no "
                           "CPU implementation)")
    if x.dtype not in _DTYPES:
        raise TypeError(f"tensors must be float32 or bfloat16; got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("x must have rows of columns")
    for name, t in named.items():
        if t is None:
            continue
        if t.shape != x.shape:
            raise ValueError(f"{name} must have the shape {tuple(x.shape)}; got "
                             f"{tuple(t.shape)}")
        if t.device != x.device:
            raise ValueError(f"{name} must be on the device of x")
        if t.dtype != x.dtype:
            raise TypeError(f"{name} must have the dtype {x.dtype} of x; got {t.dtype}")
    D = x.shape[-1]
    for name, w in weights.items():
        if w is None:
            continue
        if tuple(w.shape) != (D,):
            raise ValueError(f"{name} must be [{D}]; got {tuple(w.shape)}")
        if w.device != x.device:
            raise ValueError(f"{name} must be on the device of x")
    rows = [None if t is None else _norm_rows(t) for t in (x, *named.values())]
    return rows, [None if w is None else w.float().contiguous()
                  for w in weights.values()]


def _norm_ready(x, rows, weights) -> bool:
    """As :func:`_rotate_ready`: may x and the other rows [B, N, D] and the
    weights be passed on as they are?"""
    shape, t, dev = x.shape, x.dtype, x.get_device()
    if len(shape) != 3 or t not in _DTYPES or dev < 0 or x.stride(2) != 1:
        return False
    for r in rows:
        if r is not None and not (r.shape == shape and r.dtype is t
                                  and r.get_device() == dev and r.stride(2) == 1):
            return False
    for w in weights:
        if w is not None and not (w.dtype is torch.float32 and w.shape == shape[2:]
                                  and w.get_device() == dev and w.stride(0) == 1):
            return False
    return True


def _row_strides(t: torch.Tensor | None) -> tuple:
    return (0, 0) if t is None else t.stride()[:2]


def residual_norm(x: torch.Tensor, y: torch.Tensor,
                  w_post: torch.Tensor | None = None,
                  w_pre: torch.Tensor | None = None,
                  gate: torch.Tensor | None = None,
                  scale: torch.Tensor | None = None, eps: float = 1e-6):
    """What stands between two blocks, in one pass: the norm of a block's
    output y, its gate and residual scale, the sum with the stream x, and the
    norm before the next block. For rows of D <= 8192 columns,

        h = x + scale * sigmoid(gate) * (y / rms(y) * w_post)
        z = h / rms(h) * w_pre,   rms(t) = sqrt(mean t^2 + eps).

    x, y, gate: [..., D] fp32 or bf16 (no gate: ones in place of its sigmoid);
    ``w_post``, ``w_pre``, ``scale``: [D] or None (ones). Returns contiguous (h, z)
    in the inputs' dtype."""
    if _norm_ready(x, (y, gate), (w_post, w_pre, scale)):
        xr, yr, gr, wo, wi, sc = x, y, gate, w_post, w_pre, scale
    else:
        (xr, yr, gr), (wo, wi, sc) = _check_norm(
            x, {"y": y, "gate": gate},
            {"w_post": w_post, "w_pre": w_pre, "scale": scale})
    h, z = _empty_as(x), _empty_as(x)
    B, N, D = xr.shape
    _launch(x.get_device(), "tarmac_residual_norm", xr.data_ptr(), yr.data_ptr(),
            _ptr(gr), _PACK6(*_row_strides(xr), *_row_strides(yr), *_row_strides(gr)),
            _ptr(wo), _ptr(wi), _ptr(sc), B, N, D, _DTYPES[x.dtype], eps,
            h.data_ptr(), z.data_ptr())
    return h, z


@functools.lru_cache(maxsize=1024)
def _norm_work(B, N, D) -> int:
    return _lib.lib().tarmac_residual_norm_workspace(B, N, D)


def residual_norm_backward(x: torch.Tensor, y: torch.Tensor,
                           w_post: torch.Tensor | None,
                           w_pre: torch.Tensor | None,
                           gate: torch.Tensor | None,
                           scale: torch.Tensor | None,
                           dh: torch.Tensor | None, dz: torch.Tensor | None,
                           eps: float = 1e-6):
    """Gradients of :func:`residual_norm` for its inputs and the gradients of
    its outputs (None: zero): (dx, dy) and dgate in the inputs' dtype and
    (dw_post, dw_pre, dscale) fp32 [D], as (dx, dy, dw_post, dw_pre, dgate,
    dscale), None where the input is. Deterministic."""
    if _norm_ready(x, (y, gate, dh, dz), (w_post, w_pre, scale)):
        xr, yr, gr, hr, zr, wo, wi, sc = x, y, gate, dh, dz, w_post, w_pre, scale
    else:
        (xr, yr, gr, hr, zr), (wo, wi, sc) = _check_norm(
            x, {"y": y, "gate": gate, "dh": dh, "dz": dz},
            {"w_post": w_post, "w_pre": w_pre, "scale": scale})
    B, N, D = xr.shape
    dx, dy = _empty_as(x), _empty_as(x)
    dgate = None if gate is None else _empty_as(x)
    dwo, dwi, dsc = torch.empty((3, D), device=x.device, dtype=torch.float32)
    dwo = None if wo is None else dwo
    dwi = None if wi is None else dwi
    dsc = None if sc is None else dsc
    work = _scratch(_norm_work(B, N, D), x.device)
    _launch(x.get_device(), "tarmac_residual_norm_backward", xr.data_ptr(),
            yr.data_ptr(), _ptr(gr), _ptr(hr), _ptr(zr),
            _PACK10(*_row_strides(xr), *_row_strides(yr), *_row_strides(gr),
                    *_row_strides(hr), *_row_strides(zr)),
            _ptr(wo), _ptr(wi), _ptr(sc), B, N, D, _DTYPES[x.dtype], eps,
            dx.data_ptr(), dy.data_ptr(), _ptr(dgate), _ptr(dwo), _ptr(dwi),
            _ptr(dsc), _ptr(work))
    return dx, dy, dwo, dwi, dgate, dsc


_PLAN_OPS = {"dense": 0, "topk": 1, "streaming": 2}
_PLAN_MODES = {"argmax": _lib.SELECT_ARGMAX, "threshold": _lib.SELECT_THRESHOLD,
               "sort": _lib.SELECT_SORT}


def kernel_plan(op: str, B: int, N: int, d: int, dtype: torch.dtype = torch.float32,
                k: int = 1, mode: str = "argmax") -> dict:
    """The kernel and tiling a contiguous call of ``op`` ("dense", "topk" or
    "streaming") with these shapes takes, as the library decides it from the
    shape: e.g. {"kernel": "topk_ws", "query_tile": 128, "key_tile": 128,
    "chunk": 8, "chunks_kept": 2}. Host-only (no GPU needed); raises
    :class:`TarmacError` for arguments the call itself would reject."""
    import ctypes
    import json
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("dtype must be float32 or bfloat16")
    dt = _lib.BF16 if dtype == torch.bfloat16 else _lib.F32
    buf = ctypes.create_string_buffer(256)
    _lib.call("tarmac_kernel_plan", _PLAN_OPS[op], B, N, d, dt, k,
              _PLAN_MODES[mode], None, buf, len(buf))
    return json.loads(buf.value.decode())
