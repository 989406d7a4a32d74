"""Norms of queries and keys per head with the position rotation in the same
pass (``rq_qk_norm_rope`` of include/rq.h), and the form that puts the keys
and values straight into a 4-bit cache.  The reference rotates without a norm
and in a pass of its own (QAttn::forward, src/streaming_quantized.rs:201-240).
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import QkRope, check
from .kv4 import _PAIR, dtype_of, int32, need, stream_of
from .linear import Context


def rope_tables(max_pos: int, rot_dim: int, theta: float = 10000.0, device: int = 0):
    """(cos, sin) f32 [max_pos, rot_dim / 2], the angles taken in 64 bits."""
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    a = torch.arange(max_pos, dtype=torch.float64)[:, None] * theta ** (-i / max(rot_dim, 1))
    return a.cos().float().to(f"cuda:{device}"), a.sin().float().to(f"cuda:{device}")


def _args(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved, q_out, k_out):
    need(isinstance(q, torch.Tensor) and isinstance(k, torch.Tensor) and q.is_cuda and q.dim() == 3 and k.dim() == 3
         and q.dtype == k.dtype and q.device == k.device and q.shape[0] == k.shape[0] and q.shape[2] == k.shape[2],
         "q, k: [tokens, heads, head_dim] of one type on one CUDA device are wanted")
    dev, hd = q.device, q.shape[2]
    for name, x, like in (("q", q, q), ("k", k, k), ("q_out", q_out, q), ("k_out", k_out, k)):
        need(x is None or x.shape == like.shape and x.dtype == like.dtype and x.device == dev and x.stride(2) == 1,
             f"{name}: {list(like.shape)} {like.dtype} with contiguous elements on {dev} is wanted")
    need(cos.dtype is torch.float32 and sin.dtype is torch.float32 and cos.dim() == 2 and cos.shape == sin.shape
         and cos.is_contiguous() and sin.is_contiguous() and cos.device == dev and sin.device == dev,
         "cos, sin: contiguous float32 [max_pos, rot_dim / 2] are wanted")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        need(w is None or w.dtype is torch.float32 and w.shape == (hd,) and w.is_contiguous() and w.device == dev,
             f"{name}: a contiguous float32 [{hd}] on {dev} is wanted")
    int32(positions, "positions", dev, (q.shape[0],))
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    pair = lambda t: _PAIR(0, 0) if t is None else _PAIR(t.stride(0), t.stride(1))  # noqa: E731
    return QkRope(dtype_of(q, "q"), q.shape[0], q.shape[1], k.shape[1], hd, 2 * cos.shape[1], 1 if interleaved else 0,
                  q.data_ptr(), pair(q), ptr(q_out), pair(q_out), k.data_ptr(), pair(k), ptr(k_out), pair(k_out),
                  ptr(q_weight), ptr(k_weight), eps, cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr())


def qk_norm_rope(q, k, positions, cos, sin, q_weight=None, k_weight=None, eps: float = 1e-6, interleaved: bool = False,
                 q_out=None, k_out=None):
    """(q_out, k_out): q [tokens, n_heads, head_dim] and k [tokens,
    n_kv_heads, head_dim] normalised per head (where a weight is given) and
    rotated by positions [tokens].  Inputs may be strided views of one packed
    matrix; outputs may be the inputs.  Tokens whose position lies outside the
    tables leave their output rows as they were."""
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q_out is None else q_out
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device) if k_out is None else k_out
    a = _args(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved, q_out, k_out)
    ctx = Context.get(q.device.index)
    check(_lib.lib().rq_qk_norm_rope(ctx.handle, ctypes.byref(a), stream_of(q.device)))
    return q_out, k_out


def qk_norm_rope_append(cache, q, k, v, positions, slots, cos, sin, q_weight=None, k_weight=None, eps: float = 1e-6,
                        interleaved: bool = False, q_out=None):
    """q_out as above; the normalised, rotated k and v go into ``slots`` of
    the KV4Cache in the same launch."""
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q_out is None else q_out
    a = _args(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved, q_out, None)
    need(q.device == cache.device, f"q: on {q.device}, the cache on {cache.device}")
    cache._rows(k, "k", cache.n_kv_heads)
    cache._rows(v, "v", cache.n_kv_heads)
    need(v.dtype == k.dtype and v.shape == k.shape, "v: the shape and type of k are wanted")
    int32(slots, "slots", cache.device, (q.shape[0],))
    check(_lib.lib().rq_qk_norm_rope_append(cache.handle, ctypes.byref(a), v.data_ptr(),
                                            _PAIR(v.stride(0), v.stride(1)), slots.data_ptr(), stream_of(cache.device)))
    return q_out
