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
from .kv4 import _PAIR, dtype_of, int32, refuse, rows, stream_of
from .linear import Context


def rope_tables(max_pos: int, rot_dim: int, theta: float = 10000.0, device: int = 0):
    """(cos, sin) f32 [max_pos, rot_dim / 2], the angles taken in 64 bits."""
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    a = torch.arange(max_pos, dtype=torch.float64)[:, None] * theta ** (-i / max(rot_dim, 1))
    return a.cos().float().to(f"cuda:{device}"), a.sin().float().to(f"cuda:{device}")


def _args(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved, q_out, k_out, append):
    """The checked rq_qk_rope; outputs that are None are made (k_out not where
    the keys go into a cache)."""
    if not (isinstance(q, torch.Tensor) and isinstance(k, torch.Tensor) and q.is_cuda and q.dim() == 3 and k.dim() == 3
            and q.dtype == k.dtype and q.shape[0] == k.shape[0]):
        refuse("q, k: [tokens, heads, head_dim] of one type on one CUDA device are wanted")
    dev, n, heads, hd, kv = q.device, q.shape[0], q.shape[1], q.shape[2], k.shape[1]
    rows(q, "q", heads, hd, dev)
    rows(k, "k", kv, hd, dev)
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        rows(q_out, "q_out", heads, hd, dev)
        if q_out.dtype != q.dtype or q_out.shape[0] != n:
            refuse("q_out: the shape and type of q are wanted")
    if k_out is not None:
        rows(k_out, "k_out", kv, hd, dev)
        if k_out.dtype != k.dtype or k_out.shape[0] != n:
            refuse("k_out: the shape and type of k are wanted")
    elif not append:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    f32 = torch.float32
    if not (cos.dtype is f32 and sin.dtype is f32 and cos.dim() == 2 and cos.shape == sin.shape and cos.is_contiguous()
            and sin.is_contiguous() and cos.device == dev and sin.device == dev):
        refuse(f"cos, sin: contiguous float32 [max_pos, rot_dim / 2] on {dev} are wanted")
    for w in (q_weight, k_weight):
        if w is not None and not (w.dtype is f32 and w.shape == (hd,) and w.is_contiguous() and w.device == dev):
            refuse(f"q_weight, k_weight: contiguous float32 [{hd}] on {dev} are wanted")
    int32(positions, "positions", dev, n)
    none = k_out is None
    return QkRope(dtype_of(q, "q"), n, heads, kv, hd, 2 * cos.shape[1], 1 if interleaved else 0,
                  q.data_ptr(), (q.stride(0), q.stride(1)), q_out.data_ptr(), (q_out.stride(0), q_out.stride(1)),
                  k.data_ptr(), (k.stride(0), k.stride(1)), None if none else k_out.data_ptr(),
                  (0, 0) if none else (k_out.stride(0), k_out.stride(1)),
                  None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), eps,
                  cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr()), q_out, k_out


def qk_norm_rope(q, k, positions, cos, sin, q_weight=None, k_weight=None, eps: float = 1e-6, interleaved: bool = False,
                 q_out=None, k_out=None):
    """(q_out, k_out): q [tokens, n_heads, head_dim] and k [tokens,
    n_kv_heads, head_dim] normalised per head (where a weight is given) and
    rotated by positions [tokens].  Inputs may be strided views of one packed
    matrix; outputs may be the inputs.  Tokens whose position lies outside the
    tables leave their output rows as they were."""
    a, q_out, k_out = _args(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved, q_out, k_out, False)
    dev = q.device
    check(_lib.lib().rq_qk_norm_rope(Context.get(dev.index).handle, ctypes.byref(a), stream_of(dev)))
    return q_out, k_out


def qk_norm_rope_append(cache, q, k, v, positions, slots, cos, sin, q_weight=None, k_weight=None, eps: float = 1e-6,
                        interleaved: bool = False, q_out=None):
    """q_out as above; the normalised, rotated k and v go into ``slots`` of
    the KV4Cache in the same launch."""
    dev = cache.device
    rows(k, "k", cache.n_kv_heads, cache.head_dim, dev)
    rows(v, "v", cache.n_kv_heads, cache.head_dim, dev)
    if v.dtype != k.dtype or v.shape != k.shape:
        refuse("v: the shape and type of k are wanted")
    a, q_out, _ = _args(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved, q_out, None, True)
    int32(slots, "slots", dev, q.shape[0])
    check(_lib.lib().rq_qk_norm_rope_append(cache.handle, ctypes.byref(a), v.data_ptr(),
                                            _PAIR(v.stride(0), v.stride(1)), slots.data_ptr(), stream_of(dev)))
    return q_out
