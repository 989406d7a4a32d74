"""Norms of queries and keys per head with the position rotation in the same
pass (``rq_qk_norm_rope`` of include/rq.h), and the form that puts the keys
and values straight into a 4-bit cache.  The reference rotates without a norm
and in a pass of its own (QAttn::forward, src/streaming_quantized.rs:201-240).
"""
from __future__ import annotations

import torch

from .linear import Context

from . import _rqtorch  # isort: skip  (needs torch's libraries loaded)


def rope_tables(max_pos: int, rot_dim: int, theta: float = 10000.0, device: int = 0):
    """(cos, sin) f32 [max_pos, rot_dim / 2], the angles taken in 64 bits."""
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    a = torch.arange(max_pos, dtype=torch.float64)[:, None] * theta ** (-i / max(rot_dim, 1))
    return a.cos().float().to(f"cuda:{device}"), a.sin().float().to(f"cuda:{device}")


def qk_norm_rope(q, k, positions, cos, sin, q_weight=None, k_weight=None, eps: float = 1e-6, interleaved: bool = False,
                 q_out=None, k_out=None):
    """(q_out, k_out): q [tokens, n_heads, head_dim] and k [tokens,
    n_kv_heads, head_dim] normalised per head (where a weight is given) and
    rotated by positions [tokens].  Inputs may be strided views of one packed
    matrix; outputs may be the inputs.  Tokens whose position lies outside the
    tables leave their output rows as they were."""
    return _rqtorch.qk_norm_rope(Context.of(q), q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved, q_out, k_out)


def qk_norm_rope_append(cache, q, k, v, positions, slots, cos, sin, q_weight=None, k_weight=None, eps: float = 1e-6,
                        interleaved: bool = False, q_out=None):
    """q_out as above; the normalised, rotated k and v go into ``slots`` of
    the KV4Cache in the same launch."""
    return _rqtorch.qk_norm_rope_append(cache.native, q, k, v, positions, slots, cos, sin, q_weight, k_weight, eps,
                                        interleaved, q_out)
