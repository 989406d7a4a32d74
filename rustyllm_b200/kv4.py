"""A paged key/value cache held in 4 bits and attention over it
(``rq_kv4_*`` of include/rq.h).  No counterpart in the reference, whose cache
is one contiguous f32 buffer per layer (src/streaming_quantized.rs:93-152).

All arguments are CUDA tensors on the cache's device; calls run on torch's
current stream and read nothing back, so they can be captured in CUDA graphs.
Arguments are checked and outputs allocated by the compiled binding
(csrc/rq_torch.cpp), which raises RqError.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import check
from .linear import Context

from . import _rqtorch  # isort: skip  (needs torch's libraries loaded)


class KV4Cache:
    def __init__(self, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, device: int = 0):
        self.ctx = Context.get(device)
        self.device = torch.device("cuda", device)
        h = ctypes.c_void_p()
        self.handle = None
        check(_lib.lib().rq_kv4_create(self.ctx.handle, n_pages, page_size, n_kv_heads, head_dim, ctypes.byref(h)))
        self.handle = h
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = n_pages, page_size, n_kv_heads, head_dim
        self.native = _rqtorch.Cache(h.value, n_kv_heads, head_dim, device)
        self._scale = head_dim ** -0.5

    def device_bytes(self) -> int:
        n = ctypes.c_size_t()
        check(_lib.lib().rq_kv4_info(self.handle, None, None, None, None, ctypes.byref(n)))
        return n.value

    def append(self, k, v, slots) -> None:
        """Quantizes k, v [n, n_kv_heads, head_dim] (float32, float16 or
        bfloat16; any strides of token and head) into slots [n] (int32; those
        outside the cache, -1 for padding, are skipped).  The slots of one
        call must differ."""
        _rqtorch.append(self.native, k, v, slots)

    def read(self, slots, dtype=torch.float32):
        """(k, v) [n, n_kv_heads, head_dim]: the values held in slots [n]
        (zeros for a slot outside the cache)."""
        return _rqtorch.read(self.native, slots, dtype)

    def attention(self, q, block_table, kv_lens, cu_q=None, max_q: int | None = None, scale: float | None = None, window: int = 0,
                  out=None, max_len: int = 0):
        """Attention of the newest tokens of each sequence over the cache:
        q [tokens, n_heads, head_dim], block_table [batch, width] and kv_lens
        [batch] int32; without cu_q one query a sequence, with it (int32
        [batch + 1]) the rows cu_q[b] .. cu_q[b + 1] - 1, at most max_q each
        (rows behind that are not computed; without max_q any number is, by the
        form for many rows: give it where it is small).
        Causal; window > 0 limits a query to that many newest positions.
        Rows that belong to no sequence are left as they are in ``out`` (and
        undefined where ``out`` is not given).  max_len, an upper bound of
        kv_lens, helps to split the work; see include/rq.h for the rest."""
        return _rqtorch.attention(self.native, q, block_table, kv_lens, cu_q, max_q, self._scale if scale is None else scale,
                                  window, out, max_len)

    def close(self) -> None:
        """Frees the cache; calls that use it afterwards raise RqError."""
        if self.handle:
            if hasattr(self, "native"):
                self.native.close()
            _lib.lib().rq_kv4_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
