"""A paged key/value cache held in 4 bits and attention over it
(``rq_kv4_*`` of include/rq.h).  No counterpart in the reference, whose cache
is one contiguous f32 buffer per layer (src/streaming_quantized.rs:93-152).

All arguments are CUDA tensors on the cache's device; calls run on torch's
current stream and read nothing back, so they can be captured in CUDA graphs.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import DTYPES, Kv4Query, RqError, check
from .linear import Context

_PAIR = ctypes.c_int64 * 2


def stream_of(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def need(ok, msg: str) -> None:
    if not ok:
        raise RqError(1, msg)


def dtype_of(t, name: str) -> int:
    d = DTYPES.get(t.dtype)
    if d is None:
        raise RqError(3, f"{name}: {t.dtype} (float32, float16 or bfloat16)")
    return d


def int32(t, name: str, device, shape=None):
    """t as it is, checked: int32, contiguous, on the device."""
    need(isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.device == device and t.is_contiguous()
         and (shape is None or tuple(t.shape) == shape),
         f"{name}: a contiguous int32 tensor{'' if shape is None else f' of shape {list(shape)}'} on {device} is wanted")
    return t


class KV4Cache:
    def __init__(self, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, device: int = 0):
        self.ctx = Context.get(device)
        self.device = torch.device("cuda", device)
        h = ctypes.c_void_p()
        self.handle = None
        check(_lib.lib().rq_kv4_create(self.ctx.handle, n_pages, page_size, n_kv_heads, head_dim, ctypes.byref(h)))
        self.handle = h
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = n_pages, page_size, n_kv_heads, head_dim

    def device_bytes(self) -> int:
        n = ctypes.c_size_t()
        check(_lib.lib().rq_kv4_info(self.handle, None, None, None, None, ctypes.byref(n)))
        return n.value

    def _rows(self, x, name: str, heads: int):
        need(isinstance(x, torch.Tensor) and x.dim() == 3 and x.shape[1] == heads and x.shape[2] == self.head_dim
             and x.device == self.device and (x.stride(2) == 1 or x.shape[2] == 1),
             f"{name}: [tokens, {heads}, {self.head_dim}] on {self.device} with contiguous elements is wanted")
        return x

    def append(self, k, v, slots) -> None:
        """Quantizes k, v [n, n_kv_heads, head_dim] (float32, float16 or
        bfloat16; any strides of token and head) into slots [n] (int32; those
        outside the cache, -1 for padding, are skipped).  The slots of one
        call must differ."""
        self._rows(k, "k", self.n_kv_heads)
        self._rows(v, "v", self.n_kv_heads)
        need(k.dtype == v.dtype and k.shape[0] == v.shape[0], "append: k and v differ in type or length")
        int32(slots, "slots", self.device, (k.shape[0],))
        check(_lib.lib().rq_kv4_append(self.handle, dtype_of(k, "k"), k.data_ptr(), _PAIR(k.stride(0), k.stride(1)),
                                       v.data_ptr(), _PAIR(v.stride(0), v.stride(1)), slots.data_ptr(), k.shape[0],
                                       stream_of(self.device)))

    def read(self, slots, dtype=torch.float32):
        """(k, v) [n, n_kv_heads, head_dim]: the values held in slots [n]."""
        int32(slots, "slots", self.device, (slots.shape[0],))
        n = slots.shape[0]
        k, v = torch.empty((2, n, self.n_kv_heads, self.head_dim), dtype=dtype, device=self.device).unbind(0)
        check(_lib.lib().rq_kv4_read(self.handle, slots.data_ptr(), n, dtype_of(k, "dtype"), k.data_ptr(), v.data_ptr(),
                                     stream_of(self.device)))
        return k, v

    def attention(self, q, block_table, kv_lens, cu_q=None, max_q: int = 1, scale: float | None = None, window: int = 0,
                  out=None, max_len: int = 0):
        """Attention of the newest tokens of each sequence over the cache:
        q [tokens, n_heads, head_dim], block_table [batch, width] and kv_lens
        [batch] int32; without cu_q one query a sequence, with it (int32
        [batch + 1]) the rows cu_q[b] .. cu_q[b + 1] - 1, at most max_q each.
        Causal; window > 0 limits a query to that many newest positions.
        Rows that belong to no sequence are left as they are in ``out`` (and
        undefined where ``out`` is not given).  max_len, an upper bound of
        kv_lens, helps to split the work; see include/rq.h for the rest."""
        need(isinstance(q, torch.Tensor) and q.dim() == 3, "q: [tokens, heads, head_dim] is wanted")
        self._rows(q, "q", q.shape[1])
        dev = self.device
        need(isinstance(block_table, torch.Tensor) and block_table.dtype is torch.int32 and block_table.dim() == 2
             and block_table.device == dev and (block_table.shape[1] < 2 or block_table.stride(1) == 1),
             f"block_table: int32 [batch, width] with contiguous rows on {dev} is wanted")
        batch = block_table.shape[0]
        int32(kv_lens, "kv_lens", dev, (batch,))
        if cu_q is not None:
            int32(cu_q, "cu_q", dev, (batch + 1,))
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        else:
            self._rows(out, "out", q.shape[1])
            need(out.dtype == q.dtype and out.shape == q.shape, "out: the shape and type of q are wanted")
        a = Kv4Query(dtype_of(q, "q"), q.data_ptr(), _PAIR(q.stride(0), q.stride(1)), out.data_ptr(),
                     _PAIR(out.stride(0), out.stride(1)), q.shape[0], q.shape[1], batch, max_q,
                     None if cu_q is None else cu_q.data_ptr(), kv_lens.data_ptr(), block_table.data_ptr(),
                     block_table.stride(0), block_table.shape[1], max_len, window,
                     self.head_dim ** -0.5 if scale is None else scale, None, 0)
        L, ref = _lib.lib(), ctypes.byref(a)
        n = ctypes.c_size_t()
        check(L.rq_kv4_attention_workspace(self.handle, ref, ctypes.byref(n)))
        ws = None
        if n.value:
            # of the current stream's (and a captured graph's own) pool
            ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes = ws.data_ptr(), n.value
        check(L.rq_kv4_attention(self.handle, ref, stream_of(dev)))
        return out

    def close(self) -> None:
        if self.handle:
            _lib.lib().rq_kv4_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
