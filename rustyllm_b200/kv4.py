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
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_of(device) -> int:
    """torch's current stream on the device (without a Stream object where
    torch offers that: small calls are bound by the host)."""
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def refuse(msg: str) -> None:
    raise RqError(1, msg)


def dtype_of(t, name: str) -> int:
    d = DTYPES.get(t.dtype)
    if d is None:
        raise RqError(3, f"{name}: {t.dtype} (float32, float16 or bfloat16)")
    return d


def int32(t, name: str, device, n=None) -> None:
    """Refuses what is not a contiguous int32 tensor (of n values) on the device."""
    if not (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.device == device and t.is_contiguous()
            and (n is None or t.shape == (n,))):
        refuse(f"{name}: a contiguous int32 tensor{'' if n is None else f' of {n} values'} on {device} is wanted")


def rows(x, name: str, heads: int, dim: int, device) -> None:
    """Refuses what is not [tokens, heads, dim] on the device with contiguous elements."""
    if not (isinstance(x, torch.Tensor) and x.dim() == 3 and x.shape[1] == heads and x.shape[2] == dim
            and x.device == device and (dim == 1 or x.stride(2) == 1)):
        refuse(f"{name}: [tokens, {heads}, {dim}] on {device} with contiguous elements is wanted")


class KV4Cache:
    def __init__(self, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, device: int = 0):
        self.ctx = Context.get(device)
        self.device = torch.device("cuda", device)
        h = ctypes.c_void_p()
        self.handle = None
        check(_lib.lib().rq_kv4_create(self.ctx.handle, n_pages, page_size, n_kv_heads, head_dim, ctypes.byref(h)))
        self.handle = h
        self._workspace: dict = {}
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = n_pages, page_size, n_kv_heads, head_dim

    def device_bytes(self) -> int:
        n = ctypes.c_size_t()
        check(_lib.lib().rq_kv4_info(self.handle, None, None, None, None, ctypes.byref(n)))
        return n.value

    def append(self, k, v, slots) -> None:
        """Quantizes k, v [n, n_kv_heads, head_dim] (float32, float16 or
        bfloat16; any strides of token and head) into slots [n] (int32; those
        outside the cache, -1 for padding, are skipped).  The slots of one
        call must differ."""
        dev = self.device
        rows(k, "k", self.n_kv_heads, self.head_dim, dev)
        rows(v, "v", self.n_kv_heads, self.head_dim, dev)
        n = k.shape[0]
        if k.dtype != v.dtype or v.shape[0] != n:
            refuse("append: k and v differ in type or length")
        int32(slots, "slots", dev, n)
        check(_lib.lib().rq_kv4_append(self.handle, dtype_of(k, "k"), k.data_ptr(), _PAIR(k.stride(0), k.stride(1)),
                                       v.data_ptr(), _PAIR(v.stride(0), v.stride(1)), slots.data_ptr(), n,
                                       stream_of(dev)))

    def read(self, slots, dtype=torch.float32):
        """(k, v) [n, n_kv_heads, head_dim]: the values held in slots [n]."""
        dev = self.device
        int32(slots, "slots", dev)
        n = slots.shape[0] if slots.dim() == 1 else refuse("slots: one dimension is wanted")
        kv = torch.empty((2, n, self.n_kv_heads, self.head_dim), dtype=dtype, device=dev)
        k, v = kv.unbind(0)
        check(_lib.lib().rq_kv4_read(self.handle, slots.data_ptr(), n, dtype_of(kv, "dtype"), k.data_ptr(), v.data_ptr(),
                                     stream_of(dev)))
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
        dev = self.device
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            refuse("q: [tokens, heads, head_dim] is wanted")
        n, heads = q.shape[0], q.shape[1]
        rows(q, "q", heads, self.head_dim, dev)
        if not (isinstance(block_table, torch.Tensor) and block_table.dtype is torch.int32 and block_table.dim() == 2
                and block_table.device == dev and (block_table.shape[1] < 2 or block_table.stride(1) == 1)):
            refuse(f"block_table: int32 [batch, width] with contiguous rows on {dev} is wanted")
        batch, width = block_table.shape
        int32(kv_lens, "kv_lens", dev, batch)
        cu = None
        if cu_q is not None:
            int32(cu_q, "cu_q", dev, batch + 1)
            cu = cu_q.data_ptr()
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        else:
            rows(out, "out", heads, self.head_dim, dev)
            if out.dtype != q.dtype or out.shape[0] != n:
                refuse("out: the shape and type of q are wanted")
        dt = dtype_of(q, "q")
        a = Kv4Query(dt, q.data_ptr(), (q.stride(0), q.stride(1)), out.data_ptr(), (out.stride(0), out.stride(1)), n,
                     heads, batch, max_q, cu, kv_lens.data_ptr(), block_table.data_ptr(), block_table.stride(0), width,
                     max_len, window, self.head_dim ** -0.5 if scale is None else scale, None, 0)
        L, ref = _lib.lib(), ctypes.byref(a)
        # the workspace's size follows from these alone
        key = (dt, n, heads, batch, max_q, cu is None, width, max_len, window)
        need = self._workspace.get(key)
        if need is None:
            size = ctypes.c_size_t()
            check(L.rq_kv4_attention_workspace(self.handle, ref, ctypes.byref(size)))
            if len(self._workspace) >= 4096:
                self._workspace.clear()
            need = self._workspace[key] = size.value
        if need:
            # of the current stream's (and a captured graph's own) pool
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
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
