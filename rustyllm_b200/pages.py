"""Page tables and slot maps of a paged cache, built on the GPU from the
lengths of a batch's requests (``rq_pages_extend`` / ``rq_pages_release`` of
include/rq.h).  The reference keeps one contiguous cache per sequence and
rolls its length back on the host (src/streaming_quantized.rs:603-609)."""
from __future__ import annotations

from collections import namedtuple

import torch

from . import _lib
from ._lib import check
from .kv4 import int32, refuse, stream_of
from .linear import Context

Extended = namedtuple("Extended", "free kv_lens cu_new positions slots")


def _table(table, batch: int):
    if not (isinstance(table, torch.Tensor) and table.is_cuda and table.dtype is torch.int32 and table.dim() == 2
            and table.shape[0] == batch and (table.shape[1] < 2 or table.stride(1) == 1)):
        refuse(f"table: a CUDA int32 [{batch}, width] with contiguous rows is wanted")
    return table.device


def pages_extend(ctx_lens, new_lens, table, ring, free, page_size: int, n_tokens: int, free_out=None, kv_lens_out=None):
    """Takes the pages that new_lens [batch] more tokens on top of ctx_lens
    [batch] need from the ring of free pages into ``table`` [batch, width], in
    place, and returns (free, kv_lens, cu_new, positions, slots): the ring's
    new state {head, free, short} (``free_out``, which may be ``free``), the
    new lengths (``kv_lens_out``, which may be ctx_lens), the offsets of the
    new tokens [batch + 1], and position and slot of each of n_tokens rows (-1
    for padding and for tokens that no page is left for)."""
    batch = new_lens.shape[0]
    dev = _table(table, batch)
    int32(ctx_lens, "ctx_lens", dev, batch)
    int32(new_lens, "new_lens", dev, batch)
    int32(ring, "ring", dev)
    int32(free, "free", dev, 3)
    # one allocation: state, lengths, offsets, positions, slots
    buf = torch.empty(4 + 2 * batch + 2 * n_tokens, dtype=torch.int32, device=dev)
    state, kv, cu, pos, slots = buf.split_with_sizes((3, batch, batch + 1, n_tokens, n_tokens))
    if free_out is None:
        free_out = state
    else:
        int32(free_out, "free_out", dev, 3)
    if kv_lens_out is None:
        kv_lens_out = kv
    else:
        int32(kv_lens_out, "kv_lens_out", dev, batch)
    base = buf.data_ptr() + 4 * (3 + batch)
    at = base + 4 * (batch + 1)
    check(_lib.lib().rq_pages_extend(
        Context.get(dev.index).handle, batch, page_size, ctx_lens.data_ptr(), new_lens.data_ptr(), table.data_ptr(),
        table.stride(0), table.shape[1], ring.data_ptr(), ring.shape[0], free.data_ptr(), free_out.data_ptr(),
        kv_lens_out.data_ptr(), base, at, at + 4 * n_tokens, n_tokens, stream_of(dev)))
    return Extended(free_out, kv_lens_out, cu, pos, slots)


def pages_release(held_lens, keep_lens, table, ring, free, page_size: int) -> None:
    """Gives the pages behind the first keep_lens [batch] of held_lens [batch]
    positions back to the ring; table, ring and free change in place."""
    batch = held_lens.shape[0]
    dev = _table(table, batch)
    int32(held_lens, "held_lens", dev, batch)
    int32(keep_lens, "keep_lens", dev, batch)
    int32(ring, "ring", dev)
    int32(free, "free", dev, 3)
    check(_lib.lib().rq_pages_release(
        Context.get(dev.index).handle, batch, page_size, held_lens.data_ptr(), keep_lens.data_ptr(), table.data_ptr(),
        table.stride(0), table.shape[1], ring.data_ptr(), ring.shape[0], free.data_ptr(), stream_of(dev)))


class PageTable:
    """The tables of up to ``batch`` requests over a pool of n_pages pages,
    all on the device: ``extend`` before a step, ``release`` when a request
    ends or drafted tokens are rolled back."""

    def __init__(self, batch: int, width: int, n_pages: int, page_size: int, device: int = 0):
        dev = torch.device("cuda", device)
        self.page_size = page_size
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.ring = torch.arange(n_pages, dtype=torch.int32, device=dev)
        self.free = torch.tensor([0, n_pages, 0], dtype=torch.int32, device=dev)

    def extend(self, new_lens, n_tokens: int) -> Extended:
        """Room for new_lens [batch] more tokens (n_tokens rows in all, the
        rest padding); lens grows by new_lens."""
        return pages_extend(self.lens, new_lens, self.table, self.ring, self.free, self.page_size, n_tokens,
                            free_out=self.free, kv_lens_out=self.lens)

    def release(self, keep_lens) -> None:
        """Keeps the first keep_lens [batch] positions of every request."""
        pages_release(self.lens, keep_lens, self.table, self.ring, self.free, self.page_size)
        torch.minimum(self.lens, keep_lens.clamp(min=0), out=self.lens)
