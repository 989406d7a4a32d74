"""Page tables and slot maps of a paged cache, built on the GPU from the
lengths of a batch's requests (``rq_pages_extend`` / ``rq_pages_release`` of
include/rq.h).  The reference keeps one contiguous cache per sequence and
rolls its length back on the host (src/streaming_quantized.rs:603-609)."""
from __future__ import annotations

from collections import namedtuple

import torch

from .linear import Context

from . import _rqtorch  # isort: skip  (needs torch's libraries loaded)

Extended = namedtuple("Extended", "free kv_lens cu_new positions slots")


def pages_extend(ctx_lens, new_lens, table, ring, free, page_size: int, n_tokens: int, free_out=None, kv_lens_out=None):
    """Takes the pages that new_lens [batch] more tokens on top of ctx_lens
    [batch] need from the ring of free pages into ``table`` [batch, width], in
    place, and returns (free, kv_lens, cu_new, positions, slots): the ring's
    new state {head, free, short} (``free_out``, which may be ``free``), the
    new lengths (``kv_lens_out``, which may be ctx_lens), the offsets of the
    new tokens [batch + 1], and position and slot of each of n_tokens rows (-1
    for padding and for tokens that no page is left for)."""
    return Extended(*_rqtorch.pages_extend(Context.of(new_lens), ctx_lens, new_lens, table, ring, free, page_size, n_tokens,
                                           free_out, kv_lens_out))


def pages_release(held_lens, keep_lens, table, ring, free, page_size: int) -> None:
    """Gives the pages behind the first keep_lens [batch] of held_lens [batch]
    positions back to the ring; table, ring and free change in place."""
    _rqtorch.pages_release(Context.of(held_lens), held_lens, keep_lens, table, ring, free, page_size)


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
