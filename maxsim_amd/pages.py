"""Pages of a cache's pool: which sequences hold which, decided on the device.

``Int4KVCache`` takes page tables and lengths as they are.  ``CachePages`` keeps them
for a batch of slots: a table of pages, a length per sequence, and a stack of the
pages that no sequence holds.  One call per step moves all of it, without a copy to
the host, and says where the new rows go::

    pages = CachePages(num_pages, batch, max_pages, page_size=64)
    offsets, positions, slots = pages.update(new, rows=rows)
    q, k = rotary(q, k, positions)
    cache.append(k, v, pages.table, pages.lengths, offsets)
    out = cache.attend(q, pages.table, pages.lengths, offsets)

A sequence that ends is cut to length 0, drafted tokens that were given up are cut off
with the next step's call: ``pages.update(new, lengths=cache.keep(...), rows=rows)``.
"""
from __future__ import annotations

import numbers

from maxsim_amd import _native
from maxsim_amd.kvcache import _cuda_device


class CachePages:
    """Tables of up to max_pages pages for batch sequences, out of num_pages pages of
    page_size tokens (a power of two from 16 up), all free at first.

    ``table`` int32 [batch, max_pages] (-1 behind a sequence's pages), ``lengths``
    int32 [batch], ``free`` int32 [num_pages] (the stack, -1 behind it) and
    ``free_count`` int32 [1] are the state itself: a program saves and restores it
    through them.  Each page is in one place of them.
    """

    def __init__(self, num_pages: int, batch: int, max_pages: int, page_size: int = 64, device="cuda"):
        import torch

        num_pages, batch, max_pages, page_size = int(num_pages), int(batch), int(max_pages), int(page_size)
        if num_pages < 1 or batch < 1 or max_pages < 1:
            raise ValueError("num_pages, batch and max_pages must be positive")
        if page_size < 16 or page_size > 65536 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two from 16 to 65536")
        if num_pages >= 2**31 or batch > 2**26 or batch * max_pages >= 2**31 or max_pages * page_size >= 2**31 - 4096:
            raise NotImplementedError("less than 2^31 pages, table entries and tokens of a sequence (2^31 - 4096)")
        self.device = _cuda_device(device)
        self._calls = _native.tensor_calls()
        self._table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=self.device)
        self._lengths = torch.zeros(batch, dtype=torch.int32, device=self.device)
        # Page 0 is on top.
        self._free = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=self.device)
        self._free_count = torch.full((1,), num_pages, dtype=torch.int32, device=self.device)
        self.num_pages, self.batch, self.max_pages, self.page_size = num_pages, batch, max_pages, page_size
        self._handle = self._calls.pages(self._table, self._lengths, self._free, self._free_count, page_size)

    @property
    def table(self):
        return self._table

    @property
    def lengths(self):
        return self._lengths

    @property
    def free(self):
        return self._free

    @property
    def free_count(self):
        return self._free_count

    def update(self, new=None, lengths=None, *, rows=None):
        """Cuts every sequence to ``lengths`` (int32 [batch]; larger numbers cut
        nothing), puts the pages behind on the stack, and gives it ``new`` tokens (int32
        [batch], or a number for all) with pages from the stack.

        Sequences are served in their order.  One gets none of its tokens where they do
        not fit its row of the table, where the tokens asked for up to it are more than
        ``rows``, or where it needs pages and those asked for up to it are more than
        there are; its length tells.

        Returns (offsets int32 [batch + 1], positions int32 [rows], slots int64 [rows])
        of the tokens given, packed by sequence: their positions one after another (a
        draft of a tree stands at its sequence's first one plus its depth), and page *
        page_size + place in the page; -1 behind the last.  ``rows`` is the capacity for them;
        without it a tensor's sum is fetched from the device.  Enqueued on the current
        stream; can be captured in a HIP graph."""
        if isinstance(new, numbers.Integral):
            import torch

            new = int(new)
            if new < 0:
                raise ValueError("new must not be negative")
            if rows is None:
                rows = self.batch * new
            new = torch.full((self.batch,), min(new, 2**31 - 1), dtype=torch.int32, device=self.device)
        if rows is None:
            if new is not None and not hasattr(new, "clamp"):
                raise ValueError("new must be a tensor or a number")
            rows = 0 if new is None else int(new.clamp(min=0).sum())
        return self._calls.update(self._handle, new, lengths, rows)
