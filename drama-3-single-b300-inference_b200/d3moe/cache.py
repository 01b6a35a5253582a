"""Pages of a cache: copying them in all layers at once, and who holds which.

  copy_pages(pool, src, dst, page_dim)   pool[..., dst, ...] = pool[..., src, ...]
  PagedCache                             sequences that grow, fork, end and are compacted

copy_pages moves any pool of equal pages, slots of recurrent state among them.
The reference keeps one fixed run of pages per request slot (src/drama3/model.py:
67-76); a sequence here takes pages as it grows, and forks of it share the full
ones.
"""

from __future__ import annotations

import heapq

import torch

from . import _lib


def copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, page_dim: int = 0, *,
               status: torch.Tensor | None = None) -> None:
    """pool.select(page_dim, dst[i]) = pool.select(page_dim, src[i]) for all i, in
    place, any dtype. The axes behind page_dim must be contiguous (a page is one
    run of bytes), those before it must step evenly (planes: layers, or layers
    and k / v). src and dst int32 [n] on the device; a negative number skips its
    pair, one past the pool too, with status set to D3_STATUS_BAD_ROW. No page
    may be both copied from and copied to in one call, nor copied to twice."""
    _lib.native().copy_pages(pool, src, dst, page_dim, status)


class PagedCache:
    """Keys and values of several attention layers in one pool [layers, 2, pages,
    page_size, heads, dim], and the host's record of which sequence holds which
    pages. `table` int32 [sequences, pages per sequence] on the device is what
    paged_attention and kv_append read; row i belongs to sequence i. Every change
    of the record is written to it on the current stream.

      seq = cache.new()          an empty sequence
      cache.extend(seq, n)       room for n more tokens (write them with kv_append)
      child = cache.fork(seq)    shares the full pages; a part-filled last page is copied (tokens that
                                 have room but are not written yet: see fork)
      cache.free(seq)            gives back the pages no other sequence holds
      cache.compact()            moves the pages in use to the lowest numbers
    """

    def __init__(self, layers: int, pages: int, page_size: int, heads: int, dim: int, max_sequences: int,
                 max_len: int, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        self.page_size = page_size
        self.pool = torch.zeros((layers, 2, pages, page_size, heads, dim), dtype=dtype, device=device)
        self.table = torch.zeros((max_sequences, -(-max_len // page_size)), dtype=torch.int32, device=device)
        self.lens: list[int | None] = [None] * max_sequences  # None: no such sequence
        self._pages: list[list[int]] = [[] for _ in range(max_sequences)]
        self._holders = [0] * pages
        self._spare = list(range(pages))  # a heap: the lowest number is taken first

    def k(self, layer: int) -> torch.Tensor:
        return self.pool[layer, 0]

    def v(self, layer: int) -> torch.Tensor:
        return self.pool[layer, 1]

    @property
    def free_pages(self) -> int:
        return len(self._spare)

    def _take(self, n: int) -> list[int]:
        if n > len(self._spare):
            raise RuntimeError(f"the cache has {len(self._spare)} free pages, {n} are needed")
        got = [heapq.heappop(self._spare) for _ in range(n)]
        for p in got:
            self._holders[p] = 1
        return got

    def _drop(self, page: int) -> None:
        self._holders[page] -= 1
        if self._holders[page] == 0:
            heapq.heappush(self._spare, page)

    def _alive(self, seq: int) -> None:
        if not 0 <= seq < len(self.lens) or self.lens[seq] is None:
            raise ValueError(f"there is no sequence {seq}")

    def _write_row(self, seq: int, first: int = 0) -> None:
        pages = self._pages[seq][first:]
        if pages:
            self.table[seq, first:first + len(pages)] = torch.tensor(pages, dtype=torch.int32)

    def _copy(self, src: list[int], dst: list[int]) -> None:
        at = dict(dtype=torch.int32, device=self.pool.device)
        copy_pages(self.pool, torch.tensor(src, **at), torch.tensor(dst, **at), 2)

    def new(self) -> int:
        for seq, n in enumerate(self.lens):
            if n is None:
                self.lens[seq] = 0
                return seq
        raise RuntimeError("every sequence of the cache is in use")

    def extend(self, seq: int, tokens: int) -> range:
        """Room for `tokens` more; returns their positions."""
        self._alive(seq)
        if tokens < 0:
            raise ValueError("tokens must not be negative")
        n, pages = self.lens[seq], self._pages[seq]
        need = -(-(n + tokens) // self.page_size)
        if need > self.table.shape[1]:
            raise ValueError(f"a sequence holds at most {self.table.shape[1] * self.page_size} tokens")
        first = len(pages)
        pages += self._take(max(0, need - first))
        self.lens[seq] = n + tokens
        self._write_row(seq, first)
        return range(n, n + tokens)

    def fork(self, seq: int, written: int | None = None) -> int:
        """A new sequence with the same tokens. No page that either may still write
        is shared: a part-filled last page gets its copy here. `written`: how many of
        the sequence's tokens have been written (on the current stream) so far; by
        default all that extend made room for. Pages that hold others are the child's
        own, so each of the two writes its own tokens from there on."""
        self._alive(seq)
        if written is None:
            written = self.lens[seq]
        if not 0 <= written <= self.lens[seq]:
            raise ValueError(f"sequence {seq} has {self.lens[seq]} tokens, {written} cannot have been written")
        full = written // self.page_size
        rest = self._pages[seq][full:]  # the first of them may be part-filled, the others are not written yet
        part = rest[:written % self.page_size > 0]
        child = self.new()
        try:
            copies = self._take(len(rest))
        except RuntimeError:
            self.lens[child] = None
            raise
        shared = self._pages[seq][:full]
        for p in shared:
            self._holders[p] += 1
        self._pages[child] = shared + copies
        self.lens[child] = self.lens[seq]
        if part:
            self._copy(part, copies[:1])
        self._write_row(child)
        return child

    def free(self, seq: int) -> None:
        self._alive(seq)
        for p in self._pages[seq]:
            self._drop(p)
        self._pages[seq] = []
        self.lens[seq] = None

    def compact(self) -> int:
        """Moves the pages in use to the lowest numbers; returns how many moved."""
        used = [p for p, n in enumerate(self._holders) if n]
        src = [p for p in used if p >= len(used)]
        if not src:
            return 0
        dst = sorted(p for p in self._spare if p < len(used))  # as many, and none of them in use
        self._copy(src, dst)
        to = dict(zip(src, dst))
        for a, b in to.items():
            self._holders[b], self._holders[a] = self._holders[a], 0
        self._spare = list(range(len(used), len(self._holders)))
        for seq, pages in enumerate(self._pages):
            if any(p in to for p in pages):
                self._pages[seq] = [to.get(p, p) for p in pages]
                self._write_row(seq)
        return len(src)
