"""Copying pages of a cache (or slots of recurrent state) in all layers at once.

  copy_pages(pool, src, dst, page_dim)   pool[..., dst, ...] = pool[..., src, ...]
"""

from __future__ import annotations

import torch

from . import _lib

_native = _lib.native()


def copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, page_dim: int = 0, *,
               status: torch.Tensor | None = None) -> None:
    """pool.select(page_dim, dst[i]) = pool.select(page_dim, src[i]) for all i, in
    place, any dtype. The axes behind page_dim must be contiguous (a page is one
    run of bytes), those before it must step evenly (planes: layers, or layers
    and k / v). src and dst int32 [n] on the device; a negative number skips its
    pair, one past the pool too, with status set to D3_STATUS_BAD_ROW. No page
    may be both copied from and copied to in one call, nor copied to twice."""
    _native.copy_pages(pool, src, dst, page_dim, status)
