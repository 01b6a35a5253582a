"""Copying pages of a cache (or slots of recurrent state) in all layers at once.

  copy_pages(pool, src, dst, page_dim)   pool[..., dst, ...] = pool[..., src, ...]
"""

from __future__ import annotations

import torch

from ._lib import call
from .attention import _index_ptr, _need_cuda, _status_ptr, _stream


def copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, page_dim: int = 0, *,
               status: torch.Tensor | None = None) -> None:
    """pool.select(page_dim, dst[i]) = pool.select(page_dim, src[i]) for all i, in
    place, any dtype. The axes behind page_dim must be contiguous (a page is one
    run of bytes), those before it must step evenly (planes: layers, or layers
    and k / v). src and dst int32 [n] on the device; a negative number skips its
    pair, one past the pool too, with status set to D3_STATUS_BAD_ROW. No page
    may be both copied from and copied to in one call, nor copied to twice."""
    dev = pool.get_device()
    _need_cuda(dev)
    shape, strides = pool.shape, pool.stride()
    if not 0 <= page_dim < len(shape):
        raise ValueError("page_dim must be an axis of pool")
    elements = 1
    for i in range(len(shape) - 1, page_dim, -1):
        if shape[i] != 1 and strides[i] != elements:
            raise ValueError("the axes behind page_dim must be contiguous")
        elements *= shape[i]
    planes, plane_stride = 1, 0
    for i in range(page_dim - 1, -1, -1):
        if shape[i] == 1:
            continue
        if planes == 1:
            plane_stride = strides[i]
        elif strides[i] != planes * plane_stride:
            raise ValueError("the axes before page_dim must step evenly")
        planes *= shape[i]
    n, size = src.numel(), pool.element_size()
    call("d3_copy_pages", pool.data_ptr(), planes, plane_stride * size, shape[page_dim],
         strides[page_dim] * size, elements * size, _index_ptr(src, n, dev, "src"),
         _index_ptr(dst, n, dev, "dst"), n, _status_ptr(status, dev), _stream(dev))
