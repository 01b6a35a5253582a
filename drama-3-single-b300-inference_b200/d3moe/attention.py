"""Paged key-value attention of a decode step: appending new keys and values to
their pages, and attending to them.

  kv_append(k, v, k_cache, v_cache, page_table, positions)   new rows into their pages
  paged_attention(q, k_cache, v_cache, page_table, seq_lens) one new token per sequence

A cache is a pair of [pages, page_size, heads, dim] tensors (any strides with a
contiguous last axis, so a permuted [pages, heads, page_size, dim] cache is
taken as it is) in bf16, f16, or e4m3 with f32 scales per head: the value held
is element * scale[head]. The reference's attention layers have 16 query and 2
key heads of 256 and pages of 16 tokens (src/drama3/model.py:55-141).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import D3KvCache, call
from .ops import _ptr, _stream

_DTYPES = {torch.bfloat16: _lib.D3_DTYPE_BF16, torch.float16: _lib.D3_DTYPE_F16,
           torch.float8_e4m3fn: _lib.D3_DTYPE_E4M3}


def _scale_ptr(scale, heads: int, device) -> int | None:
    if scale is None:
        return None
    if scale.dtype != torch.float32 or scale.shape != (heads,) or not scale.is_contiguous() or scale.device != device:
        raise ValueError("cache scales must be contiguous float32 [heads] on the cache's device")
    return scale.data_ptr()


def _cache_struct(k_cache, v_cache, page_table, k_scale, v_scale) -> D3KvCache:
    if not k_cache.is_cuda:
        raise ValueError("d3moe operators take CUDA tensors; there is no CPU path")
    dtype = _DTYPES.get(k_cache.dtype)
    if dtype is None or v_cache.dtype != k_cache.dtype:
        raise ValueError("k_cache and v_cache must both be bfloat16, float16 or float8_e4m3fn")
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must be [pages, page_size, heads, dim] of one shape")
    pages, page_size, heads, dim = k_cache.shape
    ks, vs = k_cache.stride(), v_cache.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("the last axis of a cache must be contiguous")
    dev = k_cache.device
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.stride(1) != 1:
        raise ValueError("page_table must be int32 [sequences, pages per sequence], rows contiguous")
    if v_cache.device != dev or page_table.device != dev:
        raise ValueError("caches and page_table must be on one device")
    if dtype != _lib.D3_DTYPE_E4M3 and (k_scale is not None or v_scale is not None):
        raise ValueError("only an e4m3 cache has scales")
    return D3KvCache(k_cache.data_ptr(), v_cache.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                     _scale_ptr(k_scale, heads, dev), _scale_ptr(v_scale, heads, dev),
                     page_table.data_ptr(), page_table.stride(0), page_table.shape[0],
                     page_table.shape[1], pages, page_size, heads, dim, dtype)


def _index_ptr(t, n: int, device, what: str) -> int:
    if t.dtype != torch.int32 or t.shape != (n,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous int32 [{n}] on the operands' device")
    return t.data_ptr()


def _status_ptr(status, device) -> int | None:
    if status is None:
        return None
    if status.dtype != torch.int32 or status.numel() < 1 or status.device != device:
        raise ValueError("status must be an int32 tensor on the operands' device")
    return status.data_ptr()


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              page_table: torch.Tensor, positions: torch.Tensor, seq_ids: torch.Tensor | None = None, *,
              k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
              status: torch.Tensor | None = None) -> None:
    """Write k, v [T, heads, dim] to their pages, in place. Token t is at
    positions[t] (int32) of sequence seq_ids[t] (int32; None: sequence t);
    negative ones are skipped. An e4m3 cache takes bf16 rows and holds
    e4m3(clamp(x / scale[head], -448, 448)). Tokens past the table or on a page
    outside the cache are not written and set status to D3_STATUS_BAD_ROW."""
    c = _cache_struct(k_cache, v_cache, page_table, k_scale, v_scale)
    want = torch.bfloat16 if c.dtype == _lib.D3_DTYPE_E4M3 else k_cache.dtype
    if k.dtype != want or v.dtype != want:
        raise ValueError(f"k and v must be {want} for a {k_cache.dtype} cache")
    T = k.shape[0]
    if k.shape != (T, c.heads, c.dim) or v.shape != k.shape:
        raise ValueError(f"k and v must be [T, {c.heads}, {c.dim}]")
    ks, vs = k.stride(), v.stride()
    if T and (ks[2] != 1 or vs[2] != 1):
        raise ValueError("the last axis of k and v must be contiguous")
    dev = k_cache.device
    if k.device != dev or v.device != dev:
        raise ValueError("k, v and the cache must be on one device")
    call("d3_kv_append", k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], _DTYPES[want], T,
         None if seq_ids is None else _index_ptr(seq_ids, T, dev, "seq_ids"),
         _index_ptr(positions, T, dev, "positions"), ctypes.byref(c), _status_ptr(status, dev), _stream(dev))


def paged_attention_workspace(batch: int, heads: int, kv_heads: int, dim: int, device) -> torch.Tensor:
    """Scratch of paged_attention for up to these sizes, for a caller that keeps it."""
    nbytes = ctypes.c_size_t()
    call("d3_paged_attention_workspace_size", batch, heads, kv_heads, dim, ctypes.byref(nbytes))
    return torch.empty(nbytes.value, dtype=torch.uint8, device=device)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    seq_lens: torch.Tensor, scale: float | None = None, *,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None, window: int = 0,
                    max_seq_len: int | None = None, out: torch.Tensor | None = None, return_lse: bool = False,
                    workspace: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """softmax(scale * q K^T) V for one new token per sequence: q [B, heads,
    dim], over the first seq_lens[b] (int32) cached tokens, or the last `window`
    of them. scale: dim**-0.5 by default. max_seq_len bounds seq_lens on the host
    (default: what the page table can hold). Returns out (q's dtype), or (out,
    lse f32 [B, heads]) with return_lse. An empty sequence gives zeros and
    lse = -inf. Nothing is read on the host, so the call can be captured."""
    c = _cache_struct(k_cache, v_cache, page_table, k_scale, v_scale)
    dev = k_cache.device
    if q.dim() != 3 or q.shape[2] != c.dim or q.device != dev:
        raise ValueError(f"q must be [B, heads, {c.dim}] on the cache's device")
    B, Hq, D = q.shape
    want = torch.bfloat16 if c.dtype == _lib.D3_DTYPE_E4M3 else k_cache.dtype
    if q.dtype != want:
        raise ValueError(f"q must be {want} for a {k_cache.dtype} cache")
    if c.sequences != B:
        raise ValueError("page_table must have one row per query")
    if out is None:
        out = torch.empty((B, Hq, D), dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev:
        raise ValueError("out must have the shape, dtype and device of q")
    qs, os_ = q.stride(), out.stride()
    if qs[2] != 1 or os_[2] != 1:
        raise ValueError("the last axis of q and out must be contiguous")
    lse = torch.empty((B, Hq), dtype=torch.float32, device=dev) if return_lse else None
    if workspace is None:
        workspace = paged_attention_workspace(B, Hq, c.heads, D, dev)
    limit = c.table_pages * c.page_size
    call("d3_paged_attention", q.data_ptr(), qs[0], qs[1], _DTYPES[want], B, Hq, ctypes.byref(c),
         _index_ptr(seq_lens, B, dev, "seq_lens"), limit if max_seq_len is None else min(max_seq_len, limit),
         window, D ** -0.5 if scale is None else scale, out.data_ptr(), os_[0], os_[1], _ptr(lse),
         workspace.data_ptr(), workspace.numel(), _status_ptr(status, dev), _stream(dev))
    return (out, lse) if return_lse else out
