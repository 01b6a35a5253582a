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
import functools

import torch

from . import _lib
from ._lib import D3KvCache, call

_DTYPES = {torch.bfloat16: _lib.D3_DTYPE_BF16, torch.float16: _lib.D3_DTYPE_F16,
           torch.float8_e4m3fn: _lib.D3_DTYPE_E4M3}

# A decode step calls these operators once per layer on little data, so the host's
# time counts: devices are compared by index and each property is fetched once.
_stream = torch._C._cuda_getCurrentRawStream  # device index -> cudaStream_t of the current stream


def _need_cuda(index: int) -> None:
    if index < 0:
        raise ValueError("d3moe operators take CUDA tensors; there is no CPU path")


def _scale_ptr(scale, heads: int, dev: int) -> int | None:
    if scale is None:
        return None
    if (scale.dtype is not torch.float32 or scale.shape != (heads,) or not scale.is_contiguous()
            or scale.get_device() != dev):
        raise ValueError("cache scales must be contiguous float32 [heads] on the cache's device")
    return scale.data_ptr()


def _cache_struct(k_cache, v_cache, page_table, k_scale, v_scale, dev: int) -> D3KvCache:
    _need_cuda(dev)
    dtype = _DTYPES.get(k_cache.dtype)
    if dtype is None or v_cache.dtype is not k_cache.dtype:
        raise ValueError("k_cache and v_cache must both be bfloat16, float16 or float8_e4m3fn")
    shape, rows = k_cache.shape, page_table.shape
    if len(shape) != 4 or shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must be [pages, page_size, heads, dim] of one shape")
    pages, page_size, heads, dim = shape
    k0, k1, k2, k3 = k_cache.stride()
    v0, v1, v2, v3 = v_cache.stride()
    if k3 != 1 or v3 != 1:
        raise ValueError("the last axis of a cache must be contiguous")
    if page_table.dtype is not torch.int32 or len(rows) != 2:
        raise ValueError("page_table must be int32 [sequences, pages per sequence], rows contiguous")
    t0, t1 = page_table.stride()
    if t1 != 1:
        raise ValueError("page_table must be int32 [sequences, pages per sequence], rows contiguous")
    if v_cache.get_device() != dev or page_table.get_device() != dev:
        raise ValueError("caches and page_table must be on one device")
    if k_scale is not None or v_scale is not None:
        if dtype != _lib.D3_DTYPE_E4M3:
            raise ValueError("only an e4m3 cache has scales")
        k_scale, v_scale = _scale_ptr(k_scale, heads, dev), _scale_ptr(v_scale, heads, dev)
    return D3KvCache(k_cache.data_ptr(), v_cache.data_ptr(), k0, k1, k2, v0, v1, v2, k_scale, v_scale,
                     page_table.data_ptr(), t0, rows[0], rows[1], pages, page_size, heads, dim, dtype)


def _index_ptr(t, n: int, dev: int, what: str) -> int:
    if t.dtype is not torch.int32 or t.shape != (n,) or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous int32 [{n}] on the operands' device")
    return t.data_ptr()


def _status_ptr(status, dev: int) -> int | None:
    if status is None:
        return None
    if status.dtype is not torch.int32 or status.numel() < 1 or status.get_device() != dev:
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
    dev = k_cache.get_device()
    c = _cache_struct(k_cache, v_cache, page_table, k_scale, v_scale, dev)
    want = k_cache.dtype if c.dtype != _lib.D3_DTYPE_E4M3 else torch.bfloat16
    if k.dtype is not want or v.dtype is not want:
        raise ValueError(f"k and v must be {want} for a {k_cache.dtype} cache")
    shape = k.shape
    if len(shape) != 3 or shape[1:] != k_cache.shape[2:] or v.shape != shape:
        raise ValueError(f"k and v must be [T, {c.heads}, {c.dim}]")
    T = shape[0]
    k0, k1, k2 = k.stride()
    v0, v1, v2 = v.stride()
    if T and (k2 != 1 or v2 != 1):
        raise ValueError("the last axis of k and v must be contiguous")
    if k.get_device() != dev or v.get_device() != dev:
        raise ValueError("k, v and the cache must be on one device")
    call("d3_kv_append", k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, _DTYPES[want], T,
         None if seq_ids is None else _index_ptr(seq_ids, T, dev, "seq_ids"),
         _index_ptr(positions, T, dev, "positions"), ctypes.byref(c), _status_ptr(status, dev), _stream(dev))


@functools.lru_cache(maxsize=None)
def _workspace_bytes(heads: int, kv_heads: int, dim: int, dev: int) -> int:
    nbytes = ctypes.c_size_t()
    with torch.cuda.device(dev):
        call("d3_paged_attention_workspace_size", 1, heads, kv_heads, dim, ctypes.byref(nbytes))
    return nbytes.value


def paged_attention_workspace(batch: int, heads: int, kv_heads: int, dim: int, device) -> torch.Tensor:
    """Scratch of paged_attention for up to these sizes, for a caller that keeps it."""
    index = torch.device(device).index
    nbytes = _workspace_bytes(heads, kv_heads, dim, torch.cuda.current_device() if index is None else index)
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


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
    dev = k_cache.get_device()
    c = _cache_struct(k_cache, v_cache, page_table, k_scale, v_scale, dev)
    shape, dim = q.shape, c.dim
    if len(shape) != 3 or shape[2] != dim or q.get_device() != dev:
        raise ValueError(f"q must be [B, heads, {dim}] on the cache's device")
    B, Hq, _ = shape
    want = k_cache.dtype if c.dtype != _lib.D3_DTYPE_E4M3 else torch.bfloat16
    if q.dtype is not want:
        raise ValueError(f"q must be {want} for a {k_cache.dtype} cache")
    if c.sequences != B:
        raise ValueError("page_table must have one row per query")
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != shape or out.dtype is not want or out.get_device() != dev:
        raise ValueError("out must have the shape, dtype and device of q")
    q0, q1, q2 = q.stride()
    o0, o1, o2 = out.stride()
    if q2 != 1 or o2 != 1:
        raise ValueError("the last axis of q and out must be contiguous")
    lse = q.new_empty((B, Hq), dtype=torch.float32) if return_lse else None
    if workspace is None:
        workspace = q.new_empty(_workspace_bytes(Hq, c.heads, dim, dev), dtype=torch.uint8)
    limit = c.table_pages * c.page_size
    call("d3_paged_attention", q.data_ptr(), q0, q1, _DTYPES[want], B, Hq, ctypes.byref(c),
         _index_ptr(seq_lens, B, dev, "seq_lens"), limit if max_seq_len is None else min(max_seq_len, limit),
         window, dim ** -0.5 if scale is None else scale, out.data_ptr(), o0, o1,
         lse.data_ptr() if return_lse else None, workspace.data_ptr(), workspace.numel(),
         _status_ptr(status, dev), _stream(dev))
    return (out, lse) if return_lse else out
