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
from ._lib import call


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              page_table: torch.Tensor, positions: torch.Tensor, seq_ids: torch.Tensor | None = None, *,
              k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
              status: torch.Tensor | None = None) -> None:
    """Write k, v [T, heads, dim] to their pages, in place. Token t is at
    positions[t] (int32) of sequence seq_ids[t] (int32; None: sequence t);
    negative ones are skipped. An e4m3 cache takes bf16 rows and holds
    e4m3(clamp(x / scale[head], -448, 448)). Tokens past the table or on a page
    outside the cache are not written and set status to D3_STATUS_BAD_ROW. No two
    tokens of a call may name one place."""
    _lib.native().kv_append(k, v, k_cache, v_cache, page_table, positions, seq_ids, k_scale, v_scale, status)


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
    (default: what the page table can hold); tokens past it are not read. A page
    number outside the cache is read as page 0, with status set to
    D3_STATUS_BAD_ROW. Returns out (q's dtype), or (out,
    lse f32 [B, heads]) with return_lse. An empty sequence gives zeros and
    lse = -inf. Nothing is read on the host, so the call can be captured."""
    return _lib.native().paged_attention(q, k_cache, v_cache, page_table, seq_lens, scale, k_scale, v_scale, window,
                                         max_seq_len, out, return_lse, workspace, status)
