"""Host side of the sequence-memory operators at the edges of what they take, without a GPU."""

from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")


def _refused(rc, text):
    from d3moe import _lib
    lib = _lib.load()
    assert rc == _lib.D3_EINVAL and text in lib.d3_last_error_string(), (rc, lib.d3_last_error_string())


def test_attention_refuses_negative_cache_strides():
    """Row offsets below zero mark places past a sequence's end, so no key may have one."""
    from d3moe import _lib
    lib = _lib.load()
    ok = dict(k=1 << 20, v=1 << 20, k_page_stride=8192, k_token_stride=512, k_head_stride=256, v_page_stride=8192, v_token_stride=512,
              v_head_stride=256, table=4096, table_stride=4, sequences=2, table_pages=4, num_pages=8, page_size=16, heads=2, dim=256,
              dtype=_lib.D3_DTYPE_BF16)
    for name in ("k_page_stride", "k_token_stride", "v_page_stride", "v_token_stride"):
        c = _lib.D3KvCache(**{**ok, name: -ok[name]})
        _refused(lib.d3_paged_attention(4096, 4096, 256, _lib.D3_DTYPE_BF16, 2, 16, ctypes.byref(c), 4096, 64, 0, 1.0, 4096, 4096, 256,
                                        None, 4096, 1 << 30, None, None), b"negative")


def test_delta_chunk_refuses_tokens_whose_counter_would_pass_32_bits():
    from d3moe import _lib
    lib = _lib.load()
    a = _lib.D3GatedDelta(q=4096, k=4096, v=4096, g=4096, beta=4096, out=4096, state=4096, slots=1, key_heads=1, value_heads=1, key_dim=64,
                          value_dim=64, l2norm=1, scale=1.0, eps=1e-6)
    _refused(lib.d3_gated_delta_chunk(ctypes.byref(a), 4096, 2**31 - 1, 1, None, 4096, 1 << 60, None, None), b"too many tokens")
