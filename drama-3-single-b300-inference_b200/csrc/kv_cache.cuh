// Host checks and device views of the paged key-value cache (d3_kv_cache_t).
#pragma once

#include "d3_common.cuh"
#include "d3_host.h"

namespace d3 {

// Bytes of one cache element.
inline int kv_elem_bytes(int dtype) { return dtype == D3_DTYPE_E4M3 ? 1 : 2; }

// D3_OK or D3_EINVAL for the shapes, strides and alignment of a cache.
inline int check_kv_cache(const d3_kv_cache_t* c) {
  D3_REQUIRE(c != nullptr, "the cache description is NULL");
  D3_REQUIRE(c->dtype == D3_DTYPE_BF16 || c->dtype == D3_DTYPE_F16 || c->dtype == D3_DTYPE_E4M3,
             "unsupported cache dtype %d", c->dtype);
  D3_REQUIRE(c->num_pages >= 0 && c->page_size > 0 && c->heads > 0 && c->dim > 0 &&
                 c->sequences >= 0 && c->table_pages >= 0,
             "bad cache geometry");
  const int64_t e = kv_elem_bytes(c->dtype);
  const int64_t strides[6] = {c->k_page_stride, c->k_token_stride, c->k_head_stride,
                              c->v_page_stride, c->v_token_stride, c->v_head_stride};
  for (int64_t s : strides)
    D3_REQUIRE((s * e) % 16 == 0, "cache strides must be multiples of 16 bytes");
  D3_REQUIRE((c->dim * e) % 16 == 0, "cache rows must be a multiple of 16 bytes");
  D3_REQUIRE(aligned(c->k, 16) && aligned(c->v, 16), "cache pointers must be 16-byte aligned");
  D3_REQUIRE(c->dtype == D3_DTYPE_E4M3 || (c->k_scale == nullptr && c->v_scale == nullptr),
             "only an e4m3 cache has scales");
  return D3_OK;
}

}  // namespace d3
