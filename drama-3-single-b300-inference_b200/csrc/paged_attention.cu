// Attention of one new token per sequence over paged keys and values.
//
// One CTA per (sequence, key head, group of up to 8 of its query heads). Each
// of 8 warps takes every eighth key: its lanes split the row, a dot product
// per query head is joined by shuffles, and the warp keeps the running
// maximum, sum and output row of each head (fp32). The warps join at the end.
#include "kv_cache.cuh"

namespace d3 {
namespace {

constexpr int kAttnWarps = 8;
constexpr int kAttnHeads = 8;  // query heads of one CTA

struct AttnArgs {
  const uint16_t* q;
  int64_t q_row, q_head;
  uint16_t* out;
  int64_t out_row, out_head;
  float* lse;
  const uint8_t* k;
  const uint8_t* v;
  int64_t k_page, k_token, k_head, v_page, v_token, v_head;  // bytes
  const float* k_scale;
  const float* v_scale;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  int max_len, window, num_pages, page_size, q_heads, group;
  float scale;
  int32_t* status;
};

template <int DT>
__device__ __forceinline__ float half_to_f32(uint16_t b) {
  if constexpr (DT == D3_DTYPE_F16) return __half2float(__ushort_as_half(b));
  return bf16_bits_to_f32(b);
}

// E = dim / 32 consecutive elements of a row, as fp32.
template <int DT, int E>
__device__ __forceinline__ void load_row_part(const uint8_t* row, int lane, float (&f)[E]) {
  if constexpr (DT == D3_DTYPE_E4M3) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(row + lane * E);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const uint32_t h = e4m3x2_to_f16x2(p[i]);
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(row) + lane * E;
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = half_to_f32<DT>(p[i]);
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(kAttnWarps * 32) paged_attention_kernel(const AttnArgs a) {
  constexpr int E = D / 32;
  constexpr int QT = DT == D3_DTYPE_F16 ? D3_DTYPE_F16 : D3_DTYPE_BF16;
  __shared__ float s_m[kAttnWarps][kAttnHeads], s_l[kAttnWarps][kAttnHeads];
  __shared__ float s_o[kAttnWarps][D];
  pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, kh = blockIdx.y;
  const int h0 = kh * a.group + blockIdx.x * kAttnHeads;
  const int nh = min(kAttnHeads, (kh + 1) * a.group - h0);
  const int len = max(0, min(__ldg(a.lens + b), a.max_len));
  const int begin = a.window > 0 ? max(0, len - a.window) : 0;
  const float ks = a.scale * (a.k_scale ? __ldg(a.k_scale + kh) : 1.0f);
  float q[kAttnHeads][E], o[kAttnHeads][E], m[kAttnHeads], l[kAttnHeads];
#pragma unroll
  for (int h = 0; h < kAttnHeads; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      o[h][i] = 0.f;
      q[h][i] = h < nh ? half_to_f32<QT>(a.q[b * a.q_row + (h0 + h) * a.q_head + lane * E + i]) : 0.f;
    }
  }
  for (int t = begin + warp; t < len; t += kAttnWarps) {
    int page = __ldg(a.table + b * a.table_stride + t / a.page_size);
    if (page < 0 || page >= a.num_pages) {
      if (a.status) atomicExch(a.status, kDevBadRow);
      page = 0;
    }
    const int off = t % a.page_size;
    float kf[E], vf[E];
    load_row_part<DT, E>(a.k + page * a.k_page + off * a.k_token + kh * a.k_head, lane, kf);
    load_row_part<DT, E>(a.v + page * a.v_page + off * a.v_token + kh * a.v_head, lane, vf);
#pragma unroll
    for (int h = 0; h < kAttnHeads; ++h) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) s = fmaf(q[h][i], kf[i], s);
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= ks;
      const float mn = fmaxf(m[h], s);
      const float base = mn == -INFINITY ? 0.f : mn;  // a logit of -inf adds nothing
      const float c = expf(m[h] - base), p = expf(s - base);
      m[h] = mn;
      l[h] = l[h] * c + p;
#pragma unroll
      for (int i = 0; i < E; ++i) o[h][i] = fmaf(p, vf[i], o[h][i] * c);
    }
  }
  if (lane == 0)
    for (int h = 0; h < kAttnHeads; ++h) {
      s_m[warp][h] = m[h];
      s_l[warp][h] = l[h];
    }
  const float vs = a.v_scale ? __ldg(a.v_scale + kh) : 1.0f;
#pragma unroll
  for (int h = 0; h < kAttnHeads; ++h) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < E; ++i) s_o[warp][lane * E + i] = o[h][i];
    __syncthreads();
    if (h >= nh) continue;
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, s_m[w][h]);
    const float base = top == -INFINITY ? 0.f : top;
    for (int w = 0; w < kAttnWarps; ++w) sum += s_l[w][h] * expf(s_m[w][h] - base);
    for (int d = threadIdx.x; d < D; d += kAttnWarps * 32) {
      float x = 0.f;
      for (int w = 0; w < kAttnWarps; ++w) x += s_o[w][d] * expf(s_m[w][h] - base);
      x = sum == 0.f ? 0.f : x / sum * vs;  // a NaN stays one
      uint16_t r;
      if constexpr (QT == D3_DTYPE_F16) r = __half_as_ushort(__float2half_rn(x));
      else r = __bfloat16_as_ushort(__float2bfloat16_rn(x));
      a.out[b * a.out_row + (h0 + h) * a.out_head + d] = r;
    }
    if (a.lse && threadIdx.x == 0)
      a.lse[static_cast<int64_t>(b) * a.q_heads + h0 + h] = sum == 0.f ? -INFINITY : logf(sum) + top;
  }
}

template <int DT>
void launch_attention(const AttnArgs& a, int D, dim3 grid, cudaStream_t s) {
  const dim3 block(kAttnWarps * 32);
  if (D == 64) launch_kernel(paged_attention_kernel<DT, 64>, grid, block, 0, s, a);
  else if (D == 128) launch_kernel(paged_attention_kernel<DT, 128>, grid, block, 0, s, a);
  else launch_kernel(paged_attention_kernel<DT, 256>, grid, block, 0, s, a);
}

}  // namespace
}  // namespace d3

using namespace d3;

extern "C" int d3_paged_attention_workspace_size(int B, int q_heads, int kv_heads, int dim, size_t* bytes) {
  D3_REQUIRE(bytes != nullptr, "bytes is NULL");
  D3_REQUIRE(B >= 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0,
             "query heads must be a multiple of key heads");
  D3_REQUIRE(dim == 64 || dim == 128 || dim == 256, "head dim must be 64, 128 or 256");
  *bytes = 0;
  return D3_OK;
}

extern "C" int d3_paged_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride, int q_dtype,
                                  int B, int q_heads, const d3_kv_cache_t* cache, const int32_t* lens,
                                  int max_len, int window, float scale, void* out,
                                  int64_t out_row_stride, int64_t out_head_stride, float* lse,
                                  void* workspace, size_t workspace_bytes, int32_t* status,
                                  d3_stream_t stream) {
  if (int rc = check_kv_cache(cache)) return rc;
  size_t need = 0;
  if (int rc = d3_paged_attention_workspace_size(B, q_heads, cache->heads, cache->dim, &need)) return rc;
  D3_REQUIRE(q_dtype == (cache->dtype == D3_DTYPE_E4M3 ? D3_DTYPE_BF16 : cache->dtype),
             "queries of dtype %d for a cache of dtype %d", q_dtype, cache->dtype);
  D3_REQUIRE(max_len >= 0 && window >= 0, "negative length bound or window");
  D3_REQUIRE(cache->sequences == B, "the page table must have one row per query");
  if (workspace_bytes < need || (need && !workspace))
    return set_error(D3_EWORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (B == 0) return D3_OK;
  D3_REQUIRE(q && out && lens, "NULL operand");
  const int64_t held = static_cast<int64_t>(cache->table_pages) * cache->page_size;
  AttnArgs a{};
  a.max_len = static_cast<int>(held < max_len ? held : max_len);
  D3_REQUIRE(a.max_len == 0 || (cache->k && cache->v && cache->table && cache->num_pages > 0), "NULL or empty cache");
  const int64_t e = kv_elem_bytes(cache->dtype);
  a.q = static_cast<const uint16_t*>(q);
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.out = static_cast<uint16_t*>(out);
  a.out_row = out_row_stride;
  a.out_head = out_head_stride;
  a.lse = lse;
  a.k = static_cast<const uint8_t*>(cache->k);
  a.v = static_cast<const uint8_t*>(cache->v);
  a.k_page = cache->k_page_stride * e;
  a.k_token = cache->k_token_stride * e;
  a.k_head = cache->k_head_stride * e;
  a.v_page = cache->v_page_stride * e;
  a.v_token = cache->v_token_stride * e;
  a.v_head = cache->v_head_stride * e;
  a.k_scale = cache->k_scale;
  a.v_scale = cache->v_scale;
  a.table = cache->table;
  a.table_stride = cache->table_stride;
  a.lens = lens;
  a.window = window;
  a.num_pages = cache->num_pages;
  a.page_size = cache->page_size;
  a.q_heads = q_heads;
  a.group = q_heads / cache->heads;
  a.scale = scale;
  a.status = status;
  const dim3 grid((a.group + kAttnHeads - 1) / kAttnHeads, cache->heads, B);
  D3_REQUIRE(B <= 65535 && cache->heads <= 65535, "batch or heads too large");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (cache->dtype == D3_DTYPE_BF16) launch_attention<D3_DTYPE_BF16>(a, cache->dim, grid, s);
  else if (cache->dtype == D3_DTYPE_F16) launch_attention<D3_DTYPE_F16>(a, cache->dim, grid, s);
  else launch_attention<D3_DTYPE_E4M3>(a, cache->dim, grid, s);
  return check_launch("d3_paged_attention");
}
