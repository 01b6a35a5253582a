// Writes to the sequence memory: new keys and values into their pages, and
// copies of whole pages (forks, compaction). Both move each byte once in and
// once out, so they are bound by HBM (or, for a decode step, by launch latency):
// 1500 pages of 16 KB in 20 planes, 983 MB, are copied in 149 us, 6.6 TB/s, the rate of
// a plain copy; 15670 tokens of 2 x 2 x 256 are appended in 13.1 us, 4.9 TB/s; 64 tokens in
// 2.6 us, 16 pages in 20 planes in 2.9 us.
#include "kv_cache.cuh"

namespace d3 {
namespace {

struct AppendArgs {
  const uint8_t* src[2];           // k, v
  int64_t src_token[2], src_head[2];  // bytes
  uint8_t* dst[2];
  int64_t dst_page[2], dst_token[2], dst_head[2];  // bytes
  const float* scale[2];
  const int32_t* seq;
  const int32_t* pos;
  const int32_t* table;
  int64_t table_stride;
  int sequences, table_pages, num_pages, page_size;
  int heads, pieces;  // pieces: 16-byte source pieces of one row
  int T;
  int32_t* status;
};

// Place of token t: its page (or -1: not written) and the offset in it.
__device__ __forceinline__ int append_place(const AppendArgs& a, int t, int& off) {
  const int seq = a.seq ? __ldg(a.seq + t) : t;
  const int pos = __ldg(a.pos + t);
  if (seq < 0 || pos < 0) return -1;
  const int slot = pos / a.page_size;
  off = pos - slot * a.page_size;
  int page = -1;
  if (seq < a.sequences && slot < a.table_pages) page = __ldg(a.table + seq * a.table_stride + slot);
  if (page < 0 || page >= a.num_pages) {
    if (a.status) atomicExch(a.status, kDevBadRow);
    return -1;
  }
  return page;
}

// One warp per token: its page is looked up once, and its lanes take the 16-byte source
// pieces of the token's rows (k, then v), kAppendUnroll of them asked for before the
// first is written. A piece per thread with its own divisions for token and page was
// bound by those (15670 tokens of 2 x 256: 17 us).
constexpr int kAppendUnroll = 4;
constexpr int kAppendWarps = 8;
template <bool FP8>
__global__ void __launch_bounds__(kAppendWarps * 32) kv_append_kernel(const AppendArgs a) {
  pdl_enter();
  const int t = blockIdx.x * kAppendWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= a.T) return;
  const int rows = a.heads * a.pieces;  // pieces of k, and of v
  int off = 0, page = 0;
  bool placed = false;
  for (int r0 = lane; r0 < 2 * rows; r0 += 32 * kAppendUnroll) {
    uint4 v[kAppendUnroll];
    int64_t to[kAppendUnroll];
    int kvs[kAppendUnroll];
    float s[kAppendUnroll];
#pragma unroll
    for (int u = 0; u < kAppendUnroll; ++u) {
      unsigned r = r0 + u * 32;
      kvs[u] = -1;
      if (r >= 2u * rows) continue;
      const int kv = r >= static_cast<unsigned>(rows);
      r -= kv ? rows : 0;
      const unsigned head = r / static_cast<unsigned>(a.pieces), piece = r - head * a.pieces;
      v[u] = *reinterpret_cast<const uint4*>(a.src[kv] + t * a.src_token[kv] + head * a.src_head[kv] + piece * 16);
      to[u] = head * a.dst_head[kv] + piece * (FP8 ? 8 : 16);
      kvs[u] = kv;
      s[u] = FP8 && a.scale[kv] ? __ldg(a.scale[kv] + head) : 1.0f;
    }
    if (!placed) {  // the page is looked up while the rows are on their way
      page = append_place(a, t, off);
      if (page < 0) return;
      placed = true;
    }
#pragma unroll
    for (int u = 0; u < kAppendUnroll; ++u) {
      if (kvs[u] < 0) continue;
      uint8_t* at = (kvs[u] ? a.dst[1] : a.dst[0]) + page * (kvs[u] ? a.dst_page[1] : a.dst_page[0]) +
                    off * (kvs[u] ? a.dst_token[1] : a.dst_token[0]) + to[u];
      if constexpr (FP8) {
        const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
        uint32_t o[2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // x / scale; the conversion saturates to +-448 (a NaN stays one)
          const uint32_t p = f32x2_to_e4m3x2(__fdiv_rn(__uint_as_float(w[j] << 16), s[u]), __fdiv_rn(__uint_as_float(w[j] & 0xffff0000u), s[u]));
          o[j >> 1] = (j & 1) ? (o[j >> 1] | (p << 16)) : p;
        }
        *reinterpret_cast<uint2*>(at) = make_uint2(o[0], o[1]);
      } else {
        *reinterpret_cast<uint4*>(at) = v[u];
      }
    }
  }
}

struct CopyArgs {
  uint8_t* pool;
  int64_t plane_stride, page_stride, page_bytes;
  const int32_t* src;
  const int32_t* dst;
  int pages;
  int32_t* status;
};

// A CTA copies up to 16 KB of a page, every thread's four loads before its first store:
// with 8 CTAs on an SM 128 KB are on their way.
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;  // loads in flight per thread

// grid (slabs of a page, pairs, planes); V is the unit of one load.
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const CopyArgs a, int n, int planes) {
  pdl_enter();
  const int64_t units = a.page_bytes / static_cast<int64_t>(sizeof(V));
  const int64_t u0 = static_cast<int64_t>(blockIdx.x) * (kCopyThreads * kCopyUnroll) + threadIdx.x;
  for (int plane = blockIdx.z; plane < planes; plane += gridDim.z)
    for (int i = blockIdx.y; i < n; i += gridDim.y) {
      const int s = __ldg(a.src + i), d = __ldg(a.dst + i);
      if (s < 0 || d < 0) continue;
      if (s >= a.pages || d >= a.pages) {
        if (a.status && threadIdx.x == 0) atomicExch(a.status, kDevBadRow);
        continue;
      }
      const V* from = reinterpret_cast<const V*>(a.pool + plane * a.plane_stride + s * a.page_stride);
      V* to = reinterpret_cast<V*>(a.pool + plane * a.plane_stride + d * a.page_stride);
      V v[kCopyUnroll];
#pragma unroll
      for (int j = 0; j < kCopyUnroll; ++j)
        if (u0 + j * kCopyThreads < units) v[j] = from[u0 + j * kCopyThreads];
#pragma unroll
      for (int j = 0; j < kCopyUnroll; ++j)
        if (u0 + j * kCopyThreads < units) to[u0 + j * kCopyThreads] = v[j];
    }
}

}  // namespace
}  // namespace d3

using namespace d3;

extern "C" int d3_kv_append(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                            int64_t v_token_stride, int64_t v_head_stride, int dtype, int T,
                            const int32_t* seq, const int32_t* pos, const d3_kv_cache_t* cache,
                            int32_t* status, d3_stream_t stream) {
  if (int rc = check_kv_cache(cache)) return rc;
  const bool fp8 = cache->dtype == D3_DTYPE_E4M3;
  D3_REQUIRE(dtype == (fp8 ? D3_DTYPE_BF16 : cache->dtype), "rows of dtype %d for a cache of dtype %d",
             dtype, cache->dtype);
  D3_REQUIRE(T >= 0, "negative token count");
  D3_REQUIRE(T <= 0x7fffff00, "too many tokens for one call");  // a CTA's last warps may pass T
  if (T == 0) return D3_OK;
  D3_REQUIRE(k && v && pos && cache->table && cache->k && cache->v, "NULL operand");
  D3_REQUIRE(aligned(k, 16) && aligned(v, 16) && k_token_stride % 8 == 0 && k_head_stride % 8 == 0 &&
                 v_token_stride % 8 == 0 && v_head_stride % 8 == 0,
             "rows of k and v must be 16-byte aligned");
  AppendArgs a{};
  const int64_t e = kv_elem_bytes(cache->dtype);
  a.src[0] = static_cast<const uint8_t*>(k);
  a.src[1] = static_cast<const uint8_t*>(v);
  a.src_token[0] = k_token_stride * 2;
  a.src_token[1] = v_token_stride * 2;
  a.src_head[0] = k_head_stride * 2;
  a.src_head[1] = v_head_stride * 2;
  a.dst[0] = static_cast<uint8_t*>(cache->k);
  a.dst[1] = static_cast<uint8_t*>(cache->v);
  a.dst_page[0] = cache->k_page_stride * e;
  a.dst_page[1] = cache->v_page_stride * e;
  a.dst_token[0] = cache->k_token_stride * e;
  a.dst_token[1] = cache->v_token_stride * e;
  a.dst_head[0] = cache->k_head_stride * e;
  a.dst_head[1] = cache->v_head_stride * e;
  a.scale[0] = cache->k_scale;
  a.scale[1] = cache->v_scale;
  a.seq = seq;
  a.pos = pos;
  a.table = cache->table;
  a.table_stride = cache->table_stride;
  a.sequences = cache->sequences;
  a.table_pages = cache->table_pages;
  a.num_pages = cache->num_pages;
  a.page_size = cache->page_size;
  a.heads = cache->heads;
  a.pieces = cache->dim / 8;
  a.T = T;
  a.status = status;
  D3_REQUIRE(static_cast<int64_t>(a.heads) * a.pieces < 0x20000000, "rows are too long");
  launch_kernel(fp8 ? kv_append_kernel<true> : kv_append_kernel<false>,
                dim3(static_cast<unsigned>((static_cast<int64_t>(T) + kAppendWarps - 1) / kAppendWarps)), dim3(kAppendWarps * 32), 0,
                reinterpret_cast<cudaStream_t>(stream), a);
  return check_launch("d3_kv_append");
}

extern "C" int d3_copy_pages(void* pool, int planes, int64_t plane_stride, int pages,
                             int64_t page_stride, int64_t page_bytes, const int32_t* src,
                             const int32_t* dst, int n, int32_t* status, d3_stream_t stream) {
  D3_REQUIRE(planes >= 0 && pages >= 0 && page_bytes >= 0 && n >= 0, "negative size");
  D3_REQUIRE(pages <= 1 || page_stride >= page_bytes || page_stride <= -page_bytes,
             "pages overlap: page_stride is smaller than a page");
  // the kernel's counters pass the last plane and pair by up to 65535
  D3_REQUIRE(planes <= 0x40000000 && n <= 0x40000000, "too many planes or pairs for one call");
  if (planes == 0 || n == 0 || page_bytes == 0 || pages == 0) return D3_OK;
  D3_REQUIRE(pool && src && dst, "NULL operand");
  CopyArgs a{static_cast<uint8_t*>(pool), plane_stride, page_stride, page_bytes, src, dst, pages, status};
  const bool wide = aligned(pool, 16) && plane_stride % 16 == 0 && page_stride % 16 == 0 && page_bytes % 16 == 0;
  const int64_t per = static_cast<int64_t>(kCopyThreads) * kCopyUnroll * (wide ? 16 : 1);
  const int64_t slabs = (page_bytes + per - 1) / per;
  D3_REQUIRE(slabs <= 0x7fffffff, "pages of %lld bytes are too large", static_cast<long long>(page_bytes));
  const dim3 grid(static_cast<unsigned>(slabs), static_cast<unsigned>(n < 65535 ? n : 65535),
                  static_cast<unsigned>(planes < 65535 ? planes : 65535));
  // 16-byte units where every page start allows it, single bytes otherwise
  launch_kernel(wide ? copy_pages_kernel<uint4> : copy_pages_kernel<uint8_t>, grid, dim3(kCopyThreads), 0,
                reinterpret_cast<cudaStream_t>(stream), a, n, planes);
  return check_launch("d3_copy_pages");
}
