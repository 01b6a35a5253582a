// Attention of one new token per sequence over paged keys and values.
//
//   s_j = scale q.k_j,  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// Each key and value is read once and used by the query heads that share it,
// a few flops per byte: the kernel is bound by HBM, and everything else has to
// hide behind the loads.
//
// Work. A unit is a (sequence, key head, group of query heads); its keys are
// cut into tiles of 4 * NK. All units' tiles form one line, and each CTA of a
// persistent grid (two or three per SM) takes an equal share of it, so ragged lengths
// balance by themselves and a single long sequence uses every SM. A CTA's share
// may end inside a unit: such parts leave (max, sum, output row) in the
// workspace, and a second kernel joins them in CTA order (no atomics, so equal
// inputs give equal bits). Short units are taken whole, or by a thread-block cluster
// that joins its parts through shared memory, in one launch (unit_ctas).
//
// Measured (bf16, 16 query and 2 key heads of 256, pages of 16): 4 sequences of 100k to
// 131k tokens, 977 MB, in 162 us, 6.04 TB/s or 0.93 of the copy rate (a split of the line
// into more CTAs than fit at once, deeper rings and prefetches to L2 were all slower; SMs
// do not get equal shares of the bandwidth, and the slowest ends the kernel); 64 of up to
// 2048, 136 MB, in 33 us, of which start and joining take about 10; 1 of 301 in 7.5 us. 16
// of up to 16411 in e4m3 (32 query and 8 key heads of 128), 311 MB: 64 us, 4.9 TB/s, issue
// slots 0.53 busy with widening and twice the products per byte.
//
// Inside a CTA 4 warps run on their own: warp w takes keys [w*NK, (w+1)*NK) of a
// tile, loads them with cp.async into its own ring of shared-memory slots (keys
// and values of a tile are two slots; no barrier between warps), and works with
// mma.sync m16n8k16 on transposes: the keys are the 16 rows of A and 8 query heads the
// columns of B for the logits, and V^T is A for the output, so with up to 8 heads per
// key head no part of a product is idle; the probabilities turn into B operands by
// one movmatrix each. tcgen05 has nothing to add: its tile of 128 rows of keys per
// instruction would need 8 columns at most, and the operands' way through shared
// memory is the same. bf16 probabilities go in two terms (2^-17), so the output is
// rounded once, at its end. f16 ones (f16 and e4m3 caches) go in one term, 2^-11 of
// themselves: exp2(s - m) times 2^14, which f16 holds, so this is so down to 2^-28 of the
// warp's largest and off by 2^-39 of that below. (Unscaled they lose bits from 2^-14 on and
// are 0 from 2^-25 on, while the sum still counts them: a row of many small probabilities
// beside one key with a small value comes out too small.)
//
// An e4m3 cache is widened to f16 in registers (exact). Its queries are scaled by
// a power of two per row into f16's range (exact for every element within 2^-14
// of the row's largest, error at most 2^-24 of that otherwise).
#include "kv_cache.cuh"
#include "mma_tiles.cuh"

namespace d3 {
namespace {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = kAttnWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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
  int B, max_len, window, num_pages, page_size, q_heads, group;
  int parts, units;  // query-head groups per key head; units per sequence
  float scale;
  float* partial;    // [grid][2] records of ROWS * (D + 2) floats
  int grid;          // CTAs of the main kernel
  int share;         // CTAs of a cluster that shares one unit, 0: the line of all units' tiles
  int32_t* status;
};

constexpr int attn_ctas(int D, int elem) { return D * elem >= 256 ? 2 : 3; }

// Sizes of one variant. WIDE: 16 query heads per unit, else 8. (e4m3 with 256 columns and WIDE
// spills 34 bytes at 255 registers; no other variant of the main kernel does.)
template <int DT, int D, bool WIDE>
struct AttnShape {
  static constexpr int kElem = DT == D3_DTYPE_E4M3 ? 1 : 2;
  static constexpr int kRowBytes = D * kElem;
  // CTAs that share an SM, and what of its shared memory one may take: two with deep rings
  // for rows of 256 bytes and more, three for shorter ones, which need more work per byte (16
  // sequences of up to 8000 tokens, 8 bf16 key heads of 128: 60 us with two, 75 with
  // three; of up to 16000, e4m3: 65 and 64, of 64 columns 52 and 47)
  static constexpr int kCtas = attn_ctas(D, kElem);
  static constexpr int kMaxSmem = (kCtas == 2 ? 113 : 75) * 1024;
  // keys of one warp and tile, 16 or 32: a slot of the ring holds 8 KB for 256 columns, up to 4 KB else
  static constexpr int kNK = kRowBytes == 256 || kRowBytes == 512 ? (D == 256 && kElem == 1 ? 32 : 16) : 32;
  static constexpr int kTile = kNK * kAttnWarps;
  static constexpr int kRows = WIDE ? 16 : 8;
  static constexpr int kHalf = kNK * kRowBytes;  // bytes of a slot
  static constexpr int kFit = ((kCtas == 2 ? 24576 : 16384) / kHalf - 1) / 2;
  static constexpr int kAhead = kFit < 4 ? kFit : 4;  // tiles loaded ahead
  static constexpr int kSlots = 2 * kAhead + 1;
  static constexpr int kWarpRing = kSlots * kHalf;
  static constexpr int kRing = kAttnWarps * kWarpRing;
  static constexpr int kQPitch = D * 2 + 16;   // bytes of a query row, padded against bank conflicts
  static constexpr int kQ = kRows * kQPitch;
  static constexpr int kQPieces = (kRows * D * 2 / 16 + kAttnThreads - 1) / kAttnThreads;  // of one thread
  static constexpr int kStat = kAttnWarps * 32 * 4 + 64;
  // 8 output rows of kJoinWarps warps at a time are added up in shared memory
  static constexpr int kJoinPitch = D + 4;     // floats, padded likewise
  static constexpr int kJoinFit = (kMaxSmem - kRing - kQ - kStat) / (8 * kJoinPitch * 4);
  static constexpr int kJoinWarps = kJoinFit >= 4 ? 4 : kJoinFit >= 2 ? 2 : 1;
  static constexpr int kJoin = kJoinWarps * 8 * kJoinPitch * 4;
  static constexpr int kSmem = kRing + kJoin + kQ + kStat;
  static_assert(kSmem <= kMaxSmem);
  static constexpr int kRecord = kRows * (D + 2);  // floats of a partial result
};

__device__ __forceinline__ int seq_begin(const AttnArgs& a, int len) {
  return a.window > 0 ? max(0, len - a.window) : 0;
}
__device__ __forceinline__ int seq_len(const AttnArgs& a, int b) {
  return max(0, min(__ldg(a.lens + b), a.max_len));
}
template <int TILE>
__device__ __forceinline__ int seq_tiles(const AttnArgs& a, int b) {
  const int len = seq_len(a, b);
  return (len - seq_begin(a, len) + TILE - 1) / TILE;
}

// Places on the line: a unit with keys takes kUnitCost places of its own before
// its tiles, for what a unit costs besides them (fetching its queries and page
// numbers, joining the warps).
constexpr int kUnitCost = 1;
template <int TILE>
__device__ __forceinline__ int seq_places(const AttnArgs& a, int b) {
  const int tiles = seq_tiles<TILE>(a, b);
  return tiles > 0 ? (tiles + kUnitCost) * a.units : 0;
}

// Places of one CTA: an equal share of the line.
__device__ __forceinline__ int cta_share(int total, int grid) {
  return static_cast<int>((static_cast<unsigned>(total) + grid - 1) / grid);
}

// Sums over the sequences with all threads: the places of all
// sequences, and each thread's exclusive prefix over its own run of `per`
// sequences. scratch: WARPS values of shared memory.
template <int TILE, int WARPS>
__device__ __forceinline__ void line_scan(const AttnArgs& a, int per, int* scratch, int& mine, int& before,
                                          int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  mine = 0;
  for (int i = 0; i < per; ++i) {
    const int b = threadIdx.x * per + i;
    if (b < a.B) mine += seq_places<TILE>(a, b);
  }
  int x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  before = x - mine;
  total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += scratch[w];
    total += scratch[w];
  }
}

// Tile `tile` of unit `unit` of sequence b, and its place on the line.
template <int TILE>
struct Cursor {
  int b, unit, tile, tiles, len, begin, at;
  __device__ __forceinline__ void enter(const AttnArgs& a) {
    len = seq_len(a, b);
    begin = seq_begin(a, len);
    tiles = (len - begin + TILE - 1) / TILE;
  }
  // The next tile; b == a.B behind the last.
  __device__ __forceinline__ void next(const AttnArgs& a) {
    ++at;
    if (++tile < tiles) return;
    at += kUnitCost;
    tile = 0;
    if (++unit < a.units) return;
    unit = 0;
    do {
      if (++b >= a.B) return;
      enter(a);
    } while (tiles == 0);
  }
};

// The cluster's CTAs: this one's rank, a barrier over all their threads (what each wrote
// to its shared memory before is seen by the others after), and reads of CTA c's shared
// memory at the place that has address `at` in this one's.
__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return static_cast<int>(r);
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_map(uint32_t at, int c) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(c));
  return r;
}
__device__ __forceinline__ float cluster_load(uint32_t at, int c) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(cluster_map(at, c)) : "memory");
  return x;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t at, int c) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(cluster_map(at, c)) : "memory");
  return x;
}

// Four columns of a finished row: x / sum * v_scale in the output's type; lse
// with the first. A sum of 0 (no key took part) gives zeros and -inf, a NaN stays one.
template <bool BF16>
__device__ __forceinline__ void store_row(const AttnArgs& a, int b, int h, int d, const float (&x)[4], float sum,
                                          float top, float v_scale) {
  const float inv = sum == 0.f ? 0.f : v_scale / sum;
  *reinterpret_cast<uint2*>(a.out + b * a.out_row + h * a.out_head + d) =
      make_uint2(pack16<BF16>(x[0] * inv, x[1] * inv), pack16<BF16>(x[2] * inv, x[3] * inv));
  if (a.lse && d == 0)
    a.lse[static_cast<int64_t>(b) * a.q_heads + h] = sum == 0.f ? -INFINITY : (log2f(sum) + top) * kLn2;
}

// LINE: a share of the line of all units' tiles; else a cluster per unit.
template <int DT, int D, bool WIDE, bool LINE>
__global__ void __launch_bounds__(kAttnThreads, (AttnShape<DT, D, WIDE>::kCtas)) paged_attention_kernel(const AttnArgs a) {
  using Sh = AttnShape<DT, D, WIDE>;
  constexpr bool BF16 = DT == D3_DTYPE_BF16;        // type of the matrix products
  constexpr bool QBF16 = DT != D3_DTYPE_F16;        // type of q and out
  constexpr int NK = Sh::kNK, RB = Sh::kRowBytes, S = Sh::kSlots, P = Sh::kAhead, ROWS = Sh::kRows;
  constexpr int KS = D / 16, MT = NK / 16, NH = ROWS / 8;
  constexpr float PS = BF16 ? 1.f : 16384.f;        // the probabilities' factor in the products with V
  constexpr int PIECES = RB / 16, JW = LINE ? Sh::kJoinWarps : kAttnWarps, JP = Sh::kJoinPitch;
  extern __shared__ __align__(1024) uint8_t smem[];
  // without a line a CTA joins once, when its ring is empty: all warps' rows fit there,
  // and behind them the record for the cluster
  float* join = reinterpret_cast<float*>(smem + (LINE ? Sh::kRing : 0));
  constexpr int kRecordAt = kAttnWarps * 8 * JP * 4;
  static_assert(kRecordAt + Sh::kRecord * 4 <= Sh::kRing);
  uint8_t* qs = smem + Sh::kRing + Sh::kJoin;
  float* stat = reinterpret_cast<float*>(qs + Sh::kQ);  // [warps][2][16]
  int* scratch = reinterpret_cast<int*>(stat + kAttnWarps * 32);
  int* start = scratch + kAttnWarps;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int quad = lane >> 2, t4 = lane & 3;

  pdl_wait();
  pdl_trigger();  // after the wait: the joining kernel may read lens before it waits itself

  Cursor<Sh::kTile> cur;
  int end;  // of this CTA's places
  const int rank = !LINE && a.share > 1 ? cluster_rank() : 0;
  if constexpr (!LINE) {  // one unit per cluster, its tiles spread over the CTAs
    const int id = blockIdx.x / a.share;
    cur.b = id / a.units;
    cur.unit = id % a.units;
    const int tiles = seq_tiles<Sh::kTile>(a, cur.b);
    cur.tile = cur.at = rank * tiles / a.share;
    end = (rank + 1) * tiles / a.share;
  } else {
    // where this CTA's share of the line begins
    const int per = (a.B + kAttnThreads - 1) / kAttnThreads;
    int mine, before, total;
    line_scan<Sh::kTile, kAttnWarps>(a, per, scratch, mine, before, total);
    const int share = cta_share(total, a.grid);
    if (total == 0 || static_cast<int64_t>(blockIdx.x) * share >= total) return;
    const int first = blockIdx.x * share;
    end = min(first + share, total);
    if (first >= before && first < before + mine) {
      int at = before;
      for (int i = 0; i < per; ++i) {
        const int b = tid * per + i, n = seq_places<Sh::kTile>(a, b);
        if (first < at + n) {
          const int each = n / a.units, unit = (first - at) / each;
          start[0] = b;
          start[1] = unit;
          start[2] = max(0, first - at - unit * each - kUnitCost);
          start[3] = at + unit * each + kUnitCost + start[2];
          break;
        }
        at += n;
      }
    }
    __syncthreads();
    cur.b = start[0];
    cur.unit = start[1];
    cur.tile = start[2];
    cur.at = start[3];
    if (cur.at >= end) return;  // nothing but a unit's own places
  }
  cur.enter(a);
  Cursor<Sh::kTile> ld = cur;

  const uint32_t ring = smem_u32(smem) + warp * Sh::kWarpRing;

  // offsets of row `lane` of tile `ld` in the two caches (-1: past the end)
  int64_t koff, voff;
  auto look_up = [&]() {
    const int j = ld.begin + ld.tile * Sh::kTile + warp * NK + lane;
    koff = voff = -1;
    if (lane < NK && j < ld.len) {
      const int slot = j / a.page_size;
      const int64_t o = j - slot * a.page_size;
      int p = __ldg(a.table + ld.b * a.table_stride + slot);
      if (p < 0 || p >= a.num_pages) {
        if (a.status) atomicExch(a.status, kDevBadRow);
        p = 0;
      }
      koff = p * a.k_page + o * a.k_token;
      voff = p * a.v_page + o * a.v_token;
    }
  };
  // copies this warp's rows of tile `ld` (keys or values) into a slot; rows past
  // the sequence's end are zeroed (what the cache holds there may be anything,
  // NaN included)
  auto load = [&](int slot, const uint8_t* base, int64_t mine_off) {
    const uint32_t dst = ring + slot * Sh::kHalf;
#pragma unroll
    for (int it = 0; it < NK * PIECES / 32; ++it) {
      const int idx = it * 32 + lane, r = idx / PIECES, c = idx % PIECES;
      const int64_t o = __shfl_sync(0xffffffffu, mine_off, r);
      cp_async_16_zfill(dst + tile_at<RB>(r, c), base + (o < 0 ? 0 : o) + c * 16, o >= 0);
    }
  };
  int slot = 0;    // next slot to fill
  auto load_keys = [&]() {
    if (ld.at < end) load(slot, a.k + ld.unit / a.parts * a.k_head, koff);
    slot = slot + 1 == S ? 0 : slot + 1;
    cp_async_commit();
  };
  auto load_values = [&]() {
    if (ld.at < end) {
      load(slot, a.v + ld.unit / a.parts * a.v_head, voff);
      ld.next(a);
      if (ld.at < end) look_up();
    }
    slot = slot + 1 == S ? 0 : slot + 1;
    cp_async_commit();
  };

  // queries of a unit, on their way to shared memory (rows past the unit's are zero)
  uint4 qreg[Sh::kQPieces];
  auto fetch_q = [&](const Cursor<Sh::kTile>& c) {
    const int head = c.unit / a.parts, h0 = head * a.group + (c.unit % a.parts) * ROWS;
    const int nh = min(ROWS, (head + 1) * a.group - h0);
#pragma unroll
    for (int x = 0; x < Sh::kQPieces; ++x) {
      const int e = tid + x * kAttnThreads, r = e / (D / 8), d = e % (D / 8) * 8;
      qreg[x] = r < nh ? __ldg(reinterpret_cast<const uint4*>(a.q + c.b * a.q_row + (h0 + r) * a.q_head + d)) : make_uint4(0, 0, 0, 0);
    }
  };
  auto place_q = [&]() {
#pragma unroll
    for (int x = 0; x < Sh::kQPieces; ++x) {
      const int e = tid + x * kAttnThreads, r = e / (D / 8), d = e % (D / 8) * 16;
      if (r < ROWS) *reinterpret_cast<uint4*>(qs + r * Sh::kQPitch + d) = qreg[x];
    }
  };

  fetch_q(cur);
  if (ld.at < end) look_up();
#pragma unroll
  for (int s = 0; s < P; ++s) {
    load_keys();
    load_values();
  }

  place_q();
  __syncthreads();

  uint32_t qf[KS][NH][2];  // queries as B operands: a column per head
  float o[KS][NH][4];      // 16 columns of V by 8 heads each, times PS
  float m[NH][2], l[NH][2];  // of heads 2 t4 and 2 t4 + 1
  float lg[NH][2];         // their logits in units of log2, per product
  bool opened = false, whole = false;
  float* shared_rec = reinterpret_cast<float*>(smem + kRecordAt);
  const int unit0 = cur.unit, b0 = cur.b;
  const bool empty = cur.at >= end;
  int seg_slot = 0, use = 0;
  bool more = cur.at < end;
  for (bool begun = false; more; begun = true) {
    const int head = cur.unit / a.parts;
    const int h0 = head * a.group + (cur.unit % a.parts) * ROWS;
    const int nh = min(ROWS, (head + 1) * a.group - h0);
    if (!opened) {
      opened = true;
      whole = cur.tile == 0;
      seg_slot = begun;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
#pragma unroll
        for (int d = 0; d < KS; ++d)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[d][h][x] = 0.f;
        m[h][0] = m[h][1] = -INFINITY;
        l[h][0] = l[h][1] = 0.f;
        const uint8_t* row = qs + (quad + 8 * h) * Sh::kQPitch;
        float ks = a.scale * kLog2e;
        if constexpr (DT == D3_DTYPE_E4M3) {
          // the row's largest element decides its power of two
          float top = 0.f;
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const uint2 x = *reinterpret_cast<const uint2*>(row + 32 * s + 8 * t4);
            top = fmaxf(top, fmaxf(fabsf(__uint_as_float(x.x << 16)), fabsf(__uint_as_float(x.x & 0xffff0000u))));
            top = fmaxf(top, fmaxf(fabsf(__uint_as_float(x.y << 16)), fabsf(__uint_as_float(x.y & 0xffff0000u))));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          int e = 0;
          if (top > 0.f && isfinite(top)) frexpf(top, &e);
          e = max(-126, min(126, e));  // 2^-e and 2^e both exist (the largest bf16 becomes 4)
          const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
          // k index 2 t4 + {0, 1, 8, 9} stands for column 4 t4 + {0, 1, 2, 3}, as in the keys below
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const uint2 y = *reinterpret_cast<const uint2*>(row + 32 * s + 8 * t4);
            qf[s][h][0] = pack16<false>(__uint_as_float(y.x << 16) * down, __uint_as_float(y.x & 0xffff0000u) * down);
            qf[s][h][1] = pack16<false>(__uint_as_float(y.y << 16) * down, __uint_as_float(y.y & 0xffff0000u) * down);
          }
          ks *= (a.k_scale ? __ldg(a.k_scale + head) : 1.0f) * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        } else {
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            qf[s][h][0] = *reinterpret_cast<const uint32_t*>(row + 32 * s + 4 * t4);
            qf[s][h][1] = *reinterpret_cast<const uint32_t*>(row + 32 * s + 4 * t4 + 16);
          }
        }
        // from the lanes that hold the head's column to those that hold its logits
        lg[h][0] = __shfl_sync(0xffffffffu, ks, 8 * t4);
        lg[h][1] = __shfl_sync(0xffffffffu, ks, 8 * t4 + 4);
      }
    }
    // the next loads go out before this tile's work
    load_keys();
    cp_async_wait<S - 1>();
    __syncwarp();
    const uint32_t ks = ring + use * Sh::kHalf;
    use = use + 1 == S ? 0 : use + 1;
    // logits: the keys are A's rows, the queries B's columns
    float s[MT][NH][4];
#pragma unroll
    for (int r = 0; r < MT; ++r)
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[r][h][x] = 0.f;
    const int mrow = lane & 7, mhi = (lane >> 3) & 1, mtop = lane >> 4;
    if constexpr (DT == D3_DTYPE_E4M3) {
#pragma unroll
      for (int c = 0; c < KS; c += 2)  // 16 bytes of a row are one k step
#pragma unroll
        for (int r = 0; r < MT; ++r) {
          uint32_t b[4];
          ldmatrix_x4(ks + tile_at<RB>(r * 16 + mhi * 8 + mrow, c + mtop), b[0], b[1], b[2], b[3]);
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t w0 = b[2 * y], w1 = b[2 * y + 1];  // keys 0-7, keys 8-15
            const uint32_t a0 = e4m3x2_to_f16x2(static_cast<uint16_t>(w0)), a1 = e4m3x2_to_f16x2(static_cast<uint16_t>(w1));
            const uint32_t a2 = e4m3x2_to_f16x2(static_cast<uint16_t>(w0 >> 16)), a3 = e4m3x2_to_f16x2(static_cast<uint16_t>(w1 >> 16));
#pragma unroll
            for (int h = 0; h < NH; ++h) mma_16816<false>(s[r][h], a0, a1, a2, a3, qf[c + y][h][0], qf[c + y][h][1]);
          }
        }
    } else {
#pragma unroll
      for (int c = 0; c < KS; ++c)
#pragma unroll
        for (int r = 0; r < MT; ++r) {
          uint32_t b[4];
          ldmatrix_x4(ks + tile_at<RB>(r * 16 + mhi * 8 + mrow, 2 * c + mtop), b[0], b[1], b[2], b[3]);
#pragma unroll
          for (int h = 0; h < NH; ++h) mma_16816<BF16>(s[r][h], b[0], b[1], b[2], b[3], qf[c][h][0], qf[c][h][1]);
        }
    }
    // keys past the end take no part
    const int left = cur.len - (cur.begin + cur.tile * Sh::kTile + warp * NK);
    uint32_t pb[MT][NH][2], pl[MT][NH][2];  // probabilities as B operands; what their rounding lost
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      float mn[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float top = -INFINITY;
#pragma unroll
        for (int r = 0; r < MT; ++r)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float& z = s[r][h][2 * y + x];
            z = r * 16 + y * 8 + quad < left ? z * lg[h][x] : -INFINITY;
            top = fmaxf(top, z);
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        mn[x] = fmaxf(m[h][x], top);
      }
      if (__any_sync(0xffffffffu, mn[0] > m[h][0] || mn[1] > m[h][1])) {  // some head has a new maximum: rescale
        float c[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          c[x] = exp2f(m[h][x] - (mn[x] == -INFINITY ? 0.f : mn[x]));
          l[h][x] *= c[x];
        }
#pragma unroll
        for (int d = 0; d < KS; ++d)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[d][h][x] *= c[x & 1];
      }
      float base[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        m[h][x] = mn[x];
        base[x] = mn[x] == -INFINITY ? 0.f : mn[x];  // no key yet, or only logits of -inf
      }
#pragma unroll
      for (int r = 0; r < MT; ++r)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float p0 = exp2f(s[r][h][2 * y] - base[0]), p1 = exp2f(s[r][h][2 * y + 1] - base[1]);
          l[h][0] += p0;
          l[h][1] += p1;
          const uint32_t hi = pack16<BF16>(p0 * PS, p1 * PS);
          pb[r][h][y] = movmatrix_trans(hi);  // a key's row of heads becomes a head's column of keys
          if constexpr (BF16)
            pl[r][h][y] = movmatrix_trans(pack16<true>(p0 - __uint_as_float(hi << 16), p1 - __uint_as_float(hi & 0xffff0000u)));
        }
    }
    // out^T += V^T P^T
    __syncwarp();  // every lane has read the keys' slot: it may be filled again
    load_values();
    cp_async_wait<S - 1>();
    __syncwarp();
    const uint32_t vs = ring + use * Sh::kHalf;
    use = use + 1 == S ? 0 : use + 1;
    if constexpr (DT == D3_DTYPE_E4M3) {
#pragma unroll
      for (int r = 0; r < MT; ++r)
#pragma unroll
        for (int c = 0; c < KS; c += 2) {
          uint32_t b[4];
          ldmatrix_x4_trans(vs + tile_at<RB>(r * 16 + mhi * 8 + mrow, c + mtop), b[0], b[1], b[2], b[3]);
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            // a 16-bit unit holds two neighbouring columns of a key: the even ones
            // become rows 0-7 of A, the odd ones rows 8-15
            const uint32_t w0 = b[2 * y], w1 = b[2 * y + 1];
            const uint32_t a0 = e4m3x2_to_f16x2(static_cast<uint16_t>(__byte_perm(w0, 0, 0x0020)));
            const uint32_t a1 = e4m3x2_to_f16x2(static_cast<uint16_t>(__byte_perm(w0, 0, 0x0031)));
            const uint32_t a2 = e4m3x2_to_f16x2(static_cast<uint16_t>(__byte_perm(w1, 0, 0x0020)));
            const uint32_t a3 = e4m3x2_to_f16x2(static_cast<uint16_t>(__byte_perm(w1, 0, 0x0031)));
#pragma unroll
            for (int h = 0; h < NH; ++h) mma_16816<false>(o[c + y][h], a0, a1, a2, a3, pb[r][h][0], pb[r][h][1]);
          }
        }
    } else {
#pragma unroll
      for (int r = 0; r < MT; ++r)
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          uint32_t b[4];
          ldmatrix_x4_trans(vs + tile_at<RB>(r * 16 + mtop * 8 + mrow, 2 * c + mhi), b[0], b[1], b[2], b[3]);
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            mma_16816<BF16>(o[c][h], b[0], b[1], b[2], b[3], pb[r][h][0], pb[r][h][1]);
            if constexpr (BF16) mma_16816<true>(o[c][h], b[0], b[1], b[2], b[3], pl[r][h][0], pl[r][h][1]);
          }
        }
    }
    __syncwarp();  // the same for the values

    const bool last = cur.tile + 1 == cur.tiles;
    Cursor<Sh::kTile> nxt = cur;
    nxt.next(a);
    more = nxt.at < end;
    if (last || !more) {
      // join the warps: (max, sum) and output rows through shared memory
      opened = false;
      if (!LINE) cp_async_wait<0>();  // nothing is on its way to the ring any more
      if (more) fetch_q(nxt);
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          l[h][x] += __shfl_xor_sync(0xffffffffu, l[h][x], 4);
          l[h][x] += __shfl_xor_sync(0xffffffffu, l[h][x], 8);
          l[h][x] += __shfl_xor_sync(0xffffffffu, l[h][x], 16);
          if (quad == 0) {
            stat[warp * 32 + 8 * h + 2 * t4 + x] = m[h][x];
            stat[warp * 32 + 16 + 8 * h + 2 * t4 + x] = l[h][x];
          }
        }
      __syncthreads();
      whole = whole && last && (LINE || a.share < 2);
      float* rec = a.partial + (static_cast<int64_t>(blockIdx.x) * 2 + seg_slot) * Sh::kRecord;
      if (!LINE) rec = shared_rec;
      const float vsc = a.v_scale ? __ldg(a.v_scale + head) : 1.0f;
      // each warp scales its rows to the common maximum; JW at a time they are
      // added into JW buffers, in the order of the warps
#pragma unroll
      for (int w = 0; w < NH; ++w) {
        if (w) __syncthreads();
#pragma unroll 1
        for (int round = 0; round < kAttnWarps / JW; ++round) {
          if (warp / JW == round) {
            float f[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float top = -INFINITY;
#pragma unroll
              for (int y = 0; y < kAttnWarps; ++y) top = fmaxf(top, stat[y * 32 + 8 * w + 2 * t4 + x]);
              f[x] = exp2f(m[w][x] - (top == -INFINITY ? 0.f : top)) * (1.f / PS);
            }
            float* row = join + ((warp % JW) * 8 + 2 * t4) * JP;
#pragma unroll
            for (int d = 0; d < KS; ++d)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const float y0 = o[d][w][x], y1 = o[d][w][2 + x];  // rows quad, quad + 8
                if constexpr (DT == D3_DTYPE_E4M3) {
                  float2* at = reinterpret_cast<float2*>(row + x * JP + d * 16 + 2 * quad);
                  const float2 was = round ? *at : make_float2(0.f, 0.f);
                  *at = make_float2(fmaf(y0, f[x], was.x), fmaf(y1, f[x], was.y));
                } else {
                  float* at = row + x * JP + d * 16 + quad;
                  at[0] = fmaf(y0, f[x], round ? at[0] : 0.f);
                  at[8] = fmaf(y1, f[x], round ? at[8] : 0.f);
                }
              }
          }
          __syncthreads();
        }
        for (int e = tid * 4; e < 8 * D; e += kAttnThreads * 4) {
          const int r8 = e / D, d = e % D, r = r8 + 8 * w;
          if (r >= nh) continue;
          float top = -INFINITY;
#pragma unroll
          for (int x = 0; x < kAttnWarps; ++x) top = fmaxf(top, stat[x * 32 + r]);
          const float base = top == -INFINITY ? 0.f : top;
          float sum = 0.f, x[4] = {};
#pragma unroll
          for (int y = 0; y < kAttnWarps; ++y) sum += exp2f(stat[y * 32 + r] - base) * stat[y * 32 + 16 + r];
#pragma unroll
          for (int z = 0; z < JW; ++z) {
            const float4 y = *reinterpret_cast<const float4*>(join + (z * 8 + r8) * JP + d);
            x[0] += y.x;
            x[1] += y.y;
            x[2] += y.z;
            x[3] += y.w;
          }
          if (whole) {
            store_row<QBF16>(a, cur.b, h0 + r, d, x, sum, top, vsc);
          } else {
            *reinterpret_cast<float4*>(rec + r * D + d) = make_float4(x[0], x[1], x[2], x[3]);
            if (d == 0) {
              rec[ROWS * D + r] = top;
              rec[ROWS * D + ROWS + r] = sum;
            }
          }
        }
      }
      if (more) place_q();  // every warp took its queries before the barriers above
      __syncthreads();
    }
    cur = nxt;
  }
  cp_async_wait<0>();
  if (LINE || (a.share == 1 && !empty)) return;

  // join the cluster: CTA r takes the rows r, r + share, ... of all its CTAs' records
  // (one CTA alone comes here for a sequence without keys)
  if (empty)
    for (int r = tid; r < ROWS; r += kAttnThreads) {
      shared_rec[ROWS * D + r] = -INFINITY;
      shared_rec[ROWS * D + ROWS + r] = 0.f;
    }
  if (a.share > 1) cluster_sync();
  else __syncthreads();
  const int head = unit0 / a.parts, h0 = head * a.group + (unit0 % a.parts) * ROWS;
  const int nh = min(ROWS, (head + 1) * a.group - h0);
  const float vsc = a.v_scale ? __ldg(a.v_scale + head) : 1.0f;
  const uint32_t rec = smem_u32(shared_rec);
  for (int e = tid * 4; e < ((nh - rank + a.share - 1) / a.share) * D; e += kAttnThreads * 4) {
    const int r = rank + e / D * a.share, d = e % D;
    float top = -INFINITY, sum = 0.f, x[4] = {};
    for (int c = 0; c < a.share; ++c) top = fmaxf(top, cluster_load(rec + (ROWS * D + r) * 4, c));
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 4
    for (int c = 0; c < a.share; ++c) {
      const float m = cluster_load(rec + (ROWS * D + r) * 4, c), l = cluster_load(rec + (ROWS * D + ROWS + r) * 4, c);
      if (m == -INFINITY && l == 0.f) continue;  // no key: its row was never written
      const float f = exp2f(m - base);
      const float4 y = cluster_load4(rec + (r * D + d) * 4, c);
      sum = fmaf(f, l, sum);
      x[0] = fmaf(f, y.x, x[0]);
      x[1] = fmaf(f, y.y, x[1]);
      x[2] = fmaf(f, y.z, x[2]);
      x[3] = fmaf(f, y.w, x[3]);
    }
    store_row<QBF16>(a, b0, h0 + r, d, x, sum, top, vsc);
  }
  if (a.share > 1) cluster_sync();  // no CTA's shared memory goes away while another reads it
}

// One CTA per query row: rows without keys get zeros, rows of units that several
// CTAs shared are joined from their records. Groups of D / 4 threads add up every
// (32 WARPS * 4 / D)-th record, so the loads of a long unit's records overlap; the
// groups are then added in order.
template <int DT, int D, bool WIDE, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) paged_attention_join_kernel(const AttnArgs a) {
  using Sh = AttnShape<DT, D, WIDE>;
  constexpr bool QBF16 = DT != D3_DTYPE_F16;
  constexpr int ROWS = Sh::kRows, THREADS = 32 * WARPS, LANES = D / 4, GROUPS = THREADS / LANES;
  extern __shared__ __align__(1024) uint8_t smem[];
  float4* acc = reinterpret_cast<float4*>(smem);                       // [GROUPS][LANES]
  float* fac = reinterpret_cast<float*>(smem) + THREADS * 4;      // [a.grid] maximum, then weight
  float* red = fac + a.grid;                                           // [2][warps]
  int* scratch = reinterpret_cast<int*>(red + 2 * WARPS);
  int* found = scratch + WARPS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x / a.q_heads, h = blockIdx.x % a.q_heads;
  const int head = h / a.group, part = (h - head * a.group) / ROWS, r = (h - head * a.group) % ROWS;
  const int unit = head * a.parts + part;
  const int per = (a.B + THREADS - 1) / THREADS;
  pdl_trigger();
  int mine, before, total;
  line_scan<Sh::kTile, WARPS>(a, per, scratch, mine, before, total);
  const int tiles = seq_tiles<Sh::kTile>(a, b);
  if (b / per == tid) {
    int at = before;
    for (int x = tid * per; x < b; ++x) at += seq_places<Sh::kTile>(a, x);
    *found = at + unit * (tiles + kUnitCost);
  }
  __syncthreads();
  const int share = max(1, cta_share(total, a.grid));
  const int lo = *found, hi = lo + kUnitCost + tiles;  // the unit's places on the line
  const int c0 = (lo + kUnitCost) / share, n = tiles > 0 ? (hi - 1) / share - c0 + 1 : 0;
  // every CTA waits: a kernel after this one waits for this grid only, which
  // must not be complete before the main kernel is
  pdl_wait();
  if (n == 1) return;
  // the first record lies in its CTA's second place where the CTA began with another unit
  const float* rec0 = a.partial + (static_cast<int64_t>(c0) * 2 + (lo > c0 * share)) * Sh::kRecord;
  const float* rec = a.partial + static_cast<int64_t>(c0) * 2 * Sh::kRecord;  // + 2 c records, c > 0
  auto record = [&](int c) { return c == 0 ? rec0 : rec + static_cast<int64_t>(c) * 2 * Sh::kRecord; };
  float top = -INFINITY, sum = 0.f;
  for (int c = tid; c < n; c += THREADS) {
    const float m = __ldcg(record(c) + ROWS * D + r);
    fac[c] = m;
    top = fmaxf(top, m);
  }
  top = warp_max(top);
  if (lane == 0) red[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) top = fmaxf(top, red[w]);
  const float base = top == -INFINITY ? 0.f : top;
  for (int c = tid; c < n; c += THREADS) {
    const float f = exp2f(fac[c] - base);
    fac[c] = f;
    sum += f * __ldcg(record(c) + ROWS * D + ROWS + r);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) red[WARPS + warp] = sum;
  __syncthreads();
  const int d = tid % LANES, g = tid / LANES;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int c = g; c < n; c += GROUPS) {
    const float4 y = __ldcg(reinterpret_cast<const float4*>(record(c) + r * D) + d);
    const float f = fac[c];
    x.x = fmaf(f, y.x, x.x);
    x.y = fmaf(f, y.y, x.y);
    x.z = fmaf(f, y.z, x.z);
    x.w = fmaf(f, y.w, x.w);
  }
  acc[g * LANES + d] = x;
  __syncthreads();
  if (g != 0) return;
  float out[4] = {};
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) sum += red[WARPS + w];
  for (int i = 0; i < GROUPS; ++i) {
    const float4 y = acc[i * LANES + d];
    out[0] += y.x;
    out[1] += y.y;
    out[2] += y.z;
    out[3] += y.w;
  }
  store_row<QBF16>(a, b, h, d * 4, out, sum, top, a.v_scale ? __ldg(a.v_scale + head) : 1.0f);
}

// How units of up to `tiles` tiles each are taken: by clusters of the returned number of
// CTAs (1: whole), or 0: all units' tiles as one line. Measured in us (bf16, 2 key heads of
// 256, tiles of 64): 1 sequence of 256 tokens by a cluster 7.0, as a line 8.7, of 1024 9.0
// and 9.4; 64 sequences of up to 256 whole 10.1, as a line 13.4, of up to 1024 as a line
// 23.4, whole about 30. The rule counts tiles for all types and dims. Each form beside the
// others for 1 to 64 sequences of 2 to 32 tiles, all as long as the bound, with heads of 64, 128
// and 256 in bf16, of 128 and 256 in e4m3 (tiles of 64 and of 128 keys), 246 cells: its choice
// is the best form or within 5% of it in 204, within 10% in 224. Where it is not: 8 to 16 tiles
// of many sequences (64 of 512 tokens, heads of 256: line 21.6, whole 17.2; the line is there for
// ragged lengths, which the host does not know), and 16 to 24 tiles of one sequence with short
// rows (24 tiles, 2 heads of 64: cluster 8.3, line 6.5).
int unit_ctas(int tiles, int64_t units, int grid) {
  if (tiles <= 2 || (tiles <= 6 && units * 4 >= grid)) return 1;  // short, or enough of them to fill the GPU
  int n = 8;
  while (n > 1 && (n / 2 >= tiles || units * n > grid)) n /= 2;
  return n > 1 && (tiles + n - 1) / n <= 3 ? n : 0;
}

template <int DT, int D, bool WIDE>
int launch_attention(AttnArgs& a, cudaStream_t s) {
  using Sh = AttnShape<DT, D, WIDE>;
  static bool ready[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    if (cudaFuncSetAttribute(paged_attention_kernel<DT, D, WIDE, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem) != cudaSuccess ||
        cudaFuncSetAttribute(paged_attention_kernel<DT, D, WIDE, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem) != cudaSuccess)
      return check_launch("d3_paged_attention");
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  const int keys = a.window > 0 && a.window < a.max_len ? a.window : a.max_len;
  a.share = unit_ctas((keys + Sh::kTile - 1) / Sh::kTile, static_cast<int64_t>(a.B) * a.units, a.grid);
  if (a.share > 0) {  // one launch: units of their own, or clusters that join by themselves
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.B * a.units * a.share));
    cfg.blockDim = dim3(kAttnThreads);
    cfg.dynamicSmemBytes = Sh::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(a.share);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.share > 1 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, paged_attention_kernel<DT, D, WIDE, false>, static_cast<AttnArgs>(a));
    return check_launch("d3_paged_attention");
  }
  launch_kernel(paged_attention_kernel<DT, D, WIDE, true>, dim3(a.grid), dim3(kAttnThreads), Sh::kSmem, s, a);
  // 256 threads a row where they fit at once, 128 for more rows (4 long sequences 162 us
  // against 167; 200 short ones 38 against 35)
  const unsigned rows = static_cast<unsigned>(a.B * a.q_heads);
  const size_t smem = (a.grid + 25) * 4;
  if (rows <= 8u * sm_count())
    launch_kernel(paged_attention_join_kernel<DT, D, WIDE, 8>, dim3(rows), dim3(256), 256 * 16 + smem, s, a);
  else
    launch_kernel(paged_attention_join_kernel<DT, D, WIDE, 4>, dim3(rows), dim3(128), 128 * 16 + smem, s, a);
  return check_launch("d3_paged_attention");
}

template <int DT, bool WIDE>
int launch_dim(AttnArgs& a, int D, cudaStream_t s) {
  if (D == 64) return launch_attention<DT, 64, WIDE>(a, s);
  if (D == 128) return launch_attention<DT, 128, WIDE>(a, s);
  return launch_attention<DT, 256, WIDE>(a, s);
}

}  // namespace
}  // namespace d3

using namespace d3;

extern "C" int d3_paged_attention_workspace_size(int B, int q_heads, int kv_heads, int dim, size_t* bytes) {
  D3_REQUIRE(bytes != nullptr, "bytes is NULL");
  D3_REQUIRE(B >= 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0,
             "query heads must be a multiple of key heads");
  D3_REQUIRE(dim == 64 || dim == 128 || dim == 256, "head dim must be 64, 128 or 256");
  const int rows = q_heads / kv_heads > 8 ? 16 : 8;
  *bytes = static_cast<size_t>(attn_ctas(dim, 1) * sm_count()) * 2 * rows * (dim + 2) * sizeof(float);
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
  // an offset below zero marks a row past its sequence's end
  D3_REQUIRE(cache->k_page_stride >= 0 && cache->k_token_stride >= 0 && cache->v_page_stride >= 0 && cache->v_token_stride >= 0,
             "negative page or token stride");
  D3_REQUIRE(cache->sequences == B, "the page table must have one row per query");
  if (workspace_bytes < need || !workspace)
    return set_error(D3_EWORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  D3_REQUIRE(aligned(workspace, 16), "the workspace must be 16-byte aligned");
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
  a.B = B;
  a.window = window;
  a.num_pages = cache->num_pages;
  a.page_size = cache->page_size;
  a.q_heads = q_heads;
  a.group = q_heads / cache->heads;
  // two groups of 8 heads share a read of the keys where there are more than 8
  const bool wide = a.group > 8;
  a.parts = (a.group + (wide ? 15 : 7)) / (wide ? 16 : 8);
  a.units = cache->heads * a.parts;
  a.scale = scale;
  a.partial = static_cast<float*>(workspace);
  const int D = cache->dim;
  a.grid = attn_ctas(D, static_cast<int>(e)) * sm_count();
  a.status = status;
  D3_REQUIRE(aligned(q, 16) && q_row_stride % 8 == 0 && q_head_stride % 8 == 0, "rows of q must be 16-byte aligned");
  D3_REQUIRE(aligned(out, 8) && out_row_stride % 4 == 0 && out_head_stride % 4 == 0, "rows of out must be 8-byte aligned");
  // the line of tiles (64 keys at least, see AttnShape) is counted in 32 bits
  // (and a token's number in a tile that passes the end of its sequence likewise)
  D3_REQUIRE(a.max_len <= 0x7fffff00 && static_cast<int64_t>(B) * a.units * (a.max_len / 64 + 2) < 0x40000000 &&
                 static_cast<int64_t>(B) * q_heads <= 0x7fffffff,
             "batch, heads and length are too large for one call");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (cache->dtype) {
    case D3_DTYPE_BF16: return wide ? launch_dim<D3_DTYPE_BF16, true>(a, D, s) : launch_dim<D3_DTYPE_BF16, false>(a, D, s);
    case D3_DTYPE_F16: return wide ? launch_dim<D3_DTYPE_F16, true>(a, D, s) : launch_dim<D3_DTYPE_F16, false>(a, D, s);
    default: return wide ? launch_dim<D3_DTYPE_E4M3, true>(a, D, s) : launch_dim<D3_DTYPE_E4M3, false>(a, D, s);
  }
}
