// The gated delta rule: S <- exp(g) S; S <- S + k (beta (v - S^T k))^T;
// out = S^T (scale q), one token per sequence or packed prompts.
//
// With S0 the state before the token, S^T k and the output need only two sums
// over the state: a = S0^T k and c = S0^T q give
//   d = beta (v - exp(g) a),  out = exp(g) c + (k.q) d,  S = exp(g) S0 + k d^T,
// so the state is read once and written once.
//
// One CTA per (sequence, value head, 32 value columns): thread (row group,
// column quad) keeps consecutive rows of 4 columns in registers. Everything a CTA
// reads is asked for at once, and the sums over the rows (with those of q.q, k.k and
// k.q, which give the norms) meet in one exchange. Bound by HBM: 64 sequences of 32
// heads of 128 x 128 (268 MB of state in and out) take 43.5 us, 6.2 TB/s or 0.96 of the
// copy rate; with the gates and values asked for after the exchange it was 48.5 us.
//
// Packed prompts go in chunks of 64 tokens. With G_i the sum of g up to token i
// of the chunk, k_i and q_i the normalised keys and scaled queries, and S0 the state
// before the chunk, the new values N (rows n_i, what token i writes along k_i) solve
//   (I + A) N = diag(beta) R,   A_ij = beta_i exp(G_i - G_j) k_i.k_j  (j < i),
//   R_i = v_i - exp(G_i) S0^T k_i,
// and then
//   out_i = exp(G_i) S0^T q_i + sum_{j<=i} P_ij n_j,   P_ij = exp(G_i - G_j) q_i.k_j,
//   S1 = exp(G_64) S0 + sum_j exp(G_64 - G_j) k_j n_j^T.
// The first equation is solved in two halves of 32 tokens: with T_h the inverse of
// I + A's diagonal block h, times diag(beta), and B_ij = exp(G_i - G_j) k_i.k_j,
//   N_0 = T_0 R_0,   N_1 = T_1 (R_1 - B_10 N_0).
// A first kernel makes T_0, T_1, B_10 and P for all chunks in parallel (they do not
// need the state); a second one walks each sequence's chunks with the state in
// registers.
//
// Rounding. All products run on mma.sync with bf16 factors and fp32 sums. Every factor of
// a product that reaches the state (S0, R, N, T, B) goes in two bf16 terms, 2^-17 of
// itself (together 2e-6 to 5e-6 of the state's norm after thousands of tokens); keys,
// queries and values are bf16 as they come, their norms factors outside. What only an
// output sees (S0 beside the queries, P) goes in one term, 2^-9, like the output itself.
// Three terms would cost half as many products again. So the state is off by 2e-6 to 5e-6 of
// its norm where fp32 products leave 2e-7 to 4e-7, and outputs by 2.3e-3 where one
// rounding leaves 1.7e-3; one token at a time (the step) is fp32 throughout.
//
// What bounds it. The state passes from chunk to chunk, so a sequence of 2048 tokens is 32
// steps of 2.4 us however much of the GPU is free (93 us in all, 75 of them the walk);
// of a step's 4400 cycles 2500 are tensor (316 products of 8 in the first warp of a pair),
// the rest the splitting, the short dependent products of the solve, and their operands. 64
// ragged prompts of 32 heads (17.5k tokens) take 535 us: the walk 410 at 0.60 of the
// rate of mma.sync and 0.33 of HBM's, the first kernel 125. tcgen05, with three times that
// rate, has not been tried: the state would go through tensor memory and registers five
// times a chunk (state, R, N and their terms), 500 columns of 32 lanes and about 2000
// instructions a thread, against the 12000 cycles that a chunk and head take of an SM now.
#include "d3_common.cuh"
#include "d3_host.h"
#include "mma_tiles.cuh"

#include <type_traits>

namespace d3 {
namespace {

constexpr int kDeltaThreads = 128;
constexpr int kDeltaCols = 32;  // value columns of one CTA

struct DeltaArgs {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  const float* g;
  const float* beta;
  __nv_bfloat16* out;
  float* state;
  const int32_t* slot;
  int64_t q_stride, k_stride, v_stride, g_stride, beta_stride, out_stride, slot_stride;
  int slots, rep, value_heads;
  int l2norm;
  float scale, eps;
  int32_t* status;
};

// 2^x, results below 2^-126 as zero (decays: they are added to what they vanish beside).
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// State slot of sequence i, or -1 when it is left out.
__device__ __forceinline__ int delta_slot(const DeltaArgs& a, int i) {
  const int s = a.slot ? __ldg(a.slot + i) : i;
  if (s >= a.slots) {
    if (a.status) atomicExch(a.status, kDevBadRow);
    return -1;
  }
  return s;
}

// One token for each sequence.
template <int DK, int DV>
__global__ void __launch_bounds__(kDeltaThreads)
    gated_delta_step_kernel(const DeltaArgs a) {
  constexpr int R = DK / 16;  // state rows of a thread: R * (row group) ...
  __shared__ float4 s_part[4][2][kDeltaCols / 4];
  __shared__ float s_dot[4][3];
  pdl_enter();
  const int seq = blockIdx.z, h = blockIdx.y, c0 = blockIdx.x * kDeltaCols;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cq = (tid & 7) * 4, rg = tid >> 3;
  const int hk = h / a.rep;
  const int slot = delta_slot(a, seq);
  __nv_bfloat16* out = a.out + seq * a.out_stride + h * DV + c0;
  if (slot < 0) {
    if (tid < kDeltaCols / 4) *reinterpret_cast<uint2*>(out + tid * 4) = make_uint2(0, 0);
    return;
  }
  float* S = a.state + slot * a.slot_stride + static_cast<int64_t>(h) * DK * DV + (rg * R) * DV + c0 + cq;
  float4 s[R];
#pragma unroll
  for (int r = 0; r < R; ++r) s[r] = *reinterpret_cast<const float4*>(S + r * DV);
  uint32_t qw[R / 2], kw[R / 2];
  const __nv_bfloat16 *qp = a.q + seq * a.q_stride + hk * DK + rg * R, *kp = a.k + seq * a.k_stride + hk * DK + rg * R;
  if constexpr (R == 8) {
    const uint4 x = *reinterpret_cast<const uint4*>(qp), y = *reinterpret_cast<const uint4*>(kp);
    qw[0] = x.x; qw[1] = x.y; qw[2] = x.z; qw[3] = x.w;
    kw[0] = y.x; kw[1] = y.y; kw[2] = y.z; kw[3] = y.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(qp), y = *reinterpret_cast<const uint2*>(kp);
    qw[0] = x.x; qw[1] = x.y;
    kw[0] = y.x; kw[1] = y.y;
  }
  const uint2 vw = *reinterpret_cast<const uint2*>(a.v + seq * a.v_stride + h * DV + c0 + cq);
  const float g = __ldg(a.g + seq * a.g_stride + h), beta = __ldg(a.beta + seq * a.beta_stride + h);
  float k[R], pa[4] = {}, pc[4] = {}, qq = 0.f, kk = 0.f, qk = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    k[r] = __uint_as_float(r & 1 ? kw[r / 2] & 0xffff0000u : kw[r / 2] << 16);
    const float q = __uint_as_float(r & 1 ? qw[r / 2] & 0xffff0000u : qw[r / 2] << 16);
    qq = fmaf(q, q, qq);
    kk = fmaf(k[r], k[r], kk);
    qk = fmaf(q, k[r], qk);
    pa[0] = fmaf(s[r].x, k[r], pa[0]); pa[1] = fmaf(s[r].y, k[r], pa[1]);
    pa[2] = fmaf(s[r].z, k[r], pa[2]); pa[3] = fmaf(s[r].w, k[r], pa[3]);
    pc[0] = fmaf(s[r].x, q, pc[0]); pc[1] = fmaf(s[r].y, q, pc[1]);
    pc[2] = fmaf(s[r].z, q, pc[2]); pc[3] = fmaf(s[r].w, q, pc[3]);
  }
#pragma unroll
  for (int x = 8; x <= 16; x <<= 1) {  // the 4 row groups of the warp
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      pa[j] += __shfl_xor_sync(0xffffffffu, pa[j], x);
      pc[j] += __shfl_xor_sync(0xffffffffu, pc[j], x);
    }
    qq += __shfl_xor_sync(0xffffffffu, qq, x);
    kk += __shfl_xor_sync(0xffffffffu, kk, x);
    qk += __shfl_xor_sync(0xffffffffu, qk, x);
  }
  if (lane < 8) {
    s_part[warp][0][lane] = make_float4(pa[0], pa[1], pa[2], pa[3]);
    s_part[warp][1][lane] = make_float4(pc[0], pc[1], pc[2], pc[3]);
    if (lane == 0) {
      s_dot[warp][0] = qq;
      s_dot[warp][1] = kk;
      s_dot[warp][2] = qk;
    }
  }
  __syncthreads();
  qq = kk = qk = 0.f;
  float xa[4] = {}, xc[4] = {};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    qq += s_dot[w][0];
    kk += s_dot[w][1];
    qk += s_dot[w][2];
    const float4 x = s_part[w][0][tid & 7], y = s_part[w][1][tid & 7];
    xa[0] += x.x; xa[1] += x.y; xa[2] += x.z; xa[3] += x.w;
    xc[0] += y.x; xc[1] += y.y; xc[2] += y.z; xc[3] += y.w;
  }
  const float rq = a.scale * (a.l2norm ? rsqrtf(qq + a.eps) : 1.f);
  const float rk = a.l2norm ? rsqrtf(kk + a.eps) : 1.f;
  const float eg = expf(g);
  const float v[4] = {__uint_as_float(vw.x << 16), __uint_as_float(vw.x & 0xffff0000u), __uint_as_float(vw.y << 16),
                      __uint_as_float(vw.y & 0xffff0000u)};
  float d[4], o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    d[j] = beta * (v[j] - eg * rk * xa[j]);
    o[j] = rq * (eg * xc[j] + qk * rk * d[j]);
  }
  if (rg == 0) *reinterpret_cast<uint2*>(out + cq) = make_uint2(pack16<true>(o[0], o[1]), pack16<true>(o[2], o[3]));
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float kr = k[r] * rk;
    *reinterpret_cast<float4*>(S + r * DV) = make_float4(fmaf(kr, d[0], eg * s[r].x), fmaf(kr, d[1], eg * s[r].y),
                                                         fmaf(kr, d[2], eg * s[r].z), fmaf(kr, d[3], eg * s[r].w));
  }
}


// ------------------------------------------------------------------ chunks --
constexpr int kC = 64;              // tokens of a chunk
constexpr int kPrepThreads = 256;
// What the first kernel leaves for one (chunk, value head): the matrix [T_0 0; B_10 T_1]
// in two bf16 terms and P in one, row-major 64 x 64 (16 x 16 blocks above the diagonal
// are not written), then the tokens' factors exp(G) / |k|, exp(G) scale / |q|,
// exp(G_64 - G) / |k| and exp(G_64).
constexpr int kRecT = kC * kC * 2, kRecScal = 3 * kRecT, kRecBytes = kRecScal + 1024;

// The chunks of sequence i have records cu[i] / 64 + i, ...: no two sequences share
// one, and no scan over the sequences is needed.
__device__ __forceinline__ int64_t first_record(int cu_i, int i) { return cu_i / kC + i; }
inline int64_t record_count(int T, int n) { return static_cast<int64_t>(T) / kC + n; }

struct ChunkArgs {
  DeltaArgs d;
  const int32_t* cu;
  const uint8_t* fresh;
  uint8_t* rec;
  int T, n;
};

// Copies rows [t0, t0 + 64) (zeros from t1 on) of BYTES bytes each into a tile, by
// THREADS threads of which this is number `thread`.
template <int BYTES, int THREADS>
__device__ __forceinline__ void load_rows(uint32_t tile, const __nv_bfloat16* src, int64_t stride, int t0, int t1, int thread) {
  constexpr int PIECES = BYTES / 16, STEP = THREADS / PIECES;
  const int r = thread / PIECES, c = thread % PIECES;
  const uint8_t* row = reinterpret_cast<const uint8_t*>(src + (t0 + r) * stride) + c * 16;
  const int64_t step = STEP * stride * 2;
#pragma unroll
  for (int i = 0; i < kC / STEP; ++i, row += step) {
    const bool take = t0 + r + i * STEP < t1;  // past the end nothing is read
    cp_async_16_zfill(tile + tile_at<BYTES>(r + i * STEP, c), take ? row : reinterpret_cast<const uint8_t*>(src), take);
  }
}

constexpr int kLd = 36;  // floats between rows of the fp32 matrices: 64 rows of a 32 x 32 block each

template <int DK>
struct PrepShape {
  static constexpr int kTile = kC * DK * 2;
  static constexpr int kMat = kC * kLd * 4;
  static constexpr int kT = 2 * kMat + 2 * 32 * 20 * 4;  // two heads' T and 16 x 16 products, over the dead tiles
  static constexpr int kTiles = 2 * kTile > kT ? 2 * kTile : kT;
  static constexpr int kSmem = kTiles + 2 * kMat + (2 * 4 * kC + 2 * kC * 3 + 2 * kC + 8) * 4;
};

// G_i - G_j of sums kept in two terms each: after strong decays both are large, and what
// one fp32 term leaves of their difference (2^-10 at 9600) would reach the state.
__device__ __forceinline__ float log_decay(float gi, float li, float gj, float lj) { return (gi - gj) + (li - lj); }

// exp(G_i - G_j) and the norms times the products of 16-row block I with the keys: P (ROLE
// 1), or I + A's strictly lower part and B_10 (ROLE 0). Left of the diagonal block the
// exponential is one factor of the row's by one of the column's, both at most 1.
template <int ROLE, int I>
__device__ __forceinline__ void prep_elements(const float (&acc)[8][4], int heads, uint8_t* rec0, const float* sG, const float* sL,
                                              const float* sB, const float* sRk, const float* sRow, const float* sW,
                                              float* A, int quad, int t4) {
  const int i0 = 16 * I + quad;
#pragma unroll 1
  for (int h = 0; h < heads; ++h) {
    const float *hG = sG + h * kC, *hL = sL + h * kC, *hW = sW + (h * 4 + I) * kC + 2 * t4;
    uint8_t* to = rec0 + h * kRecBytes + (ROLE ? 2 * kRecT : 0) + (i0 * kC + 2 * t4) * 2;
    float* Ah = A + (h * kC + i0) * kLd + 2 * t4;
    float f[2], a[2], b[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int i = i0 + 8 * half, end = I > 0 ? 16 * I - 1 : 0;
      f[half] = sRow[i];
      a[half] = I > 0 ? exp2_fast(log_decay(hG[i], hL[i], hG[end], hL[end])) * f[half] : 0.f;
      b[half] = ROLE ? 1.f : sB[h * kC + i0 + 8 * half];
    }
#pragma unroll
    for (int n = 0; n < 2 * I + 2; ++n) {
      const int j = n * 8 + 2 * t4;
      float e[2][2];
      if (n < 2 * I) {
        const float2 w = *reinterpret_cast<const float2*>(hW + n * 8);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          e[half][0] = acc[n][2 * half] * a[half] * w.x;
          e[half][1] = acc[n][2 * half + 1] * a[half] * w.y;
        }
      } else {  // nothing above the diagonal (there the difference may overflow)
        const float2 gj = *reinterpret_cast<const float2*>(hG + j), lj = *reinterpret_cast<const float2*>(hL + j),
                     rj = *reinterpret_cast<const float2*>(sRk + j);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int i = i0 + 8 * half;
          const float gi = hG[i], li = hL[i];
          e[half][0] = j <= i - (ROLE ? 0 : 1) ? exp2_fast(log_decay(gi, li, gj.x, lj.x)) * (rj.x * f[half]) * acc[n][2 * half] : 0.f;
          e[half][1] = j + 1 <= i - (ROLE ? 0 : 1) ? exp2_fast(log_decay(gi, li, gj.y, lj.y)) * (rj.y * f[half]) * acc[n][2 * half + 1] : 0.f;
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (ROLE) {
          *reinterpret_cast<uint32_t*>(to + half * (8 * kC * 2) + n * 16) = pack16<true>(e[half][0], e[half][1]);
        } else if (I >= 2 && n < 4) {
          uint32_t x, y;
          split_bf16x2(e[half][0], e[half][1], x, y);
          *reinterpret_cast<uint32_t*>(to + half * (8 * kC * 2) + n * 16) = x;
          *reinterpret_cast<uint32_t*>(to + kRecT + half * (8 * kC * 2) + n * 16) = y;
        } else {
          *reinterpret_cast<float2*>(Ah + half * 8 * kLd + (n & 3) * 8) = make_float2(e[half][0] * b[half], e[half][1] * b[half]);
        }
      }
    }
  }
}

// One CTA per (record, key head), two of its value heads at a time: bound by latency and
// instructions, not by its 278 MB (125 us for 305 chunks of 16 key heads, 45% of issue
// slots busy with four CTAs on an SM, for which it is held at 64 registers: 8 bytes are
// spilled). Warps 0-3 make k_i.k_j, warps 4-7 q_i.k_j, each for 16 rows; the two heads
// share them.
template <int DK>
__global__ void __launch_bounds__(kPrepThreads, 4) gated_delta_prep_kernel(const ChunkArgs a) {
  using Sh = PrepShape<DK>;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* Tm = reinterpret_cast<float*>(smem);                    // [2][64][kLd]
  float* X = Tm + 2 * kC * kLd;                                  // [2][32][20]
  float* A = reinterpret_cast<float*>(smem + Sh::kTiles);        // [2][64][kLd]
  float* sW = A + 2 * kC * kLd;  // [2][4][64] exp(G at the end of block I - 1 minus G_j) / |k_j|, j before block I
  float* sG = sW + 2 * 4 * kC;   // [2][64] sums of g, in units of log2
  float* sL = sG + 2 * kC;       // [2][64] their second terms
  float* sB = sL + 2 * kC;       // [2][64]
  float* sRk = sB + 2 * kC;
  float* sRq = sRk + kC;
  int* sSeq = reinterpret_cast<int*>(sRq + kC);  // [warps]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, t4 = lane & 3;
  const DeltaArgs& d = a.d;
  const int hk = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  // the sequence of this record, each thread looking at its own ones
  int lo = -1;
  for (int i = tid; i < a.n; i += kPrepThreads)
    if (first_record(max(0, __ldg(a.cu + i)), i) <= blockIdx.x && first_record(max(0, __ldg(a.cu + i + 1)), i + 1) > blockIdx.x) lo = i;
  lo = __reduce_max_sync(0xffffffffu, lo);
  if (lane == 0) sSeq[warp] = lo;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPrepThreads / 32; ++w) lo = max(lo, sSeq[w]);
  if (lo < 0) return;
  const int c0 = max(0, __ldg(a.cu + lo)), c1 = min(a.T, __ldg(a.cu + lo + 1));
  const int64_t chunk = static_cast<int64_t>(blockIdx.x) - first_record(c0, lo);
  if (chunk < 0 || c0 + chunk * kC >= c1) return;
  const int t0 = c0 + static_cast<int>(chunk) * kC, nt = min(kC, c1 - t0);

  const uint32_t kt = smem_u32(smem), qt = kt + Sh::kTile;
  load_rows<DK * 2, kPrepThreads>(kt, d.k + hk * DK, d.k_stride, t0, c1, tid);
  load_rows<DK * 2, kPrepThreads>(qt, d.q + hk * DK, d.q_stride, t0, c1, tid);
  cp_async_commit();
  // sums of the decays, and step sizes, of value heads hv0 and hv0 + 1: a warp each, two
  // tokens per lane
  auto gates = [&](int hv0) {
    if (warp >= 2) return;
    float g[2], be[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int t = 2 * lane + x;
      const bool in = t < nt && hv0 + warp < (hk + 1) * d.rep;
      // (a decay to below 2^-126 is 0 either way; the bound takes g = -infinity, a reset)
      g[x] = in ? __ldg(d.g + (t0 + t) * d.g_stride + hv0 + warp) * 1.4426950408889634f : 0.f;
      g[x] = g[x] < -150.f ? -150.f : g[x];
      be[x] = in ? __ldg(d.beta + (t0 + t) * d.beta_stride + hv0 + warp) : 0.f;
    }
    double sum = static_cast<double>(g[0]) + g[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    double before = __shfl_up_sync(0xffffffffu, sum, 1);
    if (lane == 0) before = 0.0;
    before += g[0];
    const float2 hi = make_float2(static_cast<float>(before), static_cast<float>(sum));
    *reinterpret_cast<float2*>(sG + warp * kC + 2 * lane) = hi;
    *reinterpret_cast<float2*>(sL + warp * kC + 2 * lane) =
        make_float2(static_cast<float>(before - hi.x), static_cast<float>(sum - hi.y));
    *reinterpret_cast<float2*>(sB + warp * kC + 2 * lane) = make_float2(be[0], be[1]);
  };
  gates(hk * d.rep);  // while the tiles are on their way
  cp_async_wait<0>();
  __syncthreads();
  const int role = warp >> 2, rows = 16 * (warp & 3);
  // products of rows `rows` .. + 15 with the keys up to the diagonal block, and the rows' norms
  float acc[8][4], norm[2] = {};
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x) acc[n][x] = 0.f;
  const int mrow = lane & 7, mhi = (lane >> 3) & 1, mtop = lane >> 4;
#pragma unroll
  for (int c = 0; c < DK / 16; ++c) {
    uint32_t x[4];
    // A operand: tiles (rows 0-7, k 0-7), (rows 8-15, k 0-7), (rows 0-7, k 8-15), (rows 8-15, k 8-15)
    ldmatrix_x4(kt + role * Sh::kTile + tile_at<DK * 2>(rows + mhi * 8 + mrow, 2 * c + mtop), x[0], x[1], x[2], x[3]);
#pragma unroll
    for (int n = 0; n < 8; n += 2) {
      if (n * 8 > rows) break;
      uint32_t b[4];
      ldmatrix_x4(kt + tile_at<DK * 2>(n * 8 + mtop * 8 + mrow, 2 * c + mhi), b[0], b[1], b[2], b[3]);
      mma_16816<true>(acc[n], x[0], x[1], x[2], x[3], b[0], b[1]);
      mma_16816<true>(acc[n + 1], x[0], x[1], x[2], x[3], b[2], b[3]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) norm[i & 1] = fma_bf16x2_seq(x[i], x[i], norm[i & 1]);  // rows quad, quad + 8
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    norm[i] += __shfl_xor_sync(0xffffffffu, norm[i], 1);
    norm[i] += __shfl_xor_sync(0xffffffffu, norm[i], 2);
    const int r = rows + quad + 8 * i;
    const float f = d.l2norm ? rsqrtf(norm[i] + d.eps) : 1.f;
    if (t4 == 0) (role ? sRq : sRk)[r] = r < nt ? (role ? d.scale * f : f) : 0.f;
  }
  for (int hv0 = hk * d.rep; hv0 < (hk + 1) * d.rep; hv0 += 2) {
    const int heads = min(2, (hk + 1) * d.rep - hv0);
    uint8_t* rec0 = a.rec + (static_cast<int64_t>(blockIdx.x) * d.value_heads + hv0) * kRecBytes;
    if (hv0 > hk * d.rep) {
      __syncthreads();  // the previous heads' are no longer read
      gates(hv0);
    }
    __syncthreads();  // nor are the tiles
    const int gh = tid >> 6, gt = tid & (kC - 1);  // (threads 0-127) head, token
    if (gh < heads) {
      float* f = reinterpret_cast<float*>(rec0 + gh * kRecBytes + kRecScal);
      const float G = sG[gh * kC + gt], end = sG[gh * kC + kC - 1];
      const float after = log_decay(end, sL[gh * kC + kC - 1], G, sL[gh * kC + gt]);
      f[gt] = exp2_fast(G) * sRk[gt];
      f[kC + gt] = exp2_fast(G) * sRq[gt];
      f[2 * kC + gt] = exp2_fast(after) * sRk[gt];
      if (gt == 0) f[3 * kC] = exp2_fast(end);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int x = e * kPrepThreads + tid, h = x >> 8, block = (x >> 6) & 3, j = x & (kC - 1);
      if (j < 16 * block) {
        const int at = h * kC + 16 * block - 1;
        sW[x] = exp2_fast(log_decay(sG[at], sL[at], sG[h * kC + j], sL[h * kC + j])) * sRk[j];
      }
    }
    __syncthreads();
    switch (warp) {  // each with its own straight code: shared and predicated it took twice as long
      case 0: prep_elements<0, 0>(acc, heads, rec0, sG, sL, sB, sRk, sRk, sW, A, quad, t4); break;
      case 1: prep_elements<0, 1>(acc, heads, rec0, sG, sL, sB, sRk, sRk, sW, A, quad, t4); break;
      case 2: prep_elements<0, 2>(acc, heads, rec0, sG, sL, sB, sRk, sRk, sW, A, quad, t4); break;
      case 3: prep_elements<0, 3>(acc, heads, rec0, sG, sL, sB, sRk, sRk, sW, A, quad, t4); break;
      case 4: prep_elements<1, 0>(acc, heads, rec0, sG, sL, sB, sRk, sRq, sW, A, quad, t4); break;
      case 5: prep_elements<1, 1>(acc, heads, rec0, sG, sL, sB, sRk, sRq, sW, A, quad, t4); break;
      case 6: prep_elements<1, 2>(acc, heads, rec0, sG, sL, sB, sRk, sRq, sW, A, quad, t4); break;
      default: prep_elements<1, 3>(acc, heads, rec0, sG, sL, sB, sRk, sRq, sW, A, quad, t4); break;
    }
    __syncthreads();
    // (I + A)^-1 of the diagonal blocks of 16, one per warp: columns of the two blocks of
    // 8 by forward substitution, then [T1 0; -T2 A21 T1, T2]
    if ((warp >> 2) < heads) {
      const int b = warp & 3, at = ((warp >> 2) * kC + 16 * b) * kLd + 16 * (b & 1);
      const float* Ab = A + at;
      float *Tb = Tm + at, *Xb = X + warp * 160;
      if (lane < 16) {
        const int o = lane & 8, c = lane & 7;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float y = 0.f;
#pragma unroll
          for (int j = 0; j < i; ++j) y = fmaf(Ab[(o + i) * kLd + o + j], x[j], y);
          x[i] = i < c ? 0.f : i == c ? 1.f : -y;
          Tb[(o + i) * kLd + o + c] = x[i];
        }
      }
      __syncwarp();
      const int r = lane >> 2, c = (lane & 3) * 2;
      float x0 = 0.f, x1 = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = Ab[(8 + r) * kLd + k];
        const float2 y = *reinterpret_cast<const float2*>(Tb + k * kLd + c);
        x0 = fmaf(w, y.x, x0);
        x1 = fmaf(w, y.y, x1);
      }
      *reinterpret_cast<float2*>(Xb + r * 20 + c) = make_float2(x0, x1);
      __syncwarp();
      x0 = x1 = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = Tb[(8 + r) * kLd + 8 + k];
        const float2 y = *reinterpret_cast<const float2*>(Xb + k * 20 + c);
        x0 = fmaf(w, y.x, x0);
        x1 = fmaf(w, y.y, x1);
      }
      *reinterpret_cast<float2*>(Tb + (8 + r) * kLd + c) = make_float2(-x0, -x1);
      *reinterpret_cast<float2*>(Tb + r * kLd + 8 + c) = make_float2(0.f, 0.f);  // read by the next level
    }
    __syncthreads();
    // from 16 to 32: [T1 0; -T2 A21 T1, T2]
    {
      const int h = tid >> 7, p = (tid >> 6) & 1, r = (tid & 63) >> 2, c = (tid & 3) * 4;
      const float* Ah = A + (h * kC + 32 * p) * kLd;
      float* Th = Tm + (h * kC + 32 * p) * kLd;
      float* Xh = X + (h * 32 + 16 * p) * 20;
      float x[4] = {};
      if (h < heads) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float w = Ah[(16 + r) * kLd + k];
          const float4 y = *reinterpret_cast<const float4*>(Th + k * kLd + c);
          x[0] = fmaf(w, y.x, x[0]); x[1] = fmaf(w, y.y, x[1]); x[2] = fmaf(w, y.z, x[2]); x[3] = fmaf(w, y.w, x[3]);
        }
        *reinterpret_cast<float4*>(Xh + r * 20 + c) = make_float4(x[0], x[1], x[2], x[3]);
      }
      __syncthreads();
      if (h < heads) {
        float y[4] = {};
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float w = Th[(16 + r) * kLd + 16 + k];
          const float4 z = *reinterpret_cast<const float4*>(Xh + k * 20 + c);
          y[0] = fmaf(w, z.x, y[0]); y[1] = fmaf(w, z.y, y[1]); y[2] = fmaf(w, z.z, y[2]); y[3] = fmaf(w, z.w, y[3]);
        }
        *reinterpret_cast<float4*>(Th + (16 + r) * kLd + c) = make_float4(-y[0], -y[1], -y[2], -y[3]);
      }
    }
    __syncthreads();
    // T diag(beta) in two bf16 terms, 8 elements at a time
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int x = e * kPrepThreads + tid, h = x >> 8, i = (x >> 2) & (kC - 1), j = (x & 3) * 8;
      if (h >= heads || j >= (i & 16) + 16) continue;
      const float *row = Tm + (h * kC + i) * kLd + j, *hB = sB + h * kC + (i & 32) + j;
      uint32_t p[4], q[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) split_bf16x2(row[2 * y] * hB[2 * y], row[2 * y + 1] * hB[2 * y + 1], p[y], q[y]);
      uint8_t* at = rec0 + h * kRecBytes + (i * kC + (i & 32) + j) * 2;
      *reinterpret_cast<uint4*>(at) = make_uint4(p[0], p[1], p[2], p[3]);
      *reinterpret_cast<uint4*>(at + kRecT) = make_uint4(q[0], q[1], q[2], q[3]);
    }
  }
}

// Shared memory: keys, queries, values and factors of two chunks, and T and P of one, whose
// place is free again by the time the state is updated, so that two CTAs share an SM. With
// PAIR (below) T and P of two, and what the warps of a pair hand over. W: warps of columns.
template <int DK, bool PAIR, int W>
struct WalkShape {
  static constexpr int kKT = kC * DK * 2, kV = kC * W * 32;
  static constexpr int kQ = kKT, kVAt = 2 * kKT, kF = kVAt + kV, kMat = kF + 1024;
  static constexpr int kStage = kMat + (PAIR ? 3 * kRecT : 0);
  static constexpr int kRec = 2 * kStage;  // the matrices, or the pairs' places
  static constexpr int kPairS = DK / 16 * 512, kPair = kPairS + 8 * 512;
  static constexpr int kSmem = kRec + (PAIR ? W * kPair : 3 * kRecT);
  static_assert(kSmem <= (PAIR ? 227 : 113) * 1024);
};

// Tokens from t0 on one after another, as the rule is defined, for the 16 value columns from
// `col` of value head hv: one warp, s laid out as in the walk. Ends at t1, or when the state's
// columns quad (lost0) and quad + 8 (lost1) that were asked for are not finite any more.
template <int DK>
__device__ __noinline__ void delta_tokens(float (&s)[DK / 8][4], const DeltaArgs d, int t0, int t1, int hv, int dv, int col,
                                          bool lost0, bool lost1) {
  const int lane = threadIdx.x & 31, quad = lane >> 2, t4 = lane & 3, hk = hv / d.rep;
#pragma unroll 1
  for (int t = t0; t < t1; ++t) {
    const uint32_t* kp = reinterpret_cast<const uint32_t*>(d.k + t * d.k_stride + hk * DK) + t4;
    const uint32_t* qp = reinterpret_cast<const uint32_t*>(d.q + t * d.q_stride + hk * DK) + t4;
    const __nv_bfloat16* vp = d.v + t * d.v_stride + hv * dv + col + quad;
    const float eg = expf(__ldg(d.g + t * d.g_stride + hv)), beta = __ldg(d.beta + t * d.beta_stride + hv);
    float kk = 0.f, qq = 0.f, x[2] = {}, y[2] = {};
#pragma unroll
    for (int n = 0; n < DK / 8; ++n) {
      const uint32_t w = __ldg(kp + 4 * n);
      const float k0 = __uint_as_float(w << 16), k1 = __uint_as_float(w & 0xffff0000u);
      kk = fmaf(k0, k0, fmaf(k1, k1, kk));
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        s[n][2 * c] *= eg;
        s[n][2 * c + 1] *= eg;
        x[c] = fmaf(s[n][2 * c], k0, fmaf(s[n][2 * c + 1], k1, x[c]));
      }
    }
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {  // the 4 lanes of a column
      kk += __shfl_xor_sync(0xffffffffu, kk, o);
      x[0] += __shfl_xor_sync(0xffffffffu, x[0], o);
      x[1] += __shfl_xor_sync(0xffffffffu, x[1], o);
    }
    const float rk = d.l2norm ? rsqrtf(kk + d.eps) : 1.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) x[c] = beta * (__bfloat162float(vp[8 * c]) - rk * x[c]) * rk;
#pragma unroll
    for (int n = 0; n < DK / 8; ++n) {
      const uint32_t w = __ldg(kp + 4 * n), z = __ldg(qp + 4 * n);
      const float q0 = __uint_as_float(z << 16), q1 = __uint_as_float(z & 0xffff0000u);
      qq = fmaf(q0, q0, fmaf(q1, q1, qq));
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        s[n][2 * c] = fmaf(__uint_as_float(w << 16), x[c], s[n][2 * c]);
        s[n][2 * c + 1] = fmaf(__uint_as_float(w & 0xffff0000u), x[c], s[n][2 * c + 1]);
        y[c] = fmaf(s[n][2 * c], q0, fmaf(s[n][2 * c + 1], q1, y[c]));
      }
    }
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
      qq += __shfl_xor_sync(0xffffffffu, qq, o);
      y[0] += __shfl_xor_sync(0xffffffffu, y[0], o);
      y[1] += __shfl_xor_sync(0xffffffffu, y[1], o);
    }
    const float rq = d.scale * (d.l2norm ? rsqrtf(qq + d.eps) : 1.f);
    if (t4 < 2) d.out[t * d.out_stride + hv * dv + col + quad + 8 * t4] = __float2bfloat16_rn(rq * (t4 ? y[1] : y[0]));
    if (!__any_sync(0xffffffffu, (lost0 && isfinite(s[0][0])) || (lost1 && isfinite(s[0][2])))) return;
  }
}

// One CTA per (16 W value columns, value head, sequence) walks the sequence's
// chunks. Warp w holds the transposed state of its 16 value columns, [16, DK], as
// mma accumulators: these are laid out like A operands, so the state, R and N go from
// product to product in registers, and warps share only what they read (keys,
// queries, T, P), which cp.async brings one chunk ahead. (A full 64 x 64 inverse in place
// of the two halves cost the first kernel more than it saved here; 8 warps on 128
// columns, one CTA per SM, took the same; loads spread between the products too.)
//
// PAIR, for few CTAs, where a chunk's latency is what counts: each warp has a second one
// beside it that takes what the next chunk does not wait for, the loads, S0^T q, P N and the
// output. It gets the state's first terms and N as the A operands they are, through
// shared memory (two named barriers a chunk). 2048 tokens of one sequence: 125 us without, 118
// with 64 columns, 93 with 32, where each warp has a scheduler and its tensor unit to itself.
// With many CTAs it would only take the place of a second CTA's warps.
template <int DK, int DV, bool PAIR, int W>
__global__ void __launch_bounds__(32 * W * (PAIR ? 2 : 1), PAIR ? 1 : 2) gated_delta_walk_kernel(const ChunkArgs a) {
  using Sh = WalkShape<DK, PAIR, W>;
  constexpr int VR = W * 32, LOADERS = 32 * W, THREADS = LOADERS * (PAIR ? 2 : 1);
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, quad = lane >> 2, t4 = lane & 3;
  const int warp = (tid >> 5) & (W - 1);      // its 16 columns
  const bool second = PAIR && tid >= LOADERS;  // the pair's second warp
  const bool loads = !PAIR || second;
  const int lt = PAIR ? tid - LOADERS : tid;     // number among those that load
  const int mrow = lane & 7, mhi = (lane >> 3) & 1, mtop = lane >> 4;
  const DeltaArgs& d = a.d;
  const int seq = blockIdx.z, hv = blockIdx.y, hk = hv / d.rep;
  const int col = blockIdx.x * 16 * W;  // first value column of the CTA
  pdl_wait();
  pdl_trigger();
  const int c0 = max(0, __ldg(a.cu + seq)), c1 = min(a.T, __ldg(a.cu + seq + 1));
  const int slot = delta_slot(d, seq);
  if (slot < 0) {
    for (int64_t e = tid; e < static_cast<int64_t>(c1 - c0) * (2 * W); e += THREADS)
      *reinterpret_cast<uint4*>(d.out + (c0 + e / (2 * W)) * d.out_stride + hv * DV + col + e % (2 * W) * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  const uint8_t* rec = a.rec + (first_record(c0, seq) * d.value_heads + hv) * kRecBytes;
  const int64_t rec_step = static_cast<int64_t>(d.value_heads) * kRecBytes;
  const uint32_t sm = smem_u32(smem);
  auto load_tokens = [&](int stage, int t0, const uint8_t* rec) {
    const uint32_t s = sm + stage * Sh::kStage;
    load_rows<DK * 2, LOADERS>(s, d.k + hk * DK, d.k_stride, t0, c1, lt);
    load_rows<DK * 2, LOADERS>(s + Sh::kQ, d.q + hk * DK, d.q_stride, t0, c1, lt);
    load_rows<VR, LOADERS>(s + Sh::kVAt, d.v + hv * DV + col, d.v_stride, t0, c1, lt);
    if (lt < 49) cp_async_16(smem + stage * Sh::kStage + Sh::kF + lt * 16, rec + kRecScal + lt * 16);
  };
  auto load_matrices = [&](int stage, const uint8_t* rec) {  // blocks up to the diagonal
    uint8_t* to = smem + (PAIR ? stage * Sh::kStage + Sh::kMat : Sh::kRec);
#pragma unroll
    for (int i = 0; i < 3 * kC * 8 / LOADERS; ++i) {
      const int e = i * LOADERS + lt, r = (e >> 3) & (kC - 1), c = e & 7, m = e / (kC * 8);
      if (c < (r >> 4) * 2 + 2) cp_async_16(to + m * kRecT + tile_at<128>(r, c), rec + m * kRecT + r * 128 + c * 16);
    }
  };
  float* S = d.state + slot * d.slot_stride + static_cast<int64_t>(hv) * DK * DV + col + 16 * warp;
  float s[DK / 8][4];
  const bool zero = a.fresh && a.fresh[seq];
  if (loads && c0 < c1) {
    load_tokens(0, c0, rec);
    load_matrices(0, rec);
  }
  cp_async_commit();
#pragma unroll
  for (int n = 0; n < DK / 8; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x)
      s[n][x] = zero || second ? 0.f : S[(n * 8 + 2 * t4 + (x & 1)) * DV + quad + (x >> 1) * 8];

  int stage = 0;
  for (int t0 = c0; t0 < c1; t0 += kC, stage ^= 1) {
    cp_async_wait<0>();
    __syncthreads();     // and every warp is done with the other stage
    if (loads && t0 + kC < c1) {
      load_tokens(stage ^ 1, t0 + kC, rec + rec_step);
      if (PAIR) load_matrices(stage ^ 1, rec + rec_step);
    }
    cp_async_commit();
    const uint32_t base = sm + stage * Sh::kStage, mat = PAIR ? base + Sh::kMat : sm + Sh::kRec;
    const float* f = reinterpret_cast<const float*>(smem + stage * Sh::kStage + Sh::kF);
    float o[8][4];
    // out += P N's block k, which has the terms h and l
    auto add_pn = [&](int k, const uint32_t (&h)[4], const uint32_t (&l)[4]) {
      uint32_t b[8][2];
#pragma unroll
      for (int n = 2 * k; n < 8; n += 2)
        ldmatrix_x4(mat + 2 * kRecT + tile_at<128>(n * 8 + mtop * 8 + mrow, 2 * k + mhi), b[n][0], b[n][1], b[n + 1][0], b[n + 1][1]);
#pragma unroll
      for (int n = 2 * k; n < 8; ++n) mma_16816<true>(o[n], h[0], h[1], h[2], h[3], b[n][0], b[n][1]);
#pragma unroll
      for (int n = 2 * k; n < 8; ++n) mma_16816<true>(o[n], l[0], l[1], l[2], l[3], b[n][0], b[n][1]);
    };
    // the output's 16 columns of 64 tokens, turned in shared memory: in the place of the
    // values, which no other pair reads
    auto put_out = [&]() {
#pragma unroll
      for (int n = 0; n < 8; n += 2)
        stmatrix_x4_trans(base + Sh::kVAt + tile_at<VR>(n * 8 + mtop * 8 + mrow, 2 * warp + mhi), pack16<true>(o[n][0], o[n][1]),
                          pack16<true>(o[n][2], o[n][3]), pack16<true>(o[n + 1][0], o[n + 1][1]), pack16<true>(o[n + 1][2], o[n + 1][3]));
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = i * 16 + (lane >> 1);
        if (t0 + t < c1)
          *reinterpret_cast<uint4*>(d.out + (t0 + t) * d.out_stride + hv * DV + col + 16 * warp + (lane & 1) * 8) =
              *reinterpret_cast<const uint4*>(smem + stage * Sh::kStage + Sh::kVAt + tile_at<VR>(t, 2 * warp + (lane & 1)));
      }
    };
    auto scale_out = [&](int n) {  // by exp(G) scale / |q|
      const float2 g = *reinterpret_cast<const float2*>(f + kC + n * 8 + 2 * t4);
      o[n][0] *= g.x;
      o[n][1] *= g.y;
      o[n][2] *= g.x;
      o[n][3] *= g.y;
    };
    uint4* pair = reinterpret_cast<uint4*>(smem + Sh::kRec + warp * Sh::kPair) + lane;  // (PAIR) operands, 32 lanes each
    if (second) {
      named_bar_sync(1 + warp, 64);
#pragma unroll
      for (int c = 0; c < DK / 16; ++c) {
        const uint4 h = pair[c * 32];
#pragma unroll
        for (int n = 0; n < 8; n += 2) {
          uint32_t q[4];
          ldmatrix_x4(base + Sh::kQ + tile_at<DK * 2>(n * 8 + mtop * 8 + mrow, 2 * c + mhi), q[0], q[1], q[2], q[3]);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (c == 0) mma_16816_first<true>(o[n + x], h.x, h.y, h.z, h.w, q[2 * x], q[2 * x + 1]);
            else mma_16816<true>(o[n + x], h.x, h.y, h.z, h.w, q[2 * x], q[2 * x + 1]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < 8; ++n) scale_out(n);
      named_bar_sync(1 + W + warp, 64);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 x = pair[(DK / 16 + 2 * k) * 32], y = pair[(DK / 16 + 2 * k + 1) * 32];
        const uint32_t h[4] = {x.x, x.y, x.z, x.w}, l[4] = {y.x, y.y, y.z, y.w};
        add_pn(k, h, l);
      }
      put_out();
      rec += rec_step;
      continue;
    }
    // S0^T k_j and S0^T q_j of the chunk's tokens
    float r[8][4];
    // (operands are read one step ahead of their products, and a sum's next product comes
    // four later: it takes about 21 cycles, one issues in 8)
    uint32_t kb[2][4], qb[2][4];
    auto read_kq = [&](int i) {  // step i: 16 columns c of 16 tokens n
      const uint32_t at = tile_at<DK * 2>((i & 3) * 16 + mtop * 8 + mrow, 2 * (i >> 2) + mhi);
      ldmatrix_x4(base + at, kb[i & 1][0], kb[i & 1][1], kb[i & 1][2], kb[i & 1][3]);
      if (!PAIR) ldmatrix_x4(base + Sh::kQ + at, qb[i & 1][0], qb[i & 1][1], qb[i & 1][2], qb[i & 1][3]);
    };
    read_kq(0);
    uint32_t hs[2][4], ls[2][4];
    auto split_s = [&](int c, int x) {  // a quarter of the state's terms for columns c
      split_bf16x2(s[2 * c + (x >> 1)][2 * (x & 1)], s[2 * c + (x >> 1)][2 * (x & 1) + 1], hs[c & 1][x], ls[c & 1][x]);
    };
#pragma unroll
    for (int x = 0; x < 4; ++x) split_s(0, x);
#pragma unroll
    for (int i = 0; i < DK / 4; ++i) {
      const int c = i >> 2, n = (i & 3) * 2;
      if (i + 1 < DK / 4) read_kq(i + 1);
      const uint32_t(&h)[4] = hs[c & 1];
      const uint32_t(&l)[4] = ls[c & 1];
      if (PAIR && n == 0) pair[c * 32] = make_uint4(h[0], h[1], h[2], h[3]);
      const uint32_t(&b)[4] = kb[i & 1];
      const uint32_t(&q)[4] = qb[i & 1];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (c == 0) mma_16816_first<true>(r[n + x], h[0], h[1], h[2], h[3], b[2 * x], b[2 * x + 1]);
        else mma_16816<true>(r[n + x], h[0], h[1], h[2], h[3], b[2 * x], b[2 * x + 1]);
      }
      // only the output sees the product with q: one bf16 term (2^-9) of the state
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (PAIR) continue;
        if (c == 0) mma_16816_first<true>(o[n + x], h[0], h[1], h[2], h[3], q[2 * x], q[2 * x + 1]);
        else mma_16816<true>(o[n + x], h[0], h[1], h[2], h[3], q[2 * x], q[2 * x + 1]);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) mma_16816<true>(r[n + x], l[0], l[1], l[2], l[3], b[2 * x], b[2 * x + 1]);
      if (c + 1 < DK / 16) split_s(c + 1, i & 3);
    }
    if (PAIR) named_bar_arrive(1 + warp, 64);
    // R = v - exp(G) S0^T k; its two terms as A operands over the tokens
    uint32_t rh[4][4] = {}, rl[4][4] = {};
#pragma unroll
    for (int n = 0; n < 8; n += 2) {
      uint32_t v[4];
      ldmatrix_x4_trans(base + Sh::kVAt + tile_at<VR>(n * 8 + mtop * 8 + mrow, 2 * warp + mhi), v[0], v[1], v[2], v[3]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float2 e = *reinterpret_cast<const float2*>(f + (n + x) * 8 + 2 * t4);
        float* y = r[n + x];
        y[0] = __uint_as_float(v[2 * x] << 16) - e.x * y[0];
        y[1] = __uint_as_float(v[2 * x] & 0xffff0000u) - e.y * y[1];
        y[2] = __uint_as_float(v[2 * x + 1] << 16) - e.x * y[2];
        y[3] = __uint_as_float(v[2 * x + 1] & 0xffff0000u) - e.y * y[3];
        if (!PAIR) scale_out(n + x);
      }
    }
    // the two terms of a 16-token column block of x
    auto split = [&](const float (&x)[8][4], int k, uint32_t (&h)[4], uint32_t (&l)[4]) {
#pragma unroll
      for (int y = 0; y < 4; ++y) split_bf16x2(x[2 * k + (y >> 1)][2 * (y & 1)], x[2 * k + (y >> 1)][2 * (y & 1) + 1], h[y], l[y]);
    };
    // w += (first: =) rows (tokens) 8 n .. of the matrix, 16 for each of PAIRS pairs, columns
    // 16 k .. + 15, times block k of x; w: the pairs' accumulators one after the other
    auto times = [&](auto pairs, float (*w)[4], int n, int k, bool first) {
      constexpr int PAIRS = decltype(pairs)::value;
      uint32_t b[PAIRS][4], c[PAIRS][4];
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const uint32_t at = tile_at<128>((n + 2 * i) * 8 + mtop * 8 + mrow, 2 * k + mhi);
        ldmatrix_x4(mat + at, b[i][0], b[i][1], b[i][2], b[i][3]);
        ldmatrix_x4(mat + kRecT + at, c[i][0], c[i][1], c[i][2], c[i][3]);
      }
#pragma unroll
      for (int i = 0; i < 2 * PAIRS; ++i) {
        if (first) mma_16816_first<true>(w[i], rh[k][0], rh[k][1], rh[k][2], rh[k][3], b[i / 2][2 * (i & 1)], b[i / 2][2 * (i & 1) + 1]);
        else mma_16816<true>(w[i], rh[k][0], rh[k][1], rh[k][2], rh[k][3], b[i / 2][2 * (i & 1)], b[i / 2][2 * (i & 1) + 1]);
      }
#pragma unroll
      for (int i = 0; i < 2 * PAIRS; ++i) mma_16816<true>(w[i], rl[k][0], rl[k][1], rl[k][2], rl[k][3], b[i / 2][2 * (i & 1)], b[i / 2][2 * (i & 1) + 1]);
#pragma unroll
      for (int i = 0; i < 2 * PAIRS; ++i) mma_16816<true>(w[i], rh[k][0], rh[k][1], rh[k][2], rh[k][3], c[i / 2][2 * (i & 1)], c[i / 2][2 * (i & 1) + 1]);
    };
    constexpr std::integral_constant<int, 1> one{};
    constexpr std::integral_constant<int, 2> two{};
    float w[8][4];
    // N_0 = T_0 R_0
    split(r, 0, rh[0], rl[0]);
    split(r, 1, rh[1], rl[1]);
    times(two, w, 0, 0, true);
    times(one, w + 2, 2, 1, false);
    // R_1 - B_10 N_0
    split(w, 0, rh[0], rl[0]);
    split(w, 1, rh[1], rl[1]);
    {
      float p[4][4];
      times(two, p, 4, 0, true);
      times(two, p, 4, 1, false);
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) r[4 + x][y] -= p[x][y];
    }
    // N_1 = T_1 (...)
    split(r, 2, rh[2], rl[2]);
    split(r, 3, rh[3], rl[3]);
    times(two, w + 4, 4, 2, true);
    times(one, w + 6, 6, 3, false);
    split(w, 2, rh[2], rl[2]);
    split(w, 3, rh[3], rl[3]);
    if (PAIR) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        pair[(DK / 16 + 2 * k) * 32] = make_uint4(rh[k][0], rh[k][1], rh[k][2], rh[k][3]);
        pair[(DK / 16 + 2 * k + 1) * 32] = make_uint4(rl[k][0], rl[k][1], rl[k][2], rl[k][3]);
      }
      named_bar_arrive(1 + W + warp, 64);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) add_pn(k, rh[k], rl[k]);
      __syncthreads();  // every warp is done with the matrices
      if (t0 + kC < c1) load_matrices(0, rec + rec_step);
      cp_async_commit();
      put_out();
    }
    rec += rec_step;
    // S = exp(G_64) S + k (exp(G_64 - G) n)^T
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float2 e = *reinterpret_cast<const float2*>(f + 2 * kC + (2 * k + (x >> 1)) * 8 + 2 * t4);
        split_bf16x2(w[2 * k + (x >> 1)][2 * (x & 1)] * e.x, w[2 * k + (x >> 1)][2 * (x & 1) + 1] * e.y, rh[k][x], rl[k][x]);
      }
    const float end = f[3 * kC];
    uint32_t kt[2][4][2];
    auto read_k = [&](int i) {  // step i: tokens 16 k .. of 4 columns of 8
      const int n = (i >> 2) * 4, k = i & 3;
      uint32_t(&b)[4][2] = kt[i & 1];
#pragma unroll
      for (int x = 0; x < 4; x += 2)
        ldmatrix_x4_trans(base + tile_at<DK * 2>(k * 16 + mhi * 8 + mrow, n + x + mtop), b[x][0], b[x][1], b[x + 1][0], b[x + 1][1]);
    };
    read_k(0);
    float p[4][4];
#pragma unroll
    for (int i = 0; i < DK / 8; ++i) {
      const int n = (i >> 2) * 4, k = i & 3;
      if (i + 1 < DK / 8) read_k(i + 1);
      const uint32_t(&b)[4][2] = kt[i & 1];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (k == 0) mma_16816_first<true>(p[x], rh[k][0], rh[k][1], rh[k][2], rh[k][3], b[x][0], b[x][1]);
        else mma_16816<true>(p[x], rh[k][0], rh[k][1], rh[k][2], rh[k][3], b[x][0], b[x][1]);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) mma_16816<true>(p[x], rl[k][0], rl[k][1], rl[k][2], rl[k][3], b[x][0], b[x][1]);
      if (k < 3) continue;
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) s[n + x][y] = fmaf(s[n + x][y], end, p[x][y]);
    }
  }
  // What is not finite meets the zeros above the diagonals of T and P and so reaches tokens up
  // to 15 before its own. It also stays in its columns of the state for good, every row of
  // them, so one look at the end finds it (asked in each chunk it cost 6 of 94 us); the warp then
  // writes its outputs up to there once more, token by token (1.7 us each). Later ones and the
  // state are as they should be.
  if (PAIR) __syncthreads();  // the second warps' outputs are written
  const bool lost0 = !second && !isfinite(s[0][0]), lost1 = !second && !isfinite(s[0][2]);
  if (__any_sync(0xffffffffu, lost0 || lost1) && c0 < c1) {
    float x[DK / 8][4];
#pragma unroll
    for (int n = 0; n < DK / 8; ++n)
#pragma unroll
      for (int y = 0; y < 4; ++y) x[n][y] = zero ? 0.f : S[(n * 8 + 2 * t4 + (y & 1)) * DV + quad + (y >> 1) * 8];
    __syncwarp();  // other lanes' outputs of the same columns
    delta_tokens<DK>(x, d, c0, c1, hv, DV, col + 16 * warp, lost0, lost1);
  }
#pragma unroll
  for (int n = 0; n < DK / 8; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (!second) S[(n * 8 + 2 * t4 + (x & 1)) * DV + quad + (x >> 1) * 8] = s[n][x];
}

int delta_args(const d3_gated_delta_t* p, int n, int T, int32_t* status, DeltaArgs& a) {
  D3_REQUIRE(p != nullptr, "the operand description is NULL");
  D3_REQUIRE((p->key_dim == 64 || p->key_dim == 128) && (p->value_dim == 64 || p->value_dim == 128),
             "key_dim and value_dim must be 64 or 128");
  D3_REQUIRE(p->key_heads > 0 && p->value_heads > 0 && p->value_heads % p->key_heads == 0,
             "value heads must be a multiple of key heads");
  D3_REQUIRE(n >= 0 && T >= 0 && p->slots >= 0, "negative size");
  D3_REQUIRE(p->slot != nullptr || n <= p->slots, "%d sequences and %d slots", n, p->slots);
  D3_REQUIRE(p->q_stride % 8 == 0 && p->k_stride % 8 == 0 && p->v_stride % 8 == 0 && p->out_stride % 8 == 0 &&
                 aligned(p->q, 16) && aligned(p->k, 16) && aligned(p->v, 16) && aligned(p->out, 16),
             "rows of q, k, v and out must be 16-byte aligned");
  D3_REQUIRE(aligned(p->state, 16) && p->slot_stride % 4 == 0, "state slots must be 16-byte aligned");
  D3_REQUIRE(n <= 65535 && p->value_heads <= 65535, "too many sequences or heads in one call");
  if (T > 0 && n > 0)
    D3_REQUIRE(p->q && p->k && p->v && p->g && p->beta && p->out && p->state, "NULL operand");
  a.q = static_cast<const __nv_bfloat16*>(p->q);
  a.k = static_cast<const __nv_bfloat16*>(p->k);
  a.v = static_cast<const __nv_bfloat16*>(p->v);
  a.g = p->g;
  a.beta = p->beta;
  a.out = static_cast<__nv_bfloat16*>(p->out);
  a.state = p->state;
  a.slot = p->slot;
  a.q_stride = p->q_stride;
  a.k_stride = p->k_stride;
  a.v_stride = p->v_stride;
  a.g_stride = p->g_stride;
  a.beta_stride = p->beta_stride;
  a.out_stride = p->out_stride;
  a.slot_stride = p->slot_stride;
  a.slots = p->slots;
  a.rep = p->value_heads / p->key_heads;
  a.value_heads = p->value_heads;
  a.l2norm = p->l2norm;
  a.scale = p->scale;
  a.eps = p->eps;
  a.status = status;
  return D3_OK;
}

using StepKernel = void (*)(const DeltaArgs);

StepKernel step_kernel(int dk, int dv) {
  if (dk == 64) return dv == 64 ? gated_delta_step_kernel<64, 64> : gated_delta_step_kernel<64, 128>;
  return dv == 64 ? gated_delta_step_kernel<128, 64> : gated_delta_step_kernel<128, 128>;
}

// Lets a kernel use `bytes` of dynamic shared memory (once per device).
template <typename K>
int allow_smem(K kern, int bytes, bool (&ready)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && ready[dev]) return D3_OK;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return check_launch("d3_gated_delta_chunk");
  if (dev >= 0 && dev < 64) ready[dev] = true;
  return D3_OK;
}

template <int DK>
int launch_prep(const ChunkArgs& a, cudaStream_t s) {
  static bool ready[64] = {};
  if (int rc = allow_smem(gated_delta_prep_kernel<DK>, PrepShape<DK>::kSmem, ready)) return rc;
  launch_kernel(gated_delta_prep_kernel<DK>, dim3(static_cast<unsigned>(record_count(a.T, a.n)), a.d.value_heads / a.d.rep),
                dim3(kPrepThreads), PrepShape<DK>::kSmem, s, a);
  return check_launch("d3_gated_delta_chunk");
}

template <int DK, int DV, bool PAIR, int W>
int launch_walk(const ChunkArgs& a, cudaStream_t s) {
  constexpr int kSmem = WalkShape<DK, PAIR, W>::kSmem;
  static bool ready[64] = {};
  if (int rc = allow_smem(gated_delta_walk_kernel<DK, DV, PAIR, W>, kSmem, ready)) return rc;
  launch_kernel(gated_delta_walk_kernel<DK, DV, PAIR, W>, dim3(DV / (16 * W), a.d.value_heads, a.n), dim3(32 * W * (PAIR ? 2 : 1)),
                kSmem, s, a);
  return check_launch("d3_gated_delta_chunk");
}

template <int DK, int DV>
int launch_walks(const ChunkArgs& a, cudaStream_t s) {
  // pairs of warps where every CTA has an SM of its own, with half the columns where
  // that still holds, so that no two warps of a CTA share a scheduler
  const int64_t heads = static_cast<int64_t>(a.d.value_heads) * a.n;
  if (heads * (DV / 32) <= sm_count()) return launch_walk<DK, DV, true, 2>(a, s);
  if (heads * (DV / 64) <= sm_count()) return launch_walk<DK, DV, true, 4>(a, s);
  return launch_walk<DK, DV, false, 4>(a, s);
}

template <int DK>
int launch_chunk(const ChunkArgs& a, int dv, cudaStream_t s) {
  if (a.T > 0)
    if (int rc = launch_prep<DK>(a, s)) return rc;
  return dv == 64 ? launch_walks<DK, 64>(a, s) : launch_walks<DK, 128>(a, s);
}

}  // namespace
}  // namespace d3

using namespace d3;

extern "C" int d3_gated_delta_step(const d3_gated_delta_t* args, int n, int32_t* status, d3_stream_t stream) {
  DeltaArgs a{};
  if (int rc = delta_args(args, n, n, status, a)) return rc;
  if (n == 0) return D3_OK;
  launch_kernel(step_kernel(args->key_dim, args->value_dim),
                dim3(args->value_dim / kDeltaCols, args->value_heads, n), dim3(kDeltaThreads), 0,
                reinterpret_cast<cudaStream_t>(stream), a);
  return check_launch("d3_gated_delta_step");
}

extern "C" int d3_gated_delta_chunk_workspace_size(int T, int n, int value_heads, int key_dim, int value_dim,
                                                   size_t* bytes) {
  D3_REQUIRE(bytes != nullptr, "bytes is NULL");
  D3_REQUIRE(T >= 0 && n >= 0 && value_heads > 0, "negative size");
  D3_REQUIRE((key_dim == 64 || key_dim == 128) && (value_dim == 64 || value_dim == 128),
             "key_dim and value_dim must be 64 or 128");
  *bytes = static_cast<size_t>(record_count(T, n)) * value_heads * kRecBytes;
  return D3_OK;
}

extern "C" int d3_gated_delta_chunk(const d3_gated_delta_t* args, const int32_t* cu, int T, int n,
                                    const uint8_t* fresh, void* workspace, size_t workspace_bytes,
                                    int32_t* status, d3_stream_t stream) {
  DeltaArgs a{};
  if (int rc = delta_args(args, n, T, status, a)) return rc;
  D3_REQUIRE(T <= 0x7fffff00, "too many tokens for one call");  // the last chunk's counter passes T
  size_t need = 0;
  if (int rc = d3_gated_delta_chunk_workspace_size(T, n, args->value_heads, args->key_dim, args->value_dim, &need)) return rc;
  if (workspace_bytes < need || (need && !workspace))
    return set_error(D3_EWORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (n == 0) return D3_OK;
  D3_REQUIRE(cu != nullptr && a.state != nullptr, "NULL operand");
  D3_REQUIRE(aligned(workspace, 16), "the workspace must be 16-byte aligned");
  const ChunkArgs c{a, cu, fresh, static_cast<uint8_t*>(workspace), T, n};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return args->key_dim == 64 ? launch_chunk<64>(c, args->value_dim, st) : launch_chunk<128>(c, args->value_dim, st);
}
