// The gated delta rule: S <- exp(g) S; S <- S + k (beta (v - S^T k))^T;
// out = S^T (scale q), one token per sequence or packed prompts.
//
// With S0 the state before the token, S^T k and the output need only two sums
// over the state: a = S0^T k and c = S0^T q give
//   d = beta (v - exp(g) a),  out = exp(g) c + (k.q) d,  S = exp(g) S0 + k d^T,
// so the state is read once and written once.
//
// One CTA per (sequence, value head, 32 value columns): thread (row group,
// column quad) keeps rows r, r + 16, ... of 4 columns in registers.
//
// Packed prompts go in chunks of 64 tokens. With G_i the sum of g up to token i
// of the chunk, k_i and q_i the normalised keys and scaled queries, and S0 the state
// before the chunk, the new values N (rows n_i, what token i writes along k_i) solve
//   (I + A) N = diag(beta) R,   A_ij = beta_i exp(G_i - G_j) k_i.k_j  (j < i),
//   R_i = v_i - exp(G_i) S0^T k_i,
// and then
//   out_i = exp(G_i) S0^T q_i + sum_{j<=i} P_ij n_j,   P_ij = exp(G_i - G_j) q_i.k_j,
//   S1 = exp(G_64) S0 + sum_j exp(G_64 - G_j) k_j n_j^T.
// A first kernel makes T = (I + A)^-1 diag(beta) and P for all chunks in parallel
// (they do not need the state); a second one walks each sequence's chunks with the
// state in registers. What follows from products of 16-bit factors runs on
// mma.sync; the state has to stay exact to fp32's neighbourhood, so every factor of
// a product that reaches it (S0, R, N, T) is split into two bf16 terms (2^-17),
// and the keys are taken as they come, bf16, with their norms as factors outside.
#include "d3_common.cuh"
#include "d3_host.h"
#include "mma_tiles.cuh"

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
  constexpr int R = DK / 16;  // state rows of a thread
  __shared__ float s_q[DK], s_k[DK];
  __shared__ float s_part[2][4][kDeltaCols];
  __shared__ float s_dot[3][4];
  pdl_enter();
  const int seq = blockIdx.z, h = blockIdx.y, c0 = blockIdx.x * kDeltaCols;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cq = (tid & 7) * 4, rg = tid >> 3;
  const int hk = h / a.rep;
  const int t = seq;
  const int slot = delta_slot(a, seq);
  if (slot < 0) {
    if (tid < kDeltaCols) a.out[t * a.out_stride + h * DV + c0 + tid] = __float2bfloat16_rn(0.f);
    return;
  }
  float* S = a.state + slot * a.slot_stride + static_cast<int64_t>(h) * DK * DV + c0 + cq;
  float s[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float4 x = *reinterpret_cast<const float4*>(S + (rg + 16 * r) * DV);
    s[r][0] = x.x; s[r][1] = x.y; s[r][2] = x.z; s[r][3] = x.w;
  }
  float qv = 0.f, kv = 0.f;
  if (tid < DK) {
    qv = __bfloat162float(a.q[t * a.q_stride + hk * DK + tid]);
    kv = __bfloat162float(a.k[t * a.k_stride + hk * DK + tid]);
    s_q[tid] = qv;
    s_k[tid] = kv;
  }
  float qq = qv * qv, kk = kv * kv, qk = qv * kv;
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    qq += __shfl_xor_sync(0xffffffffu, qq, x);
    kk += __shfl_xor_sync(0xffffffffu, kk, x);
    qk += __shfl_xor_sync(0xffffffffu, qk, x);
  }
  if (lane == 0) {
    s_dot[0][warp] = qq;
    s_dot[1][warp] = kk;
    s_dot[2][warp] = qk;
  }
  __syncthreads();
  qq = s_dot[0][0] + s_dot[0][1] + s_dot[0][2] + s_dot[0][3];
  kk = s_dot[1][0] + s_dot[1][1] + s_dot[1][2] + s_dot[1][3];
  qk = s_dot[2][0] + s_dot[2][1] + s_dot[2][2] + s_dot[2][3];
  const float rq = a.scale * (a.l2norm ? rsqrtf(qq + a.eps) : 1.f);
  const float rk = a.l2norm ? rsqrtf(kk + a.eps) : 1.f;
  float pa[4] = {}, pc[4] = {};
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float kr = s_k[rg + 16 * r], qr = s_q[rg + 16 * r];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      pa[j] = fmaf(s[r][j], kr, pa[j]);
      pc[j] = fmaf(s[r][j], qr, pc[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int x = 8; x <= 16; x <<= 1) {
      pa[j] += __shfl_xor_sync(0xffffffffu, pa[j], x);
      pc[j] += __shfl_xor_sync(0xffffffffu, pc[j], x);
    }
    if (lane < 8) {
      s_part[0][warp][cq + j] = pa[j];
      s_part[1][warp][cq + j] = pc[j];
    }
  }
  __syncthreads();
  const float eg = expf(__ldg(a.g + t * a.g_stride + h)), be = __ldg(a.beta + t * a.beta_stride + h);
  float d[4], o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float xa = s_part[0][0][cq + j] + s_part[0][1][cq + j] + s_part[0][2][cq + j] + s_part[0][3][cq + j];
    const float xc = s_part[1][0][cq + j] + s_part[1][1][cq + j] + s_part[1][2][cq + j] + s_part[1][3][cq + j];
    d[j] = be * (__bfloat162float(a.v[t * a.v_stride + h * DV + c0 + cq + j]) - eg * rk * xa);
    o[j] = rq * (eg * xc + qk * rk * d[j]);
  }
  if (rg == 0)
#pragma unroll
    for (int j = 0; j < 4; ++j) a.out[t * a.out_stride + h * DV + c0 + cq + j] = __float2bfloat16_rn(o[j]);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float kr = s_k[rg + 16 * r] * rk;
#pragma unroll
    for (int j = 0; j < 4; ++j) s[r][j] = fmaf(kr, d[j], eg * s[r][j]);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
    *reinterpret_cast<float4*>(S + (rg + 16 * r) * DV) = make_float4(s[r][0], s[r][1], s[r][2], s[r][3]);
}


// ------------------------------------------------------------------ chunks --
constexpr int kC = 64;              // tokens of a chunk
constexpr int kPrepThreads = 128;
// What the first kernel leaves for one (chunk, value head): T in two bf16 terms
// and P, row-major 64 x 64 (16 x 16 blocks above the diagonal are not written), then the
// tokens' factors exp(G) / |k|, exp(G) scale / |q|, exp(G_64 - G) / |k| and exp(G_64).
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

// Copies rows [t0, t0 + 64) (zeros from t1 on) of BYTES bytes each into a tile.
template <int BYTES, int THREADS>
__device__ __forceinline__ void load_rows(uint32_t tile, const __nv_bfloat16* src, int64_t stride, int t0, int t1) {
  constexpr int PIECES = BYTES / 16;
#pragma unroll
  for (int i = 0; i < kC * PIECES / THREADS; ++i) {
    const int e = i * THREADS + threadIdx.x, r = e / PIECES, c = e % PIECES;
    const bool take = t0 + r < t1;
    cp_async_16_zfill(tile + tile_at<BYTES>(r, c), reinterpret_cast<const uint8_t*>(src + (take ? t0 + r : t0) * stride) + c * 16, take);
  }
}

constexpr int kLd = 68;  // floats between rows of the 64 x 64 fp32 matrices

template <int DK>
struct PrepShape {
  static constexpr int kTile = kC * DK * 2;
  static constexpr int kT = kC * kLd * 4 + 32 * 36 * 4;  // T and a 32 x 32 product, over the dead tiles
  static constexpr int kTiles = 2 * kTile > kT ? 2 * kTile : kT;
  static constexpr int kSmem = kTiles + kC * kLd * 4 + 6 * kC * 4;
};

// One CTA per (record, key head): T, P and the factors of its value heads.
template <int DK>
__global__ void __launch_bounds__(kPrepThreads) gated_delta_prep_kernel(const ChunkArgs a) {
  using Sh = PrepShape<DK>;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* Tm = reinterpret_cast<float*>(smem);
  float* X = Tm + kC * kLd;
  float* A = reinterpret_cast<float*>(smem + Sh::kTiles);
  float* sG = A + kC * kLd;  // sums of g, in units of log2
  float* sB = sG + kC;
  float* sRk = sB + kC;
  float* sRq = sRk + kC;
  float* sScan = sRq + kC;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, t4 = lane & 3;
  const DeltaArgs& d = a.d;
  const int hk = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  // the sequence of this record: the last one whose first record is not behind it
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first_record(max(0, __ldg(a.cu + mid)), mid) <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const int c0 = max(0, __ldg(a.cu + lo)), c1 = min(a.T, __ldg(a.cu + lo + 1));
  const int64_t chunk = static_cast<int64_t>(blockIdx.x) - first_record(c0, lo);
  if (chunk < 0 || c0 + chunk * kC >= c1) return;
  const int t0 = c0 + static_cast<int>(chunk) * kC, nt = min(kC, c1 - t0);

  const uint32_t kt = smem_u32(smem), qt = kt + Sh::kTile;
  load_rows<DK * 2, kPrepThreads>(kt, d.k + hk * DK, d.k_stride, t0, c1);
  load_rows<DK * 2, kPrepThreads>(qt, d.q + hk * DK, d.q_stride, t0, c1);
  cp_async_commit();
  cp_async_wait<0>();
  __syncthreads();
  // norms: two threads per row
  {
    const int r = tid >> 1;
    float kk = 0.f, qq = 0.f;
#pragma unroll
    for (int c = 0; c < DK / 16; ++c) {
      const uint32_t at = tile_at<DK * 2>(r, c * 2 + (tid & 1));
      const uint4 x = *reinterpret_cast<const uint4*>(smem + at), y = *reinterpret_cast<const uint4*>(smem + Sh::kTile + at);
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        kk = fma_bf16x2_seq(xs[i], xs[i], kk);
        qq = fma_bf16x2_seq(ys[i], ys[i], qq);
      }
    }
    kk += __shfl_xor_sync(0xffffffffu, kk, 1);
    qq += __shfl_xor_sync(0xffffffffu, qq, 1);
    if ((tid & 1) == 0) {
      const bool in = r < nt;
      sRk[r] = !in ? 0.f : d.l2norm ? rsqrtf(kk + d.eps) : 1.f;
      sRq[r] = !in ? 0.f : d.scale * (d.l2norm ? rsqrtf(qq + d.eps) : 1.f);
    }
  }
  // k_i.k_j and q_i.k_j of rows 16 warp .. + 15, columns up to the diagonal block
  float kk[8][4], qk[8][4];
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x) kk[n][x] = qk[n][x] = 0.f;
  const int mrow = lane & 7, mhi = (lane >> 3) & 1, mtop = lane >> 4;
#pragma unroll
  for (int c = 0; c < DK / 16; ++c) {
    uint32_t ak[4], aq[4];
    // A operand: tiles (rows 0-7, k 0-7), (rows 8-15, k 0-7), (rows 0-7, k 8-15), (rows 8-15, k 8-15)
    const uint32_t at = tile_at<DK * 2>(16 * warp + mhi * 8 + mrow, 2 * c + mtop);
    ldmatrix_x4(kt + at, ak[0], ak[1], ak[2], ak[3]);
    ldmatrix_x4(qt + at, aq[0], aq[1], aq[2], aq[3]);
#pragma unroll
    for (int n = 0; n < 8; n += 2) {
      if (n > 2 * warp) break;
      uint32_t b[4];
      ldmatrix_x4(kt + tile_at<DK * 2>(n * 8 + mtop * 8 + mrow, 2 * c + mhi), b[0], b[1], b[2], b[3]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        mma_16816<true>(kk[n + x], ak[0], ak[1], ak[2], ak[3], b[2 * x], b[2 * x + 1]);
        mma_16816<true>(qk[n + x], aq[0], aq[1], aq[2], aq[3], b[2 * x], b[2 * x + 1]);
      }
    }
  }
  for (int hv = hk * d.rep; hv < (hk + 1) * d.rep; ++hv) {
    uint8_t* rec = a.rec + (static_cast<int64_t>(blockIdx.x) * d.value_heads + hv) * kRecBytes;
    __syncthreads();  // the tiles, or the previous head's matrices, are no longer read
    float G = 0.f;
    if (tid < kC) {
      G = tid < nt ? __ldg(d.g + (t0 + tid) * d.g_stride + hv) * 1.4426950408889634f : 0.f;
      sB[tid] = tid < nt ? __ldg(d.beta + (t0 + tid) * d.beta_stride + hv) : 0.f;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float y = __shfl_up_sync(0xffffffffu, G, o);
        if (lane >= o) G += y;
      }
      if (lane == 31) sScan[warp] = G;
    }
    __syncthreads();
    if (tid < kC) {
      if (warp == 1) G += sScan[0];
      sG[tid] = G;
    }
    __syncthreads();
    if (tid < kC) {
      float* f = reinterpret_cast<float*>(rec + kRecScal);
      const float end = sG[kC - 1];
      f[tid] = exp2f(G) * sRk[tid];
      f[kC + tid] = exp2f(G) * sRq[tid];
      f[2 * kC + tid] = exp2f(end - G) * sRk[tid];
      if (tid == 0) f[3 * kC] = exp2f(end);
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int i = 16 * warp + quad + 8 * half;
      const float gi = sG[i], bi = sB[i] * sRk[i], qi = sRq[i];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        if (n > 2 * warp + 1) break;
        const int j = n * 8 + 2 * t4;
        float p[2], w[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float e = j + x <= i ? exp2f(gi - sG[j + x]) * sRk[j + x] : 0.f;
          w[x] = j + x < i ? bi * e * kk[n][2 * half + x] : 0.f;
          p[x] = j + x <= i ? qi * e * qk[n][2 * half + x] : 0.f;
        }
        *reinterpret_cast<float2*>(A + i * kLd + j) = make_float2(w[0], w[1]);
        *reinterpret_cast<uint32_t*>(rec + 2 * kRecT + (i * kC + j) * 2) = pack16<true>(p[0], p[1]);
      }
    }
    __syncthreads();
    // T = (I + A)^-1. Diagonal blocks of 16: thread (block, column) substitutes forward.
    if (tid < kC) {
      const int b = tid >> 4, c = tid & 15;
      const float* Ab = A + (16 * b) * kLd + 16 * b;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < i; ++j) s = fmaf(Ab[i * kLd + j], x[j], s);
        x[i] = i < c ? 0.f : i == c ? 1.f : -s;
        Tm[(16 * b + i) * kLd + 16 * b + c] = x[i];
      }
    }
    __syncthreads();
    // [T1 0; -T2 A21 T1, T2] from 16 to 32
    {
      const int p = tid >> 6, r = (tid & 63) >> 2, c = (tid & 3) * 4, o = 32 * p;
      float x[4] = {};
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float w = A[(o + 16 + r) * kLd + o + k];
        const float4 y = *reinterpret_cast<const float4*>(Tm + (o + k) * kLd + o + c);
        x[0] = fmaf(w, y.x, x[0]); x[1] = fmaf(w, y.y, x[1]); x[2] = fmaf(w, y.z, x[2]); x[3] = fmaf(w, y.w, x[3]);
      }
      *reinterpret_cast<float4*>(X + (16 * p + r) * 36 + c) = make_float4(x[0], x[1], x[2], x[3]);
      __syncthreads();
      float y[4] = {};
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float w = Tm[(o + 16 + r) * kLd + o + 16 + k];
        const float4 z = *reinterpret_cast<const float4*>(X + (16 * p + k) * 36 + c);
        y[0] = fmaf(w, z.x, y[0]); y[1] = fmaf(w, z.y, y[1]); y[2] = fmaf(w, z.z, y[2]); y[3] = fmaf(w, z.w, y[3]);
      }
      *reinterpret_cast<float4*>(Tm + (o + 16 + r) * kLd + o + c) = make_float4(-y[0], -y[1], -y[2], -y[3]);
      // the block above the diagonal is read by the next level
      *reinterpret_cast<float4*>(Tm + (o + r) * kLd + o + 16 + c) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
    // and from 32 to 64
    {
      const int r = tid >> 2, c = (tid & 3) * 8;
      float x[8] = {};
#pragma unroll 8
      for (int k = 0; k < 32; ++k) {
        const float w = A[(32 + r) * kLd + k];
        const float4 y = *reinterpret_cast<const float4*>(Tm + k * kLd + c), z = *reinterpret_cast<const float4*>(Tm + k * kLd + c + 4);
        x[0] = fmaf(w, y.x, x[0]); x[1] = fmaf(w, y.y, x[1]); x[2] = fmaf(w, y.z, x[2]); x[3] = fmaf(w, y.w, x[3]);
        x[4] = fmaf(w, z.x, x[4]); x[5] = fmaf(w, z.y, x[5]); x[6] = fmaf(w, z.z, x[6]); x[7] = fmaf(w, z.w, x[7]);
      }
      *reinterpret_cast<float4*>(X + r * 36 + c) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(X + r * 36 + c + 4) = make_float4(x[4], x[5], x[6], x[7]);
      __syncthreads();
      float u[8] = {};
#pragma unroll 8
      for (int k = 0; k < 32; ++k) {
        const float w = Tm[(32 + r) * kLd + 32 + k];
        const float4 y = *reinterpret_cast<const float4*>(X + k * 36 + c), z = *reinterpret_cast<const float4*>(X + k * 36 + c + 4);
        u[0] = fmaf(w, y.x, u[0]); u[1] = fmaf(w, y.y, u[1]); u[2] = fmaf(w, y.z, u[2]); u[3] = fmaf(w, y.w, u[3]);
        u[4] = fmaf(w, z.x, u[4]); u[5] = fmaf(w, z.y, u[5]); u[6] = fmaf(w, z.z, u[6]); u[7] = fmaf(w, z.w, u[7]);
      }
      *reinterpret_cast<float4*>(Tm + (32 + r) * kLd + c) = make_float4(-u[0], -u[1], -u[2], -u[3]);
      *reinterpret_cast<float4*>(Tm + (32 + r) * kLd + c + 4) = make_float4(-u[4], -u[5], -u[6], -u[7]);
    }
    __syncthreads();
    // T diag(beta) in two bf16 terms, 8 elements at a time
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = (e * kPrepThreads + tid) >> 3, j = (tid & 7) * 8;
      if (j >= (i & ~15) + 16) continue;
      uint32_t h[4], l[4];
#pragma unroll
      for (int x = 0; x < 4; ++x)
        split_bf16x2(Tm[i * kLd + j + 2 * x] * sB[j + 2 * x], Tm[i * kLd + j + 2 * x + 1] * sB[j + 2 * x + 1], h[x], l[x]);
      *reinterpret_cast<uint4*>(rec + (i * kC + j) * 2) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4*>(rec + kRecT + (i * kC + j) * 2) = make_uint4(l[0], l[1], l[2], l[3]);
    }
  }
}

template <int DK, int WARPS>
struct WalkShape {
  static constexpr int kKT = kC * DK * 2, kVRow = WARPS * 32;
  static constexpr int kV = kC * kVRow;
  static constexpr int kK = 0, kQ = kKT, kRec = 2 * kKT, kVAt = kRec + kRecBytes, kStage = kVAt + kV;
  static constexpr int kOut = 2 * kStage;                 // 2 KB per warp
  static constexpr int kSmem = kOut + WARPS * 2048;
};

// One CTA per (16 WARPS value columns, value head, sequence) walks the sequence's
// chunks. Warp w holds the transposed state of its 16 value columns, [16, DK], as
// mma accumulators: these are laid out like A operands, so the state, R and N go from
// product to product in registers, and warps share only what they read (keys,
// queries, T, P), which cp.async brings one chunk ahead.
template <int DK, int DV, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) gated_delta_walk_kernel(const ChunkArgs a) {
  using Sh = WalkShape<DK, WARPS>;
  constexpr int THREADS = WARPS * 32, VR = Sh::kVRow;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, t4 = lane & 3;
  const int mrow = lane & 7, mhi = (lane >> 3) & 1, mtop = lane >> 4;
  const DeltaArgs& d = a.d;
  const int seq = blockIdx.z, hv = blockIdx.y, hk = hv / d.rep;
  const int col = blockIdx.x * WARPS * 16;  // first value column of the CTA
  pdl_wait();
  pdl_trigger();
  const int c0 = max(0, __ldg(a.cu + seq)), c1 = min(a.T, __ldg(a.cu + seq + 1));
  const int slot = delta_slot(d, seq);
  if (slot < 0) {
    for (int e = tid; e < (c1 - c0) * WARPS * 2; e += THREADS)
      *reinterpret_cast<uint4*>(d.out + (c0 + e / (WARPS * 2)) * d.out_stride + hv * DV + col + e % (WARPS * 2) * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  const uint8_t* rec = a.rec + (first_record(c0, seq) * d.value_heads + hv) * kRecBytes;
  const int64_t rec_step = static_cast<int64_t>(d.value_heads) * kRecBytes;
  auto load = [&](int stage, int t0) {
    const uint32_t s = smem_u32(smem) + stage * Sh::kStage;
    load_rows<DK * 2, THREADS>(s + Sh::kK, d.k + hk * DK, d.k_stride, t0, c1);
    load_rows<DK * 2, THREADS>(s + Sh::kQ, d.q + hk * DK, d.q_stride, t0, c1);
    load_rows<VR, THREADS>(s + Sh::kVAt, d.v + hv * DV + col, d.v_stride, t0, c1);
    // T (two terms) and P: blocks up to the diagonal
#pragma unroll
    for (int i = 0; i < 3 * kC * 8 / THREADS; ++i) {
      const int e = i * THREADS + tid, r = (e >> 3) & (kC - 1), c = e & 7, m = e / (kC * 8);
      if (c < (r >> 4) * 2 + 2) cp_async_16(smem + stage * Sh::kStage + Sh::kRec + m * kRecT + tile_at<128>(r, c), rec + m * kRecT + r * 128 + c * 16);
    }
    if (tid < 49) cp_async_16(smem + stage * Sh::kStage + Sh::kRec + kRecScal + tid * 16, rec + kRecScal + tid * 16);
    rec += rec_step;
  };
  float* S = d.state + slot * d.slot_stride + static_cast<int64_t>(hv) * DK * DV + col + 16 * warp;
  float s[DK / 8][4];
  const bool zero = a.fresh && a.fresh[seq];
  if (c0 < c1) load(0, c0);
  cp_async_commit();
#pragma unroll
  for (int n = 0; n < DK / 8; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x)
      s[n][x] = zero ? 0.f : S[(n * 8 + 2 * t4 + (x & 1)) * DV + quad + (x >> 1) * 8];

  int stage = 0;
  for (int t0 = c0; t0 < c1; t0 += kC, stage ^= 1) {
    if (t0 + kC < c1) load(stage ^ 1, t0 + kC);
    cp_async_commit();
    cp_async_wait<1>();
    __syncthreads();
    const uint32_t base = smem_u32(smem) + stage * Sh::kStage;
    const float* f = reinterpret_cast<const float*>(smem + stage * Sh::kStage + Sh::kRec + kRecScal);
    // S0^T k_j and S0^T q_j of the chunk's tokens
    float r[8][4], o[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) r[n][x] = o[n][x] = 0.f;
#pragma unroll
    for (int c = 0; c < DK / 16; ++c) {
      uint32_t h[4], l[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) split_bf16x2(s[2 * c + (x >> 1)][2 * (x & 1)], s[2 * c + (x >> 1)][2 * (x & 1) + 1], h[x], l[x]);
#pragma unroll
      for (int n = 0; n < 8; n += 2) {
        uint32_t b[4], q[4];
        const uint32_t at = tile_at<DK * 2>(n * 8 + mtop * 8 + mrow, 2 * c + mhi);
        ldmatrix_x4(base + Sh::kK + at, b[0], b[1], b[2], b[3]);
        ldmatrix_x4(base + Sh::kQ + at, q[0], q[1], q[2], q[3]);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          mma_16816<true>(r[n + x], h[0], h[1], h[2], h[3], b[2 * x], b[2 * x + 1]);
          mma_16816<true>(r[n + x], l[0], l[1], l[2], l[3], b[2 * x], b[2 * x + 1]);
          // only the output sees this product: one bf16 term (2^-9) of the state
          mma_16816<true>(o[n + x], h[0], h[1], h[2], h[3], q[2 * x], q[2 * x + 1]);
        }
      }
    }
    // R = v - exp(G) S0^T k; its two terms as A operands over the tokens
    uint32_t rh[4][4], rl[4][4];
#pragma unroll
    for (int n = 0; n < 8; n += 2) {
      uint32_t v[4];
      ldmatrix_x4_trans(base + Sh::kVAt + tile_at<VR>(n * 8 + mtop * 8 + mrow, 2 * warp + mhi), v[0], v[1], v[2], v[3]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float2 e = *reinterpret_cast<const float2*>(f + (n + x) * 8 + 2 * t4);
        const float2 g = *reinterpret_cast<const float2*>(f + kC + (n + x) * 8 + 2 * t4);
        float* y = r[n + x];
        y[0] = __uint_as_float(v[2 * x] << 16) - e.x * y[0];
        y[1] = __uint_as_float(v[2 * x] & 0xffff0000u) - e.y * y[1];
        y[2] = __uint_as_float(v[2 * x + 1] << 16) - e.x * y[2];
        y[3] = __uint_as_float(v[2 * x + 1] & 0xffff0000u) - e.y * y[3];
        o[n + x][0] *= g.x;
        o[n + x][1] *= g.y;
        o[n + x][2] *= g.x;
        o[n + x][3] *= g.y;
        split_bf16x2(y[0], y[1], rh[n / 2][2 * x], rl[n / 2][2 * x]);
        split_bf16x2(y[2], y[3], rh[n / 2][2 * x + 1], rl[n / 2][2 * x + 1]);
      }
    }
    // N = T R: token i needs tokens j <= i
    float w[8][4];
#pragma unroll
    for (int n = 0; n < 8; n += 2) {
#pragma unroll
      for (int x = 0; x < 4; ++x) w[n][x] = w[n + 1][x] = 0.f;
#pragma unroll
      for (int k = 0; k <= n / 2; ++k) {
        uint32_t b[4], c[4];
        const uint32_t at = tile_at<128>(n * 8 + mtop * 8 + mrow, 2 * k + mhi);
        ldmatrix_x4(base + Sh::kRec + at, b[0], b[1], b[2], b[3]);
        ldmatrix_x4(base + Sh::kRec + kRecT + at, c[0], c[1], c[2], c[3]);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          mma_16816<true>(w[n + x], rh[k][0], rh[k][1], rh[k][2], rh[k][3], b[2 * x], b[2 * x + 1]);
          mma_16816<true>(w[n + x], rl[k][0], rl[k][1], rl[k][2], rl[k][3], b[2 * x], b[2 * x + 1]);
          mma_16816<true>(w[n + x], rh[k][0], rh[k][1], rh[k][2], rh[k][3], c[2 * x], c[2 * x + 1]);
        }
      }
    }
    // out += P N
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int x = 0; x < 4; ++x) split_bf16x2(w[2 * k + (x >> 1)][2 * (x & 1)], w[2 * k + (x >> 1)][2 * (x & 1) + 1], rh[k][x], rl[k][x]);
#pragma unroll
      for (int n = 2 * k; n < 8; n += 2) {
        uint32_t b[4];
        ldmatrix_x4(base + Sh::kRec + 2 * kRecT + tile_at<128>(n * 8 + mtop * 8 + mrow, 2 * k + mhi), b[0], b[1], b[2], b[3]);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          mma_16816<true>(o[n + x], rh[k][0], rh[k][1], rh[k][2], rh[k][3], b[2 * x], b[2 * x + 1]);
          mma_16816<true>(o[n + x], rl[k][0], rl[k][1], rl[k][2], rl[k][3], b[2 * x], b[2 * x + 1]);
        }
      }
    }
    // S = exp(G_64) S + k (exp(G_64 - G) n)^T
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float2 e = *reinterpret_cast<const float2*>(f + 2 * kC + (2 * k + (x >> 1)) * 8 + 2 * t4);
        split_bf16x2(w[2 * k + (x >> 1)][2 * (x & 1)] * e.x, w[2 * k + (x >> 1)][2 * (x & 1) + 1] * e.y, rh[k][x], rl[k][x]);
      }
    const float end = f[3 * kC];
#pragma unroll
    for (int n = 0; n < DK / 8; n += 2) {
      float p[2][4] = {};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t b[4];
        ldmatrix_x4_trans(base + Sh::kK + tile_at<DK * 2>(k * 16 + mhi * 8 + mrow, n + mtop), b[0], b[1], b[2], b[3]);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          mma_16816<true>(p[x], rh[k][0], rh[k][1], rh[k][2], rh[k][3], b[2 * x], b[2 * x + 1]);
          mma_16816<true>(p[x], rl[k][0], rl[k][1], rl[k][2], rl[k][3], b[2 * x], b[2 * x + 1]);
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) s[n + x][y] = fmaf(s[n + x][y], end, p[x][y]);
    }
    // the output's 16 columns of 64 tokens, turned in shared memory
    uint8_t* ob = smem + Sh::kOut + warp * 2048;
#pragma unroll
    for (int n = 0; n < 8; n += 2)
      stmatrix_x4_trans(smem_u32(ob) + (n * 8 + mtop * 8 + mrow) * 32 + mhi * 16, pack16<true>(o[n][0], o[n][1]),
                        pack16<true>(o[n][2], o[n][3]), pack16<true>(o[n + 1][0], o[n + 1][1]), pack16<true>(o[n + 1][2], o[n + 1][3]));
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = i * 16 + (lane >> 1);
      if (t0 + t < c1)
        *reinterpret_cast<uint4*>(d.out + (t0 + t) * d.out_stride + hv * DV + col + 16 * warp + (lane & 1) * 8) =
            *reinterpret_cast<const uint4*>(ob + t * 32 + (lane & 1) * 16);
    }
    __syncthreads();  // this stage may be filled again
  }
#pragma unroll
  for (int n = 0; n < DK / 8; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x) S[(n * 8 + 2 * t4 + (x & 1)) * DV + quad + (x >> 1) * 8] = s[n][x];
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

template <int DK, int DV, int WARPS>
int launch_walk(const ChunkArgs& a, cudaStream_t s) {
  static bool ready[64] = {};
  if (int rc = allow_smem(gated_delta_walk_kernel<DK, DV, WARPS>, WalkShape<DK, WARPS>::kSmem, ready)) return rc;
  launch_kernel(gated_delta_walk_kernel<DK, DV, WARPS>, dim3(DV / (16 * WARPS), a.d.value_heads, a.n), dim3(WARPS * 32),
                WalkShape<DK, WARPS>::kSmem, s, a);
  return check_launch("d3_gated_delta_chunk");
}

template <int DK>
int launch_chunk(const ChunkArgs& a, int dv, cudaStream_t s) {
  if (a.T > 0)
    if (int rc = launch_prep<DK>(a, s)) return rc;
  if (dv == 64) return launch_walk<DK, 64, 4>(a, s);
  // few sequences: twice the CTAs of half the columns
  if (static_cast<int64_t>(a.n) * a.d.value_heads < sm_count()) return launch_walk<DK, 128, 4>(a, s);
  return launch_walk<DK, 128, 8>(a, s);
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
