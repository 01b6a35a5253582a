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
#include "d3_common.cuh"
#include "d3_host.h"

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

// Tokens [cu[i], cu[i+1]) of sequence i (cu == NULL: token i alone).
template <int DK, int DV>
__global__ void __launch_bounds__(kDeltaThreads)
    gated_delta_kernel(const DeltaArgs a, const int32_t* cu, int T, const uint8_t* fresh) {
  constexpr int R = DK / 16;  // state rows of a thread
  __shared__ float s_q[DK], s_k[DK];
  __shared__ float s_part[2][4][kDeltaCols];
  __shared__ float s_dot[3][4];
  pdl_enter();
  const int seq = blockIdx.z, h = blockIdx.y, c0 = blockIdx.x * kDeltaCols;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cq = (tid & 7) * 4, rg = tid >> 3;
  const int hk = h / a.rep;
  int t0 = seq, t1 = seq + 1;
  if (cu) {
    t0 = max(0, __ldg(cu + seq));
    t1 = min(T, __ldg(cu + seq + 1));
  }
  const int slot = delta_slot(a, seq);
  if (slot < 0) {
    for (int t = t0; t < t1; ++t)
      if (tid < kDeltaCols) a.out[t * a.out_stride + h * DV + c0 + tid] = __float2bfloat16_rn(0.f);
    return;
  }
  float* S = a.state + slot * a.slot_stride + static_cast<int64_t>(h) * DK * DV + c0 + cq;
  float s[R][4];
  const bool zero = fresh && fresh[seq];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float4 x = zero ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(S + (rg + 16 * r) * DV);
    s[r][0] = x.x; s[r][1] = x.y; s[r][2] = x.z; s[r][3] = x.w;
  }
  for (int t = t0; t < t1; ++t) {
    __syncthreads();
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
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
    *reinterpret_cast<float4*>(S + (rg + 16 * r) * DV) = make_float4(s[r][0], s[r][1], s[r][2], s[r][3]);
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

using DeltaKernel = void (*)(const DeltaArgs, const int32_t*, int, const uint8_t*);

DeltaKernel delta_kernel(int dk, int dv) {
  if (dk == 64) return dv == 64 ? gated_delta_kernel<64, 64> : gated_delta_kernel<64, 128>;
  return dv == 64 ? gated_delta_kernel<128, 64> : gated_delta_kernel<128, 128>;
}

}  // namespace
}  // namespace d3

using namespace d3;

extern "C" int d3_gated_delta_step(const d3_gated_delta_t* args, int n, int32_t* status, d3_stream_t stream) {
  DeltaArgs a{};
  if (int rc = delta_args(args, n, n, status, a)) return rc;
  if (n == 0) return D3_OK;
  launch_kernel(delta_kernel(args->key_dim, args->value_dim),
                dim3(args->value_dim / kDeltaCols, args->value_heads, n), dim3(kDeltaThreads), 0,
                reinterpret_cast<cudaStream_t>(stream), a, static_cast<const int32_t*>(nullptr), n,
                static_cast<const uint8_t*>(nullptr));
  return check_launch("d3_gated_delta_step");
}

extern "C" int d3_gated_delta_chunk_workspace_size(int T, int n, int value_heads, int key_dim, int value_dim,
                                                   size_t* bytes) {
  D3_REQUIRE(bytes != nullptr, "bytes is NULL");
  D3_REQUIRE(T >= 0 && n >= 0 && value_heads > 0, "negative size");
  D3_REQUIRE((key_dim == 64 || key_dim == 128) && (value_dim == 64 || value_dim == 128),
             "key_dim and value_dim must be 64 or 128");
  *bytes = 0;
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
  launch_kernel(delta_kernel(args->key_dim, args->value_dim),
                dim3(args->value_dim / kDeltaCols, args->value_heads, n), dim3(kDeltaThreads), 0,
                reinterpret_cast<cudaStream_t>(stream), a, cu, T, fresh);
  return check_launch("d3_gated_delta_chunk");
}
