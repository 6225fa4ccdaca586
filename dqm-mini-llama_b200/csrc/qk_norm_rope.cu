// qk_norm_rope.cu -- RMSNorm of every query and key head with the rotary
// rotation in the same pass, for many tokens at device-resident positions.
//
// For a head row x of D values with weight w:
//   n = x / sqrt(mean(x^2) + eps) * w                  (src/ops.cc:68-90)
//   pair i < D/2 (NeoX: elements i, i + D/2; else 2i, 2i + 1), angle
//   a_i = pos * theta^(-2i/D):  (n_a cos - n_b sin, n_a sin + n_b cos)
// dqmk_rope takes its angles from the reference's float expressions; here
// they are exact to a float: pos times the frequency in turns is formed and
// reduced to [-1/2, 1/2] turns in 64 bits, because a float product is off by
// up to 2^-24 of the angle, 0.06 rad at position 10^6.  The reduced angle is
// rounded once to float (at most 2^-25 half turns, 1e-7 rad).
//
// Every value is read once and written once, so the kernel is bound by
// memory: 8 bytes a value.  One CTA takes one token, so that the angles are
// computed once for all its heads, and its row loads are issued before the
// angles are computed.  A group of lanes holds a row in registers (4 pairs,
// two 16-byte loads a lane), so a row is reduced by shuffles and may be
// written in place.
#include "common.cuh"
#include "internal.h"

namespace dqmk {
namespace {

constexpr int kMaxHalf = 128;
constexpr int kMaxRows = 1 << 30;  // rows of a token are counted in 32 bits
constexpr int kThreads = 128;  // 84 us (92 by a call on new inputs) for 16384 tokens of 32 heads of 128, 88 with 256

struct NormRopeArgs {
  const float *q, *k;
  int64_t ldq, ldk;  // elements from one token's heads to the next token's
  float *q_out, *k_out;
  int64_t ldqo, ldko;
  int n_heads, n_kv_heads, head_dim;
  const float *q_norm, *k_norm;
  float eps;
  const int* positions;
  int neox;
  double turns[kMaxHalf];  // theta^(-2i/D) / (2 pi)
};

// 16 bytes that no other thread reads, past L1; not through the read-only path,
// for the row may be written in place.
__device__ __forceinline__ float4 load_once(const float* p) {
  float4 v;
  asm volatile("ld.global.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "l"(p));
  return v;
}

// V pairs a lane at a time (4: 16-byte accesses, 1: any alignment), LANES
// lanes a row, J steps of V * LANES pairs.
template <int V, int LANES, int J>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const __grid_constant__ NormRopeArgs a) {
  constexpr int kGroups = kThreads / LANES;
  __shared__ float2 cs[kMaxHalf];
  const int tid = threadIdx.x, lane = tid % LANES, group = tid / LANES;
  const int half = a.head_dim >> 1, rows = a.n_heads + a.n_kv_heads;
  const int64_t token = blockIdx.x;
  // element offsets of this lane's pairs within a row
  const int step_a = a.neox ? 1 : 2, off_b = a.neox ? half : 1;

  float xa[J][V], xb[J][V];
  auto load = [&](int r) {
    const float* x = r < a.n_heads ? a.q + token * a.ldq + (int64_t)r * a.head_dim
                                   : a.k + token * a.ldk + (int64_t)(r - a.n_heads) * a.head_dim;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int p = (j * LANES + lane) * V;  // first pair
      const bool in = r < rows && p < half;
      if constexpr (V == 4) {
        const float* pa = x + (int64_t)p * step_a;
        const float* pb = a.neox ? pa + half : pa + 4;
        const float4 u = in ? load_once(pa) : make_float4(0, 0, 0, 0);
        const float4 v = in ? load_once(pb) : make_float4(0, 0, 0, 0);
        if (a.neox) {
          xa[j][0] = u.x, xa[j][1] = u.y, xa[j][2] = u.z, xa[j][3] = u.w;
          xb[j][0] = v.x, xb[j][1] = v.y, xb[j][2] = v.z, xb[j][3] = v.w;
        } else {
          xa[j][0] = u.x, xb[j][0] = u.y, xa[j][1] = u.z, xb[j][1] = u.w;
          xa[j][2] = v.x, xb[j][2] = v.y, xa[j][3] = v.z, xb[j][3] = v.w;
        }
      } else {
        xa[j][0] = in ? x[p * step_a] : 0.0f;
        xb[j][0] = in ? x[p * step_a + off_b] : 0.0f;
      }
    }
  };

  load(group);
  if (tid < half) {
    double t = (double)a.positions[token] * a.turns[tid];
    t -= rint(t);
    float s, c;
    sincospif((float)(2.0 * t), &s, &c);
    cs[tid] = make_float2(c, s);
  }
  __syncthreads();
  // rows of a warp's groups differ, the trip count does not: every lane
  // reaches the shuffles
  for (int r0 = 0; r0 < rows; r0 += kGroups) {
    const int r = r0 + group;
    if (r0) load(r);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) sum = fmaf(xa[j][i], xa[j][i], fmaf(xb[j][i], xb[j][i], sum));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (r >= rows) continue;
    const float inv = __fdiv_rn(1.0f, sqrtf(__fdiv_rn(sum, (float)a.head_dim) + a.eps));
    const bool is_q = r < a.n_heads;
    const float* w = is_q ? a.q_norm : a.k_norm;
    float* y = is_q ? a.q_out + token * a.ldqo + (int64_t)r * a.head_dim
                    : a.k_out + token * a.ldko + (int64_t)(r - a.n_heads) * a.head_dim;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int p = (j * LANES + lane) * V;
      if (p >= half) continue;
      float ya[V], yb[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int ea = (p + i) * step_a, eb = ea + off_b;
        const float na = xa[j][i] * inv * __ldg(w + ea), nb = xb[j][i] * inv * __ldg(w + eb);
        const float2 t = cs[p + i];
        ya[i] = na * t.x - nb * t.y;
        yb[i] = na * t.y + nb * t.x;
      }
      if constexpr (V == 4) {
        float4* pa = reinterpret_cast<float4*>(y + (int64_t)p * step_a);
        if (a.neox) {
          *pa = make_float4(ya[0], ya[1], ya[2], ya[3]);
          *reinterpret_cast<float4*>(y + p + half) = make_float4(yb[0], yb[1], yb[2], yb[3]);
        } else {
          pa[0] = make_float4(ya[0], yb[0], ya[1], yb[1]);
          pa[1] = make_float4(ya[2], yb[2], ya[3], yb[3]);
        }
      } else {
        y[p * step_a] = ya[0];
        y[p * step_a + off_b] = yb[0];
      }
    }
  }
}

}  // namespace
}  // namespace dqmk

// ------------------------------------------------------------------ C ABI
using namespace dqmk;

extern "C" int dqmk_qk_norm_rope(const float* q, int64_t ldq, const float* k, int64_t ldk,
                                 int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                                 const float* q_norm, const float* k_norm, float eps,
                                 const int* positions, float theta, int neox, float* q_out,
                                 int64_t ldq_out, float* k_out, int64_t ldk_out, void* stream) {
  const std::string api = "QkNormRope";
  if (n_tokens < 0 || n_heads < 0 || n_kv_heads < 0)
    return fail(DQMK_ERR_INVALID, api + ": counts must not be negative");
  if ((int64_t)n_heads + n_kv_heads > kMaxRows) return fail(DQMK_ERR_UNSUPPORTED, api + ": too many heads");
  if (head_dim <= 0 || head_dim % 2 != 0)
    return fail(DQMK_ERR_INVALID, api + ": head_dim must be positive and even");
  if (head_dim / 2 > kMaxHalf) return fail(DQMK_ERR_UNSUPPORTED, api + ": head_dim larger than 256");
  if (!(theta > 0.0f) || theta > 3.4e38f)
    return fail(DQMK_ERR_INVALID, api + ": theta must be finite and positive");
  if (!(eps >= 0.0f) || eps > 3.4e38f)
    return fail(DQMK_ERR_INVALID, api + ": eps must be finite and not negative");
  const int64_t wq = (int64_t)n_heads * head_dim, wk = (int64_t)n_kv_heads * head_dim;
  if (ldq < wq || ldq_out < wq || ldk < wk || ldk_out < wk)
    return fail(DQMK_ERR_INVALID, api + ": row stride shorter than the row");
  if (n_tokens == 0 || n_heads + n_kv_heads == 0) return DQMK_OK;
  if (!positions || (n_heads && (!q || !q_norm || !q_out)) ||
      (n_kv_heads && (!k || !k_norm || !k_out)))
    return fail(DQMK_ERR_INVALID, api + ": null pointer");
  NormRopeArgs a = {};
  a.q = q, a.k = k, a.ldq = ldq, a.ldk = ldk;
  a.q_out = q_out, a.k_out = k_out, a.ldqo = ldq_out, a.ldko = ldk_out;
  a.n_heads = n_heads, a.n_kv_heads = n_kv_heads, a.head_dim = head_dim;
  a.q_norm = q_norm, a.k_norm = k_norm, a.eps = eps;
  a.positions = positions, a.neox = neox != 0;
  const double step = -2.0 * log2((double)theta) / head_dim;
  for (int i = 0; i < head_dim / 2; ++i) a.turns[i] = exp2(step * i) * 0.15915494309189533577;
  uintptr_t bits = 0;
  if (n_heads) bits |= reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) | (uintptr_t)((ldq | ldq_out) * 4);
  if (n_kv_heads) bits |= reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out) | (uintptr_t)((ldk | ldk_out) * 4);
  const bool vec = head_dim % 8 == 0 && (bits & 15u) == 0;
  const int chunks = (head_dim / 2 + 3) / 4;  // 4-pair chunks a row
  const dim3 grid(n_tokens), block(kThreads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (!vec)
    e = launch(qk_norm_rope_kernel<1, 32, 4>, grid, block, 0, st, false, a);
  else if (chunks <= 8)
    e = launch(qk_norm_rope_kernel<4, 8, 1>, grid, block, 0, st, false, a);
  else if (chunks <= 16)
    e = launch(qk_norm_rope_kernel<4, 16, 1>, grid, block, 0, st, false, a);
  else
    e = launch(qk_norm_rope_kernel<4, 32, 1>, grid, block, 0, st, false, a);
  DQMK_CUDA_RET(api.c_str(), e);
  return DQMK_OK;
}
