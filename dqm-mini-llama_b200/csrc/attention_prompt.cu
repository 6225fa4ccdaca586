// attention_prompt.cu -- causal attention over packed prompts.
//
// Sequence s holds tokens starts[s] .. starts[s+1]-1 of the packed rows; token
// i of it, query head h, key/value head h / group:
//   s_ij = q_i . k_j / sqrt(D) for j <= i, softmax over j, out_i = sum p_ij v_j
#include <climits>

#include "common.cuh"
#include "internal.h"

namespace dqmk {
namespace {

__device__ unsigned int g_prompt_error;  // kErrTimeout / kErrBadIndex

constexpr int kMaxDim = 128;
constexpr float kLog2e = 1.44269504088896341f;

struct PromptArgs {
  const float *q, *k, *v;
  int64_t ldq, ldk, ldv;
  const int* starts;
  int n_seqs, n_tokens, n_heads, n_kv_heads, group, head_dim;
  float* out;
  int64_t ldo;
  float scale;  // log2(e) / sqrt(D)
};

constexpr int kThreads = 128, kRows = 16, kKeys = 32, kRowsPerWarp = kRows / 4;

// One CTA: 16 rows (token, head of the group) of one sequence and KV head.
__global__ void __launch_bounds__(kThreads) attention_prompt_kernel(const PromptArgs a) {
  __shared__ float ks[kKeys][kMaxDim + 1], vs[kKeys][kMaxDim];
  __shared__ float qs[kRows][kMaxDim];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = a.head_dim;
  const int kvh = blockIdx.y;
  // block x -> (sequence, first row)
  int seq = 0, t0 = 0, n = 0;
  int64_t blk = blockIdx.x;
  for (; seq < a.n_seqs; ++seq) {
    t0 = a.starts[seq];
    const int t1 = a.starts[seq + 1];
    if (t0 < 0 || t1 < t0 || t1 > a.n_tokens) {
      if (tid == 0) atomicOr(&g_prompt_error, kErrBadIndex);
      continue;
    }
    n = t1 - t0;
    const int64_t blocks = ((int64_t)n * a.group + kRows - 1) / kRows;
    if (blk < blocks) break;
    blk -= blocks;
  }
  if (seq == a.n_seqs) return;
  const int64_t f0 = blk * kRows, rows = (int64_t)n * a.group;
  for (int i = tid; i < kRows * D; i += kThreads) {
    const int r = i / D, d = i % D;
    const int64_t f = f0 + r;
    qs[r][d] = f < rows ? a.q[(t0 + f / a.group) * a.ldq + (kvh * a.group + f % a.group) * D + d] * a.scale : 0.0f;
  }
  float m[kRowsPerWarp], l[kRowsPerWarp], o[kRowsPerWarp][4];
  int token[kRowsPerWarp];
#pragma unroll
  for (int r = 0; r < kRowsPerWarp; ++r) {
    const int64_t f = f0 + warp * kRowsPerWarp + r;
    token[r] = f < rows ? (int)(f / a.group) : -1;
    m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[r][e] = 0.0f;
  }
  const int last = (int)(min(f0 + kRows, rows) - 1) / a.group;
  for (int k0 = 0; k0 <= last; k0 += kKeys) {
    __syncthreads();
    for (int i = tid; i < kKeys * D; i += kThreads) {
      const int j = i / D, d = i % D;
      const bool in = k0 + j < n;
      ks[j][d] = in ? a.k[(t0 + k0 + j) * a.ldk + kvh * D + d] : 0.0f;
      vs[j][d] = in ? a.v[(t0 + k0 + j) * a.ldv + kvh * D + d] : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; ++r) {
      const float* q = qs[warp * kRowsPerWarp + r];
      float s = 0.0f;
      for (int d = 0; d < D; ++d) s = fmaf(q[d], ks[lane][d], s);
      if (k0 + lane > token[r]) s = -INFINITY;
      const float mx = fmaxf(m[r], warp_max(s)), ref = mx == -INFINITY ? 0.0f : mx;
      const float corr = exp2f(m[r] - ref), p = exp2f(s - ref);
      l[r] = fmaf(l[r], corr, warp_sum(p));
      m[r] = mx;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[r][e] *= corr;
      for (int j = 0; j < kKeys && k0 + j <= token[r]; ++j) {
        const float pj = __shfl_sync(0xffffffffu, p, j);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (lane + 32 * e < D) o[r][e] = fmaf(pj, vs[j][lane + 32 * e], o[r][e]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kRowsPerWarp; ++r) {
    const int64_t f = f0 + warp * kRowsPerWarp + r;
    if (f >= rows) continue;
    float* y = a.out + (t0 + f / a.group) * a.ldo + (kvh * a.group + f % a.group) * D;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 32 * e < D) y[lane + 32 * e] = __fdiv_rn(o[r][e], l[r]);
  }
}

}  // namespace

cudaError_t read_prompt_error(unsigned int* flags, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(flags, g_prompt_error, sizeof(unsigned int));
  if (e == cudaSuccess && clear && *flags) {
    const unsigned int zero = 0;
    e = cudaMemcpyToSymbol(g_prompt_error, &zero, sizeof(unsigned int));
  }
  return e;
}

}  // namespace dqmk

// ------------------------------------------------------------------ C ABI
using namespace dqmk;

namespace {
bool prompt_shape_ok(int n_heads, int n_kv_heads, int head_dim) {
  return n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && head_dim > 0;
}
}  // namespace

extern "C" size_t dqmk_attention_prompt_workspace(int n_tokens, int n_seqs, int n_heads,
                                                  int n_kv_heads, int head_dim) {
  if (n_tokens <= 0 || n_seqs <= 0 || !prompt_shape_ok(n_heads, n_kv_heads, head_dim)) return 0;
  return 16;
}

extern "C" int dqmk_attention_prompt(const float* q, int64_t ldq, const float* k, int64_t ldk,
                                     const float* v, int64_t ldv, const int* starts, int n_seqs,
                                     int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                                     float* out, int64_t ldo, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const std::string api = "AttentionPrompt";
  if (n_tokens < 0 || n_seqs < 0) return fail(DQMK_ERR_INVALID, api + ": counts must not be negative");
  if (!prompt_shape_ok(n_heads, n_kv_heads, head_dim))
    return fail(DQMK_ERR_INVALID, api + ": invalid head configuration");
  if (head_dim % 4 != 0 || head_dim > kMaxDim)
    return fail(DQMK_ERR_UNSUPPORTED, api + ": head_dim must be a multiple of 4 of at most 128");
  const int64_t wq = (int64_t)n_heads * head_dim, wk = (int64_t)n_kv_heads * head_dim;
  if (ldq < wq || ldo < wq || ldk < wk || ldv < wk)
    return fail(DQMK_ERR_INVALID, api + ": row stride shorter than the row");
  if (n_tokens == 0 || n_seqs == 0) return DQMK_OK;
  if (!q || !k || !v || !starts || !out || !workspace)
    return fail(DQMK_ERR_INVALID, api + ": null pointer");
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
        reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out) |
        reinterpret_cast<uintptr_t>(workspace) | (uintptr_t)((ldq | ldk | ldv | ldo) * 4)) & 15u) != 0)
    return fail(DQMK_ERR_INVALID, api + ": rows and workspace must be 16-byte aligned");
  const size_t need = dqmk_attention_prompt_workspace(n_tokens, n_seqs, n_heads, n_kv_heads, head_dim);
  if (workspace_bytes < need)
    return fail(DQMK_ERR_INVALID, api + ": workspace of " + std::to_string(workspace_bytes) +
                                      " bytes, needs " + std::to_string(need));
  PromptArgs a = {};
  a.q = q, a.k = k, a.v = v, a.ldq = ldq, a.ldk = ldk, a.ldv = ldv;
  a.starts = starts, a.n_seqs = n_seqs, a.n_tokens = n_tokens;
  a.n_heads = n_heads, a.n_kv_heads = n_kv_heads, a.group = n_heads / n_kv_heads;
  a.head_dim = head_dim, a.out = out, a.ldo = ldo;
  a.scale = kLog2e / sqrtf((float)head_dim);
  // blocks of a sequence round up, so at most one more than their share each
  const int64_t blocks = ((int64_t)n_tokens * a.group) / kRows + n_seqs;
  if (blocks > INT_MAX || n_kv_heads > 65535) return fail(DQMK_ERR_UNSUPPORTED, api + ": too many rows");
  DQMK_CUDA_RET(api.c_str(), launch(attention_prompt_kernel, dim3((unsigned)blocks, n_kv_heads),
                                    dim3(kThreads), 0, static_cast<cudaStream_t>(stream), false, a));
  return DQMK_OK;
}
