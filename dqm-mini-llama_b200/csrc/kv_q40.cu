// kv_q40.cu -- a KV cache held in 4 bits: write, read back, attention.
//
// Rows are quantized to Q4_0 blocks exactly as dqmk_quantize_q40 does (a
// block of 32 values: fp16 scale d = absmax / 7, codes n = round(v / d + 8) in
// 0..15, value d (n - 8)).  Each of the two buffers (keys, values) holds, for
// every layer, slot and KV head, the rows of its positions one after the
// other, first all quants, then all scales:
//
//   quants [layer][slot][kv_head][rows][D/2 bytes]
//   scales [layer][slot][kv_head][rows][D/32 fp16]     rows = max_seq up to 32
//
// so the positions that a query reads are one contiguous run a head.  Inside a
// row the bytes of the blocks (byte j: value j low, value j + 16 high) are
// interleaved so that one thread's share of a matrix operand is contiguous:
//   keys    4-byte words [t][block], word t = bytes 4t .. 4t+3 of the block
//   values  2-byte units [g][block], unit g = bytes 2g, 2g+1 of the block
#include <climits>

#include "common.cuh"
#include "internal.h"
#include "tc_dev.cuh"

namespace dqmk {
namespace {

__device__ unsigned int g_kv_error;  // kErrTimeout / kErrBadIndex

constexpr int kMaxBlocks = 4;  // 32-value blocks of a row: head_dim at most 128

__host__ __device__ __forceinline__ int64_t padded_rows(int max_seq) {
  return ((int64_t)max_seq + 31) / 32 * 32;
}

// One layer of the cache.
struct Plane {
  uint8_t* kq;
  uint16_t* kd;
  uint8_t* vq;
  uint16_t* vd;
  int n_slots, max_seq, n_kv_heads, nb;
  int64_t rows;  // padded rows of one head
};

__device__ __forceinline__ int64_t plane_row(const Plane& c, int slot, int head, int pos) {
  return ((int64_t)slot * c.n_kv_heads + head) * c.rows + pos;
}

// --------------------------------------------------------- write and read
struct RowsArgs {
  Plane c;
  const float *k, *v;  // write: sources
  float *ko, *vo;      // read: destinations
  int64_t ldk, ldv;    // elements from one token's heads to the next token's
  const int *slots, *positions;
  int n_tokens;
};

// The cache row a token names, or -1: a padding token (position -1), or a slot
// or position outside the cache, which is recorded.
__device__ __forceinline__ int64_t token_row(const RowsArgs& a, int token, int head) {
  const int pos = a.positions[token], slot = a.slots ? a.slots[token] : token;
  if (pos == -1) return -1;
  if (pos < 0 || pos >= a.c.max_seq || slot < 0 || slot >= a.c.n_slots) {
    atomicOr(&g_kv_error, kErrBadIndex);
    return -1;
  }
  return plane_row(a.c, slot, head, pos);
}

// 8 lanes take one block, 4 values each.  VEC: 16-byte accesses to the f32
// rows.
template <bool VEC>
__global__ void __launch_bounds__(256) kv_q40_write_kernel(RowsArgs a) {
  const int nb = a.c.nb, lane = threadIdx.x & 31, i8 = lane & 7;
  const int64_t per_token = (int64_t)2 * a.c.n_kv_heads * nb;  // blocks of K, then of V
  const int64_t total = per_token * a.n_tokens;
  const int64_t stride = (int64_t)gridDim.x * (blockDim.x / 8);
  int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 8;
  // whole warps stay in the loop: the shuffles name every lane
  for (; item - (lane >> 3) < total; item += stride) {
    const bool live = item < total;
    const int token = live ? (int)(item / per_token) : 0;
    int r = live ? (int)(item % per_token) : 0;
    const bool is_v = r >= a.c.n_kv_heads * nb;
    if (is_v) r -= a.c.n_kv_heads * nb;
    const int head = r / nb, b = r % nb;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
      const float* src = (is_v ? a.v + token * a.ldv : a.k + token * a.ldk) +
                         ((int64_t)head * nb + b) * 32 + 4 * i8;
      if constexpr (VEC) {
        const float4 f = ldg_f4_stream(src);
        x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = src[e];
      }
    }
    float top = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    uint16_t d = 0;
    uint32_t codes = 0;  // byte e: the code of value 4 i8 + e
    if (top > 0.0f) {
      d = f2h_ref(__fdiv_rn(top, 7.0f));
      const float stored = h2f(d);
      const float inv = stored == 0.0f ? 0.0f : __fdiv_rn(1.0f, stored);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        int q = (int)roundf(__fadd_rn(__fmul_rn(x[e], inv), 8.0f));
        q = q < 0 ? 0 : (q > 15 ? 15 : q);
        codes |= (uint32_t)q << (8 * e);
      }
    }
    // lanes 0-3 hold values 0..15 of the block, lanes 4-7 values 16..31
    const uint32_t high = __shfl_down_sync(0xffffffffu, codes, 4, 8);
    const int64_t row = live ? token_row(a, token, head) : -1;
    if (row < 0) continue;
    const uint32_t word = codes | high << 4;
    if (i8 < 4) {
      if (is_v) {
        uint16_t* u = reinterpret_cast<uint16_t*>(a.c.vq + row * (16 * nb));
        u[2 * i8 * nb + b] = (uint16_t)word;
        u[(2 * i8 + 1) * nb + b] = (uint16_t)(word >> 16);
      } else {
        reinterpret_cast<uint32_t*>(a.c.kq + row * (16 * nb))[i8 * nb + b] = word;
      }
    }
    if (i8 == 0) (is_v ? a.c.vd : a.c.kd)[row * nb + b] = d;
  }
}

template <bool VEC>
__global__ void __launch_bounds__(256) kv_q40_read_kernel(RowsArgs a) {
  const int nb = a.c.nb;
  const int64_t per_token = (int64_t)2 * a.c.n_kv_heads * nb;
  const int64_t total = per_token * a.n_tokens * 8;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int i8 = (int)(i & 7);
    const int64_t item = i >> 3;
    const int token = (int)(item / per_token);
    int r = (int)(item % per_token);
    const bool is_v = r >= a.c.n_kv_heads * nb;
    if (is_v) r -= a.c.n_kv_heads * nb;
    const int head = r / nb, b = r % nb, t = i8 & 3;
    const int64_t row = token_row(a, token, head);
    if (row < 0) continue;
    uint32_t word;
    if (is_v) {
      const uint16_t* u = reinterpret_cast<const uint16_t*>(a.c.vq + row * (16 * nb));
      word = u[2 * t * nb + b] | (uint32_t)u[(2 * t + 1) * nb + b] << 16;
    } else {
      word = reinterpret_cast<const uint32_t*>(a.c.kq + row * (16 * nb))[t * nb + b];
    }
    if (i8 >= 4) word >>= 4;
    const float d = h2f((is_v ? a.c.vd : a.c.kd)[row * nb + b]);
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __fmul_rn(d, (float)(int)((word >> (8 * e)) & 15u) - 8.0f);
    float* dst = (is_v ? a.vo + token * a.ldv : a.ko + token * a.ldk) +
                 ((int64_t)head * nb + b) * 32 + 4 * i8;
    if constexpr (VEC) {
      *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[e] = y[e];
    }
  }
}

// -------------------------------------------------------------- attention
// One column is one query token: q [n_heads][D] against the first `length`
// positions of its slot.  A group of up to 8 query heads that share a KV head
// is one unit of the tensor-core products (mma.sync m16n8k16, fp16 operands,
// fp32 sums); groups of more than 8 heads run as several.
//
// With f32 queries and weights the products have to keep f32 precision.  A
// code is exact in fp16, so only the other operand is split into two fp16
// terms (22 bits), and the two terms are stacked in the 16 rows of the A
// operand (rows 0-7: high terms of 8 heads, rows 8-15: low terms), so that one
// product does both:
//   scores   A = q 2^-e, B = codes n - 8 (rows of K), one sum for each block:
//            S = 2^e / sqrt(D) sum_b d_b sum q (n - 8)
//   output   A = w = p d_b 2^(15-E), B = codes n - 8 (columns of V):
//            O[c] = 2^(E-15) sum_j w_j (n_jc - 8), a block's channels at a time
// E is a running bound of the exponents of V's scales, kept like the running
// maximum of the scores: when it grows, the sums are scaled down.
//
// A code becomes a half by one AND/OR, (w & 0x000f) | 0x6400 = 1024 + n, and
// one addition that centres it: n - 8 (16 (n - 8) from a high nibble; its
// channel of q takes 1/16).  The code's own bits are n 2^-24 as a subnormal
// half and would need neither, but the products align their sums by the
// operands' exponent fields, and 10 bits of every sum are lost (measured: 2e-6
// of the output against 3e-7).
//
// Bound: 18 bytes for 32 values, each used by every head of the group; at the
// memory rate an SM has about 1.4 instruction slots a value, and the unpacking,
// scaling and splitting above take most of them.
//
// Work: the positions of all columns and heads form one list of chunks of
// kChunk positions, cut into equal runs for the CTAs, whatever the lengths; a
// CTA that holds only part of a (column, group)'s chunks leaves its partial
// sums in the workspace for a second kernel.  Each warp streams its own tiles
// of 32 positions through a ring of bulk copies.
constexpr int kWarps = 4, kThreads = 32 * kWarps, kTile = 32, kChunk = kTile * kWarps;
constexpr int kStages = 3, kGroup = 8;
constexpr float kLog2e = 1.44269504088896341f;

struct AttnQ40Args {
  Plane c;
  const float* q;
  int64_t ldq;
  float* out;
  int64_t ldo;
  const int *lengths, *slots;
  int n_cols, n_heads, group, subs;  // subs: (KV head, 8-head group) pairs of a column
  float scale;                       // log2(e) / sqrt(D)
  float* part;                       // [CTA][2][part_floats]
  int n_ctas;                        // CTAs of the first kernel
};

template <int NB>
struct Shape {
  static constexpr int kD = 32 * NB;
  static constexpr int kQuantBytes = kTile * 16 * NB, kScaleBytes = kTile * 2 * NB;
  static constexpr int kStageBytes = 2 * (kQuantBytes + kScaleBytes);
  static constexpr int kPartFloats = kGroup * (kD + 2);
};

// Visible positions of a column: 0 for a length or slot outside the cache.
__device__ __forceinline__ int visible(const AttnQ40Args& a, int col) {
  const int n = a.lengths[col];
  const int s = a.slots ? a.slots[col] : col;
  return n > 0 && n <= a.c.max_seq && s >= 0 && s < a.c.n_slots ? n : 0;
}
__device__ __forceinline__ int64_t units_of(const AttnQ40Args& a, int len) {
  return (int64_t)((len + kChunk - 1) / kChunk) * a.subs;
}
// The CTA whose run of the `total` units holds unit u: run i is
// [i total / n, (i + 1) total / n).
__device__ __forceinline__ int cta_of(int64_t u, int64_t total, int n) {
  return (int)(((u + 1) * n - 1) / total);
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          tc::su32(dst)),
      "l"(src), "r"(bytes), "r"(tc::su32(bar))
      : "memory");
}
// Two values to packed fp16 pairs with x = hi + lo + r, |r| <= 2^-22 |x|.
__device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x0, x1);
  const float2 back = __half22float2(h);
  const __half2 l = __floats2half2_rn(__fsub_rn(x0, back.x), __fsub_rn(x1, back.y));
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
// The codes in bits 0-3 and 16-19 of a word as the halves n - 8, and those in
// bits 4-7 and 20-23 as 16 (n - 8).
__device__ __forceinline__ uint32_t add_h2(uint32_t x, uint32_t y) {
  const __half2 z = __hadd2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
  return *reinterpret_cast<const uint32_t*>(&z);
}
__device__ __forceinline__ uint32_t codes_low(uint32_t w) {
  return add_h2((w & 0x000f000fu) | 0x64006400u, 0xe408e408u);  // -1032
}
__device__ __forceinline__ uint32_t codes_high(uint32_t w) {
  return add_h2((w & 0x00f000f0u) | 0x64006400u, 0xe480e480u);  // -1152
}
__device__ __forceinline__ float pow2f(int e) { return __int_as_float((127 + e) << 23); }

template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&r)[N], const void* p) {
  if constexpr (N == 4) {
    const uint4 v = *static_cast<const uint4*>(p);
    r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *static_cast<const uint2*>(p);
    r[0] = v.x, r[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = static_cast<const uint32_t*>(p)[i];
  }
}
__device__ __forceinline__ float half_at(uint32_t w, int i) {
  return h2f((uint16_t)(i ? w >> 16 : w));
}

template <int NB>
__global__ void __launch_bounds__(kThreads, 3) kv_q40_attention_kernel(const AttnQ40Args a) {
  using S = Shape<NB>;
  constexpr int D = S::kD;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[kWarps][kStages];
  __shared__ uint4 qfrag[NB][2][32];
  __shared__ float qscale[kGroup];
  __shared__ float red_m[kWarps][kGroup], red_l[kWarps][kGroup];
  __shared__ int red_e[kWarps];
  __shared__ int64_t warp_sums[kWarps];
  __shared__ int64_t s_first;
  __shared__ int s_col;
  __shared__ volatile int abort_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;

  if (tid < kWarps * kStages) tc::bar_init(&bars[tid / kStages][tid % kStages], 1);
  if (tid == 0) {
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }

  // ---- this CTA's run of the chunk list
  int64_t total = 0;
  for (int c0 = 0; c0 < a.n_cols; c0 += kThreads) {
    const int col = c0 + tid;
    int64_t before;
    const int len = col < a.n_cols ? visible(a, col) : 0;
    total += block_scan(units_of(a, len), &before, warp_sums);
    // columns that see nothing: their rows are zero, shared out over the CTAs
    if (col < a.n_cols && blockIdx.x == 0) {
      const int n = a.lengths[col], s = a.slots ? a.slots[col] : col;
      if (n < 0 || n > a.c.max_seq || s < 0 || s >= a.c.n_slots) atomicOr(&g_kv_error, kErrBadIndex);
    }
  }
  for (int col = blockIdx.x; col < a.n_cols; col += gridDim.x)
    if (visible(a, col) == 0)
      for (int i = tid; i < a.n_heads * D; i += kThreads) a.out[col * a.ldo + i] = 0.0f;
  const int n_ctas = (int)min((int64_t)gridDim.x, total);
  if ((int)blockIdx.x >= n_ctas) {
    pdl_trigger();
    return;
  }
  const int64_t u0 = blockIdx.x * total / n_ctas, u1 = (blockIdx.x + 1) * total / n_ctas;
  {
    int64_t run = 0;
    for (int c0 = 0; c0 < a.n_cols; c0 += kThreads) {
      const int col = c0 + tid;
      int64_t before;
      const int64_t x = col < a.n_cols ? units_of(a, visible(a, col)) : 0;
      const int64_t sum = block_scan(x, &before, warp_sums);
      before += run;
      if (before <= u0 && u0 < before + x) {
        s_col = col;
        s_first = before;
      }
      run += sum;
      if (run > u0) break;
    }
  }
  __syncthreads();
  int col = s_col;
  int64_t first = s_first;  // unit 0 of the column

  unsigned char* ring = smem + (size_t)warp * kStages * S::kStageBytes;
  uint32_t used = 0;  // tiles this warp has waited for: stage used % kStages
  uint32_t issued = 0;
  bool ok = true;

  for (int64_t u = u0; u < u1 && ok;) {
    const int len = visible(a, col);
    const int chunks = (len + kChunk - 1) / kChunk;
    const int64_t rel = u - first;
    if (rel >= (int64_t)chunks * a.subs) {  // past this column (or it is empty)
      first += (int64_t)chunks * a.subs;
      ++col;
      continue;
    }
    const int sub = (int)(rel / chunks), ch0 = (int)(rel % chunks);
    const int take = (int)min((int64_t)(chunks - ch0), u1 - u);
    const int kvh = sub % a.c.n_kv_heads, h0 = (sub / a.c.n_kv_heads) * kGroup;
    const int n_here = min(kGroup, a.group - h0);  // heads of this group
    const int slot = a.slots ? a.slots[col] : col;
    const int64_t row0 = plane_row(a.c, slot, kvh, 0);
    const int tile_end = min((ch0 + take) * kWarps, (len + kTile - 1) / kTile);
    const int tile0 = ch0 * kWarps + warp;
    const int mine = tile0 < tile_end ? (tile_end - tile0 + kWarps - 1) / kWarps : 0;

    auto issue = [&](int i) {  // lane 0: this warp's tile i of the piece
      unsigned char* st = ring + (issued % kStages) * S::kStageBytes;
      uint64_t* bar = &bars[warp][issued % kStages];
      const int64_t row = row0 + (int64_t)(tile0 + i * kWarps) * kTile;
      tc::bar_expect_tx(bar, S::kStageBytes);
      bulk_load(st, a.c.kq + row * (16 * NB), S::kQuantBytes, bar);
      bulk_load(st + S::kQuantBytes, a.c.vq + row * (16 * NB), S::kQuantBytes, bar);
      bulk_load(st + 2 * S::kQuantBytes, a.c.kd + row * NB, S::kScaleBytes, bar);
      bulk_load(st + 2 * S::kQuantBytes + S::kScaleBytes, a.c.vd + row * NB, S::kScaleBytes, bar);
    };
    for (int i = 0; i < min(mine, kStages); ++i) {
      if (lane == 0) issue(i);
      ++issued;
    }

    // ---- the group's queries as A operands (high and low terms)
    for (int hh = warp * 2; hh < warp * 2 + 2; ++hh) {
      float x[NB], top = 0.0f;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int64_t head = (int64_t)kvh * a.group + h0 + hh;
        x[b] = hh < n_here ? a.q[col * a.ldq + head * D + 32 * b + lane] : 0.0f;
        top = fmaxf(top, fabsf(x[b]));
      }
      top = warp_max(top);
      // 2^-e brings the row's largest value into [2^14, 2^15)
      const int e = top > 0.0f ? min(max(((__float_as_int(top) >> 23) & 0xff) - 141, -120), 120) : 0;
      const bool high = lane >= 16;
      const int jj = lane & 15, tq = jj >> 2, el = jj & 3;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        // a high nibble stands for 16 (n - 8): its channel takes 1/16
        const float v = x[b] * pow2f(-e) * (high ? 0.0625f : 1.0f);
        const __half hi = __float2half_rn(v);
        const __half lo = __float2half_rn(v - __half2float(hi));
        __half* dst = reinterpret_cast<__half*>(&qfrag[b][el & 1][hh * 4 + tq]) + (high ? 4 : 0) + (el >> 1);
        dst[0] = hi;
        dst[2] = lo;
      }
      if (lane == 0) qscale[hh] = pow2f(e) * a.scale;
    }
    __syncthreads();

    float o[NB][4][4];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[b][s][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    int ev = -20;  // V's scales so far are below 2^ev
    const float qs = qscale[g];

    for (int i = 0; i < mine; ++i) {
      const uint32_t stage = used % kStages;
      const bool landed = tc::bar_wait(&bars[warp][stage], (used / kStages) & 1, &abort_flag, &g_kv_error);
      ok = __all_sync(0xffffffffu, landed);
      if (!ok) break;
      ++used;
      unsigned char* st = ring + stage * S::kStageBytes;
      const unsigned char* kq = st;
      const unsigned char* vq = st + S::kQuantBytes;
      uint16_t* kd = reinterpret_cast<uint16_t*>(st + 2 * S::kQuantBytes);
      uint16_t* vd = kd + kTile * NB;
      const int left = len - (tile0 + i * kWarps) * kTile;  // live positions of the tile
      if (left < kTile) {
        // rows past the end may hold anything: zero scales take them out
        if (lane >= left) {
#pragma unroll
          for (int b = 0; b < NB; ++b) kd[lane * NB + b] = vd[lane * NB + b] = 0;
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
      }

      // ---- scores of keys 8 j + 2 t + {0, 1} for head g
      float s[4][2];
      {
        uint32_t kw[4][NB], dk[4][NB];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lds_words<NB>(kw[j], kq + (8 * j + g) * (16 * NB) + t * (4 * NB));
          lds_words<NB>(dk[j], kd + (8 * j + 2 * t) * NB);
          s[j][0] = s[j][1] = 0.0f;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint4 a0 = qfrag[b][0][lane], a1 = qfrag[b][1][lane];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t w = kw[j][b], w8 = w >> 8;
            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma16816(c, a0, codes_low(w), codes_high(w));
            mma16816(c, a1, codes_low(w8), codes_high(w8));
            // scales of keys 2t (halves 0 .. NB-1) and 2t + 1 (NB .. 2 NB - 1)
            s[j][0] = fmaf(half_at(dk[j][b >> 1], b & 1), c[0] + c[2], s[j][0]);
            s[j][1] = fmaf(half_at(dk[j][(NB + b) >> 1], (NB + b) & 1), c[1] + c[3], s[j][1]);
          }
        }
      }
      float mx = m;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[j][e] *= qs;
          if (left < kTile && 8 * j + 2 * t + e >= left) s[j][e] = -INFINITY;
          mx = fmaxf(mx, s[j][e]);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mref = mx == -INFINITY ? 0.0f : mx;
      uint32_t dv[4][NB], dtop = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        lds_words<NB>(dv[j], vd + (8 * j + 2 * t) * NB);
#pragma unroll
        for (int b = 0; b < NB; ++b) dtop = __vmaxu2(dtop, dv[j][b]);
      }
      dtop = max(dtop >> 16, dtop & 0xffffu);
      dtop = max(dtop, __shfl_xor_sync(0xffffffffu, dtop, 1));
      dtop = max(dtop, __shfl_xor_sync(0xffffffffu, dtop, 2));
      const int enew = max(ev, (int)(dtop >> 10) - 14);
      const float corr = exp2f(m - mref);
      float psum = 0.0f;
      const float up = pow2f(15 - enew);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[j][e] = exp2f(s[j][e] - mref);
          psum += s[j][e];
          s[j][e] *= up;
        }
      l = fmaf(l, corr, psum);
      m = mx;
      const float down = corr * pow2f(ev - enew);
      ev = enew;
      if (__any_sync(0xffffffffu, down != 1.0f)) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[b][c][r] *= down;
      }

      // ---- output: 16 keys at a time
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        constexpr int W = (NB + 1) / 2;
        uint32_t vw[4][W];  // keys 16 h + {2t, 2t+1, 2t+8, 2t+9}, unit g of every block
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const unsigned char* p = vq + (16 * h + 2 * t + (k & 1) + (k >> 1) * 8) * (16 * NB) + g * (2 * NB);
          if constexpr (NB % 2 == 0) {
            lds_words<W>(vw[k], p);
          } else {
            const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int w = 0; w < W; ++w)
              vw[k][w] = u[2 * w] | (2 * w + 1 < NB ? (uint32_t)u[2 * w + 1] << 16 : 0u);
          }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          uint4 w4;
          {
            const int j0 = 2 * h, j1 = 2 * h + 1;
            split2(s[j0][0] * half_at(dv[j0][b >> 1], b & 1),
                   s[j0][1] * half_at(dv[j0][(NB + b) >> 1], (NB + b) & 1), w4.x, w4.y);
            split2(s[j1][0] * half_at(dv[j1][b >> 1], b & 1),
                   s[j1][1] * half_at(dv[j1][(NB + b) >> 1], (NB + b) & 1), w4.z, w4.w);
          }
#pragma unroll
          for (int byte = 0; byte < 2; ++byte) {
            const uint32_t i0 = (b & 1) * 2 + byte;
            const uint32_t sel = i0 | i0 << 4 | (i0 + 4) << 8 | (i0 + 4) << 12;
            const uint32_t x0 = __byte_perm(vw[0][b >> 1], vw[1][b >> 1], sel);
            const uint32_t x1 = __byte_perm(vw[2][b >> 1], vw[3][b >> 1], sel);
            // channels 2g + byte (low nibbles) and 2g + byte + 16 (high)
            mma16816(o[b][byte], w4, codes_low(x0), codes_low(x1));
            mma16816(o[b][2 + byte], w4, codes_high(x0), codes_high(x1));
          }
        }
      }
      __syncwarp();
      if (i + kStages < mine) {
        if (lane == 0) issue(i + kStages);
        ++issued;
      }
    }
    ok = __syncthreads_and(ok);
    if (!ok) break;

    // ---- join the warps' sums, in warp order
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) {
      red_m[warp][g] = m;
      red_l[warp][g] = l;
    }
    if (lane == 0) red_e[warp] = ev;
    const int warps_used = min(kWarps, tile_end - ch0 * kWarps);
    if (mine) {
      float* ro = reinterpret_cast<float*>(ring);  // [head][channel], this warp's ring is empty
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // column 2t + e of the products: channels 2 (2t + e) + byte, + 16
          float2* lo = reinterpret_cast<float2*>(ro + g * D + 32 * b + 4 * t + 2 * e);
          lo[0] = make_float2(o[b][0][e] + o[b][0][e + 2], o[b][1][e] + o[b][1][e + 2]);
          lo[8] = make_float2((o[b][2][e] + o[b][2][e + 2]) * 0.0625f,
                              (o[b][3][e] + o[b][3][e + 2]) * 0.0625f);
        }
    }
    __syncthreads();
    const bool whole = take == chunks;
    float* part = a.part + ((int64_t)blockIdx.x * 2 + (ch0 == 0 ? 1 : 0)) * S::kPartFloats;
    for (int i = tid; i < n_here * D; i += kThreads) {
      const int h = i / D;
      float mm = -INFINITY, ll = 0.0f, acc = 0.0f;
      for (int w = 0; w < warps_used; ++w) mm = fmaxf(mm, red_m[w][h]);
      const float ref = mm == -INFINITY ? 0.0f : mm;
      for (int w = 0; w < warps_used; ++w) {
        const float f = exp2f(red_m[w][h] - ref);
        ll = fmaf(red_l[w][h], f, ll);
        const float x = reinterpret_cast<const float*>(smem + (size_t)w * kStages * S::kStageBytes)[i];
        acc = fmaf(x * pow2f(red_e[w] - 15), f, acc);
      }
      if (whole) {
        a.out[col * a.ldo + ((int64_t)kvh * a.group + h0) * D + i] = __fdiv_rn(acc, ll);
      } else {
        part[i] = acc;
        if (i % D == 0) {
          part[kGroup * D + h] = mm;
          part[kGroup * D + kGroup + h] = ll;
        }
      }
    }
    tc::fence_proxy_async_smem();  // the next piece's copies overwrite the sums
    __syncthreads();
    u += take;
  }
  if (!ok) {  // a wait ran out: leave once this warp's own copies have landed or given up
    for (; used < issued; ++used) {
      const unsigned long long t0 = tc::now_ns();
      while (!tc::bar_try(&bars[warp][used % kStages], (used / kStages) & 1))
        if (tc::now_ns() - t0 > tc::kWaitNs) break;
    }
  }
  pdl_trigger();
}

// Joins the partial sums of a (column, group) whose chunks lie in more than
// one CTA's run, in CTA order: one CTA for one head, D / 4 lanes for a
// partial sum.
constexpr int kJoinThreads = 256;
template <int NB>
__global__ void __launch_bounds__(kJoinThreads) kv_q40_join_kernel(const AttnQ40Args a) {
  using S = Shape<NB>;
  constexpr int D = S::kD, kLanes = D / 4, kSlots = kJoinThreads / kLanes;
  __shared__ int64_t warp_sums[kJoinThreads / 32];
  __shared__ float4 acc_s[kSlots][kLanes];
  __shared__ float l_s[kSlots], m_s[kJoinThreads / 32];
  const int tid = threadIdx.x, col = blockIdx.x / a.subs, sub = blockIdx.x % a.subs, h = blockIdx.y;
  const int kvh = sub % a.c.n_kv_heads, h0 = (sub / a.c.n_kv_heads) * kGroup;
  int64_t total = 0, first = 0, before;
  for (int c0 = 0; c0 < a.n_cols; c0 += kJoinThreads) {
    const int c = c0 + tid;
    const int64_t x = c < a.n_cols ? units_of(a, visible(a, c)) : 0;
    total += block_scan(x, &before, warp_sums);
    if (c0 < col) first += block_scan(c < col ? x : 0, &before, warp_sums);
  }
  const int len = visible(a, col), chunks = (len + kChunk - 1) / kChunk;
  // every CTA waits, so that this grid's end is also the first kernel's
  pdl_wait();
  if (chunks == 0 || h0 + h >= a.group) return;
  const int n_ctas = (int)min((int64_t)a.n_ctas, total);
  first += (int64_t)sub * chunks;
  const int i0 = cta_of(first, total, n_ctas), i1 = cta_of(first + chunks - 1, total, n_ctas);
  if (i0 == i1) return;
  // the first run ends with this group's start, the others begin inside it
  auto part = [&](int i) { return a.part + ((int64_t)i * 2 + (i == i0 ? 1 : 0)) * S::kPartFloats; };
  float mm = -INFINITY;
  for (int i = i0 + tid; i <= i1; i += kJoinThreads) mm = fmaxf(mm, __ldcg(part(i) + kGroup * D + h));
  mm = warp_max(mm);
  if ((tid & 31) == 0) m_s[tid >> 5] = mm;
  __syncthreads();
  for (int w = 0; w < kJoinThreads / 32; ++w) mm = fmaxf(mm, m_s[w]);
  const float ref = mm == -INFINITY ? 0.0f : mm;
  const int lane = tid % kLanes, row = tid / kLanes;
  if (row < kSlots) {
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
#pragma unroll 4
    for (int i = i0 + row; i <= i1; i += kSlots) {
      const float* p = part(i);
      const float f = exp2f(__ldcg(p + kGroup * D + h) - ref);
      const float4 x = __ldcg(reinterpret_cast<const float4*>(p + h * D) + lane);
      l = fmaf(__ldcg(p + kGroup * D + kGroup + h), f, l);
      acc.x = fmaf(x.x, f, acc.x);
      acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z);
      acc.w = fmaf(x.w, f, acc.w);
    }
    acc_s[row][lane] = acc;
    if (lane == 0) l_s[row] = l;
  }
  __syncthreads();
  if (tid < D) {
    float x = 0.0f, l = 0.0f;
    for (int s = 0; s < kSlots; ++s) {
      x += reinterpret_cast<const float*>(&acc_s[s][0])[tid];
      l += l_s[s];
    }
    a.out[col * a.ldo + ((int64_t)kvh * a.group + h0 + h) * D + tid] = __fdiv_rn(x, l);
  }
}

template <int NB>
constexpr size_t attention_smem() {
  return (size_t)kWarps * kStages * Shape<NB>::kStageBytes;
}
static_assert(Shape<1>::kStageBytes * kStages >= kGroup * 32 * 4 &&
                  Shape<4>::kStageBytes * kStages >= kGroup * 128 * 4,
              "a warp's ring holds its sums");

template <int NB>
cudaError_t launch_attention_q40(const AttnQ40Args& args, bool join, cudaStream_t st) {
  static DeviceOnce once;
  cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(kv_q40_attention_kernel<NB>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)attention_smem<NB>());
  });
  if (e != cudaSuccess) return e;
  e = launch(kv_q40_attention_kernel<NB>, dim3(args.n_ctas), dim3(kThreads), attention_smem<NB>(),
             st, false, args);
  if (e != cudaSuccess || !join) return e;
  return launch(kv_q40_join_kernel<NB>, dim3((unsigned)(args.n_cols * args.subs), kGroup),
                dim3(kJoinThreads), 0, st, use_pdl(), args);
}

// CTAs of the attention kernel: three for each SM, or the most chunks there can be.
int attention_ctas(int n_cols, int subs, int max_seq) {
  const int64_t units = (int64_t)n_cols * subs * ((max_seq + kChunk - 1) / kChunk);
  const int64_t most = (int64_t)3 * sm_count();
  return (int)(units < most ? units : most);
}
size_t part_bytes(int n_cols, int subs, int max_seq, int head_dim) {
  return (size_t)attention_ctas(n_cols, subs, max_seq) * 2 * kGroup * (head_dim + 2) * sizeof(float);
}

bool shape_ok(int n_layers, int n_slots, int max_seq, int n_kv_heads, int head_dim) {
  return n_layers > 0 && n_slots > 0 && max_seq > 0 && max_seq <= INT_MAX - 256 && n_kv_heads > 0 &&
         head_dim > 0 && head_dim % 32 == 0 && head_dim <= 32 * kMaxBlocks;
}

// The status of a cache argument; on success its layer `layer`.
int check_cache(const std::string& api, const dqmk_kv_q40* kv, int layer, Plane* out) {
  if (!kv || !kv->keys_dev || !kv->values_dev) return fail(DQMK_ERR_INVALID, api + ": null pointer");
  if (kv->n_layers <= 0 || kv->n_slots <= 0 || kv->max_seq <= 0 || kv->n_kv_heads <= 0)
    return fail(DQMK_ERR_INVALID, api + ": invalid cache shape");
  if (!shape_ok(kv->n_layers, kv->n_slots, kv->max_seq, kv->n_kv_heads, kv->head_dim))
    return fail(DQMK_ERR_UNSUPPORTED, api + ": head_dim must be a multiple of 32 of at most 128");
  if ((reinterpret_cast<uintptr_t>(kv->keys_dev) | reinterpret_cast<uintptr_t>(kv->values_dev)) & 15u)
    return fail(DQMK_ERR_INVALID, api + ": KV cache must be 16-byte aligned");
  if (layer < 0 || layer >= kv->n_layers) return fail(DQMK_ERR_RANGE, api + ": layer out of range");
  const int64_t rows = padded_rows(kv->max_seq);
  const int64_t per_layer = (int64_t)kv->n_slots * kv->n_kv_heads * rows, all = per_layer * kv->n_layers;
  const int nb = kv->head_dim / 32;
  uint8_t* kb = static_cast<uint8_t*>(kv->keys_dev);
  uint8_t* vb = static_cast<uint8_t*>(kv->values_dev);
  out->kq = kb + per_layer * layer * 16 * nb;
  out->vq = vb + per_layer * layer * 16 * nb;
  out->kd = reinterpret_cast<uint16_t*>(kb + all * 16 * nb) + per_layer * layer * nb;
  out->vd = reinterpret_cast<uint16_t*>(vb + all * 16 * nb) + per_layer * layer * nb;
  out->n_slots = kv->n_slots, out->max_seq = kv->max_seq, out->n_kv_heads = kv->n_kv_heads;
  out->nb = nb, out->rows = rows;
  return DQMK_OK;
}

unsigned rows_grid(const Plane& c, int n_tokens) {
  const int64_t threads = (int64_t)2 * c.n_kv_heads * c.nb * n_tokens * 8;
  const int64_t blocks = (threads + 255) / 256, most = (int64_t)sm_count() * 32;
  return (unsigned)(blocks < most ? blocks : most);
}

bool vec_rows(const void* k, const void* v, int64_t ldk, int64_t ldv) {
  return ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
           (uintptr_t)((ldk | ldv) * 4)) & 15u) == 0;
}

int check_rows(const std::string& api, const Plane& c, const void* k, const void* v, int64_t ldk,
               int64_t ldv, const int* positions, int n_tokens) {
  const int64_t width = (int64_t)c.n_kv_heads * c.nb * 32;
  if (n_tokens < 0) return fail(DQMK_ERR_INVALID, api + ": negative token count");
  if (ldk < width || ldv < width)
    return fail(DQMK_ERR_INVALID, api + ": row stride shorter than the row");
  if (n_tokens && (!k || !v || !positions)) return fail(DQMK_ERR_INVALID, api + ": null pointer");
  return DQMK_OK;
}

}  // namespace

cudaError_t read_kv_error(unsigned int* flags, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(flags, g_kv_error, sizeof(unsigned int));
  if (e == cudaSuccess && clear && *flags) {
    const unsigned int zero = 0;
    e = cudaMemcpyToSymbol(g_kv_error, &zero, sizeof(unsigned int));
  }
  return e;
}

}  // namespace dqmk

// ------------------------------------------------------------------ C ABI
using namespace dqmk;

extern "C" size_t dqmk_kv_q40_bytes(int n_layers, int n_slots, int max_seq, int n_kv_heads,
                                    int head_dim) {
  if (!shape_ok(n_layers, n_slots, max_seq, n_kv_heads, head_dim)) return 0;
  return (size_t)n_layers * n_slots * n_kv_heads * padded_rows(max_seq) * (head_dim / 32) * 18;
}

extern "C" int dqmk_kv_q40_write(const dqmk_kv_q40* kv, int layer, const float* k, int64_t ldk,
                                 const float* v, int64_t ldv, const int* slots,
                                 const int* positions, int n_tokens, void* stream) {
  const std::string api = "KvQ40Write";
  RowsArgs a = {};
  int rc = check_cache(api, kv, layer, &a.c);
  if (rc) return rc;
  if ((rc = check_rows(api, a.c, k, v, ldk, ldv, positions, n_tokens))) return rc;
  if (n_tokens == 0) return DQMK_OK;
  a.k = k, a.v = v, a.ldk = ldk, a.ldv = ldv;
  a.slots = slots, a.positions = positions, a.n_tokens = n_tokens;
  const dim3 grid(rows_grid(a.c, n_tokens)), block(256);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  DQMK_CUDA_RET(api.c_str(), vec_rows(k, v, ldk, ldv)
                                 ? launch(kv_q40_write_kernel<true>, grid, block, 0, st, false, a)
                                 : launch(kv_q40_write_kernel<false>, grid, block, 0, st, false, a));
  return DQMK_OK;
}

extern "C" int dqmk_kv_q40_read(const dqmk_kv_q40* kv, int layer, const int* slots,
                                const int* positions, int n_tokens, float* k, int64_t ldk, float* v,
                                int64_t ldv, void* stream) {
  const std::string api = "KvQ40Read";
  RowsArgs a = {};
  int rc = check_cache(api, kv, layer, &a.c);
  if (rc) return rc;
  if ((rc = check_rows(api, a.c, k, v, ldk, ldv, positions, n_tokens))) return rc;
  if (n_tokens == 0) return DQMK_OK;
  a.ko = k, a.vo = v, a.ldk = ldk, a.ldv = ldv;
  a.slots = slots, a.positions = positions, a.n_tokens = n_tokens;
  const dim3 grid(rows_grid(a.c, n_tokens)), block(256);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  DQMK_CUDA_RET(api.c_str(), vec_rows(k, v, ldk, ldv)
                                 ? launch(kv_q40_read_kernel<true>, grid, block, 0, st, false, a)
                                 : launch(kv_q40_read_kernel<false>, grid, block, 0, st, false, a));
  return DQMK_OK;
}

extern "C" size_t dqmk_kv_q40_attention_workspace(const dqmk_kv_q40* kv, int n_cols, int n_heads) {
  if (!kv || !shape_ok(kv->n_layers, kv->n_slots, kv->max_seq, kv->n_kv_heads, kv->head_dim) ||
      n_cols <= 0 || n_heads <= 0 || n_heads % kv->n_kv_heads != 0)
    return 0;
  const int subs = kv->n_kv_heads * ((n_heads / kv->n_kv_heads + kGroup - 1) / kGroup);
  return part_bytes(n_cols, subs, kv->max_seq, kv->head_dim);
}

extern "C" int dqmk_kv_q40_attention(const dqmk_kv_q40* kv, int layer, const float* q, int64_t ldq,
                                     const int* slots, const int* lengths, int n_cols, int n_heads,
                                     float* out, int64_t ldo, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const std::string api = "KvQ40Attention";
  AttnQ40Args a = {};
  int rc = check_cache(api, kv, layer, &a.c);
  if (rc) return rc;
  if (n_heads <= 0 || n_heads % kv->n_kv_heads != 0)
    return fail(DQMK_ERR_INVALID, api + ": invalid head configuration");
  if (n_cols < 0) return fail(DQMK_ERR_INVALID, api + ": negative column count");
  const int64_t width = (int64_t)n_heads * kv->head_dim;
  if (ldq < width || ldo < width)
    return fail(DQMK_ERR_INVALID, api + ": row stride shorter than the row");
  if (n_cols == 0) return DQMK_OK;
  if (!q || !lengths || !out || !workspace) return fail(DQMK_ERR_INVALID, api + ": null pointer");
  if (reinterpret_cast<uintptr_t>(workspace) & 15u)
    return fail(DQMK_ERR_INVALID, api + ": workspace must be 16-byte aligned");
  a.group = n_heads / kv->n_kv_heads;
  const int64_t subs = (int64_t)kv->n_kv_heads * ((a.group + kGroup - 1) / kGroup);
  if (subs * n_cols > INT_MAX) return fail(DQMK_ERR_UNSUPPORTED, api + ": too many columns");
  a.subs = (int)subs;
  const size_t need = part_bytes(n_cols, a.subs, kv->max_seq, kv->head_dim);
  if (workspace_bytes < need)
    return fail(DQMK_ERR_INVALID, api + ": workspace of " + std::to_string(workspace_bytes) +
                                      " bytes, needs " + std::to_string(need));
  a.q = q, a.ldq = ldq, a.out = out, a.ldo = ldo;
  a.lengths = lengths, a.slots = slots, a.n_cols = n_cols, a.n_heads = n_heads;
  a.scale = kLog2e / sqrtf((float)kv->head_dim);
  a.part = static_cast<float*>(workspace);
  a.n_ctas = attention_ctas(n_cols, a.subs, kv->max_seq);
  const bool join = kv->max_seq > kChunk;  // else every run ends with a whole group
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (a.c.nb) {
    case 1: e = launch_attention_q40<1>(a, join, st); break;
    case 2: e = launch_attention_q40<2>(a, join, st); break;
    case 3: e = launch_attention_q40<3>(a, join, st); break;
    default: e = launch_attention_q40<4>(a, join, st); break;
  }
  DQMK_CUDA_RET(api.c_str(), e);
  return DQMK_OK;
}
