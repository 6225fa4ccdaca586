// attention_prompt.cu -- causal attention over packed prompts, on tcgen05.
//
// Sequence s holds tokens starts[s] .. starts[s+1]-1 of the packed rows; token
// i of it, query head h, key/value head h / group:
//   s_ij = q_i . k_j / sqrt(D) for j <= i, softmax over j, out_i = sum p_ij v_j
//
// Both products run on the tensor cores with f32 results: an operand is scaled
// by a power of two that brings the largest of those that share it into [2^14,
// 2^15) and split into two fp16 terms (x = hi + lo + r, |r| <= 2^-22 |x|, or 2^-25
// where lo is subnormal), and A_hi B_hi + A_hi B_lo + A_lo B_hi accumulate in fp32
// tensor memory.  That is three products for one, 562 TFLOP/s of the measured 1686;
// f32 FMAs have an eighth of it.
//
// First kernel (prompt_split): K and V of every sequence, in tiles of 64 keys
// that start at the sequence's first token, become the shared-memory images of
// the second kernel's operands (K rows, V columns, both terms, 128-byte
// swizzle), so that a tile is one contiguous bulk copy and needs neither a
// tensor map nor any alignment of the sequence's first token.  K and V each take
// one power of two a tile.  A tile whose rows and channels differ in size by more
// than 2^14 together would lose bits of the smaller ones, and one that holds an
// infinity or a NaN would reach queries that must not see it; it is marked, and the
// second kernel takes it in f32 straight from the inputs.  With r, c and t the
// largest of an element's row, channel and tile, r c / t is then at least 2^-2 in the
// scale of the terms, so an element is off by at most 2^-22 |x| or 2^-23 r c / t,
// whatever sizes rows and channels have.
//
// One more CTA of that kernel lists the second kernel's items, those with the
// most keys first.
//
// Second kernel: an item is 128 rows (token, head of the group) of one sequence
// and KV head, row f = token * group + head: the heads that share keys fill a
// tile also where the sequence is short, and a tile of rows spans few tokens,
// so little of the masked triangle is computed.  Row r is TMEM lane r.  A CTA
// stays on its SM and takes items from the list.  One warp streams the tiles
// (past the item's end, on into the next one's), one issues the products, eight
// run the softmax, warps w and w + 4 on the same 32 rows and half of the columns
// each:
//   S(j) = Q K_j^T      A = Q (TMEM), B = K_j
//   P(j) = exp2(S f - m) 2^14, two terms, over S(j)'s own columns
//   O'(j) = P(j) V_j    A = P(j) (TMEM), B = V_j; o = o corr + O' 2^e in registers
// S(j+1) is issued before P(j) is waited for, so the tensor cores work on the
// next scores while the softmax runs, and the next item's queries go to TMEM
// while the last O' is computed.  A row a thread would touch 32 lines with each
// load and store: queries come and outputs go in whole rows through a shared-memory stage, the
// queries of the next item under this one's last tiles, the outputs under the
// next one's first (with the list, 396 -> 260 us for 33 ragged prompts of 28 / 4
// heads of 128; the queries under the last tiles 240 -> 233).
//
// Bound: a tile's products, 1840 cycles at 128 and 1075 at 64, and its softmax, which
// they overlap in part (2670 and 1950 cycles a tile); an item's ends where it has few
// keys.  28 / 4 heads of 128 on one B200, graphs of calls: 8192 tokens 1069 us, 1350
// TFLOP/s of fp16 products (80% of the measured 1686; 1249 us at 1477 MHz in a run of
// seconds, at the power limit), 33 ragged prompts 233 us (280 by a call on new inputs);
// 602 tokens of 14 / 2 heads of 64 19.5 us.  A score product of 64 keys takes 44.8
// cycles, 32 by its operations; one of 128 its full 64.
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "tc_dev.cuh"

namespace dqmk {
namespace {

__device__ unsigned int g_prompt_error;  // kErrTimeout / kErrBadIndex

constexpr int kMaxDim = 128;
constexpr int kRows = 128, kKeys = 64;
constexpr int kMaxGroup = 1 << 20;  // small_div
constexpr float kLog2e = 1.44269504088896341f;

struct PromptArgs {
  const float *q, *k, *v;
  int64_t ldq, ldk, ldv;
  const int* starts;
  int n_seqs, n_tokens, n_heads, n_kv_heads, group, head_dim;
  float* out;
  int64_t ldo;
  float scale;            // log2(e) / sqrt(D)
  unsigned char* images;  // [tile][kv_head] operand images
  float4* meta;           // [tile][kv_head]: 2^ek, K marked, 2^ev, V marked
  struct Item* items;     // row tiles, those with the most keys first
  int* heads;             // [0]: row tiles listed, [1]: items taken past each CTA's first
  int max_tiles, max_items;
};

// 128 rows of one sequence: its first token, its tokens, the first row, and the
// key tiles before the sequence.
struct Item {
  int first, n, row, key_tiles;
};

// DP: head_dim rounded up to 64 or 128.  CTAS: CTAs of the second kernel on an SM,
// which its registers are shared among.
template <int DP, int CTAS = 1>
struct Cfg {
  static constexpr int kPlane = kKeys * DP * 2;     // one term of K or V
  static constexpr int kOperand = 2 * kPlane;       // both terms
  static constexpr int kImage = 2 * kOperand;       // K, then V
  static constexpr int kStages = 2;
  static constexpr int kBufs = DP == 128 ? 3 : 2;   // score buffers
  static constexpr int kParts = 2;  // softmax warps on the same rows
  static constexpr int kSoftWarps = 4 * kParts, kThreads = 32 * (kSoftWarps + 2);
  // the stage: a row's queries or outputs, rows 16 bytes apart modulo the 128 of all banks
  static constexpr int kRowBytes = DP * 4 + 16;
  static constexpr int kSmem = kStages * kImage + kRows * kRowBytes + 1024;
  static constexpr uint32_t kTmem = DP == 128 ? 512 : 256;
  static constexpr uint32_t kColQ = 0, kColO = DP, kColS = 2 * DP;
  static_assert(2 * DP + 64 * kBufs <= kTmem, "tensor memory plan");
};

__device__ __forceinline__ int seq_len(const PromptArgs& a, int s) {
  const int t0 = a.starts[s], t1 = a.starts[s + 1];
  return t0 >= 0 && t1 >= t0 && t1 <= a.n_tokens ? t1 - t0 : 0;
}
__device__ __forceinline__ int key_tiles_of(int n) { return (n + kKeys - 1) / kKeys; }
__device__ __forceinline__ int row_tiles_of(const PromptArgs& a, int n) {
  return (int)(((int64_t)n * a.group + kRows - 1) / kRows);
}
// Key tiles that rows row .. row + 127 of a sequence of n tokens see.
__device__ __forceinline__ int item_tiles(const PromptArgs& a, int n, int row) {
  const int64_t last = min((int64_t)row + kRows, (int64_t)n * a.group) - 1;
  return (int)(last / a.group) / kKeys + 1;
}

// ------------------------------------------------------------ first kernel
constexpr int kSplitThreads = 256;
// Exponents from a tile's largest value to its smallest row's largest, and to its
// smallest channel's, added up (rows and channels of zeros left out).
constexpr int kMostSpread = 14;

constexpr int kBins = 1024;      // items are listed by their key tiles, up to this many

// The list of row tiles, by one CTA of kSplitThreads.  Sequences whose key tiles
// do not fit the workspace (only offsets that overlap have any) are left out.
__device__ void list_items(const PromptArgs& a) {
  __shared__ int bins[kBins], lens[kSplitThreads], firsts[kSplitThreads], tiles[kSplitThreads];
  __shared__ int64_t warp_sums[kSplitThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < kBins; i += kSplitThreads) bins[i] = 0;
  // twice over the sequences: first the bins' sizes, then the places
  for (int pass = 0; pass < 2; ++pass) {
    int64_t before_chunk = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += kSplitThreads) {
      const int s = s0 + tid, n = s < a.n_seqs ? seq_len(a, s) : 0;
      int64_t before;
      const int64_t sum = block_scan(key_tiles_of(n), &before, warp_sums);
      before += before_chunk;
      const bool fits = before + key_tiles_of(n) <= a.max_tiles;
      if (pass == 0 && s < a.n_seqs) {
        const int t0 = a.starts[s], t1 = a.starts[s + 1];
        if (!fits || t0 < 0 || t1 < t0 || t1 > a.n_tokens) atomicOr(&g_prompt_error, kErrBadIndex);
      }
      lens[tid] = fits ? n : 0;
      firsts[tid] = n ? a.starts[s] : 0;
      tiles[tid] = fits ? (int)before : 0;
      __syncthreads();
      for (int i = warp; i < min(kSplitThreads, a.n_seqs - s0); i += kSplitThreads / 32) {
        const int len = lens[i], count = row_tiles_of(a, len);
        for (int r = lane; r < count; r += 32) {
          const int bin = kBins - min(item_tiles(a, len, r * kRows), kBins);
          const int at = atomicAdd(&bins[bin], 1);
          if (pass && at < a.max_items) a.items[at] = Item{firsts[i], len, r * kRows, tiles[i]};
        }
      }
      __syncthreads();
      before_chunk += sum;
    }
    if (pass == 0) {
      constexpr int kEach = kBins / kSplitThreads;
      int own[kEach], sum = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) sum += own[i] = bins[tid * kEach + i];
      int64_t before;
      const int64_t total = block_scan(sum, &before, warp_sums);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        bins[tid * kEach + i] = (int)before;
        before += own[i];
      }
      if (tid == 0) {
        a.heads[0] = (int)min(total, (int64_t)a.max_items);
        a.heads[1] = 0;
      }
      __syncthreads();
    }
  }
}

template <int DP>
__global__ void __launch_bounds__(kSplitThreads) prompt_split_kernel(const PromptArgs a) {
  using C = Cfg<DP>;
  constexpr int kF4 = DP / 4, kPer = kKeys * kF4 / kSplitThreads;  // float4s a row, a thread
  __shared__ int64_t warp_sums[kSplitThreads / 32];
  __shared__ int place[3];  // the tile's sequence: first token, tokens, key tiles before it
  __shared__ float vt[kKeys][DP + 1];
  __shared__ int top_bits, low_row, channel_bits[DP];
  const int tid = threadIdx.x, kvh = blockIdx.y >> 1, is_v = blockIdx.y & 1, D = a.head_dim;
  pdl_trigger();
  if (blockIdx.x == 0) {  // first, so that it does not end last
    if (blockIdx.y == 0) list_items(a);
    return;
  }
  const int64_t tile = (int64_t)blockIdx.x - 1;  // < max_tiles: the grid's size
  if (tid == 0) {
    place[1] = 0;
    top_bits = 0;
    low_row = INT_MAX;
  }
  if (tid < DP) channel_bits[tid] = 0;
  int64_t done = 0;
  for (int s0 = 0; s0 < a.n_seqs && done <= tile; s0 += kSplitThreads) {
    const int s = s0 + tid, n = s < a.n_seqs ? seq_len(a, s) : 0;
    int64_t before;
    const int64_t sum = block_scan(key_tiles_of(n), &before, warp_sums);
    before += done;
    if (tile >= before && tile < before + key_tiles_of(n)) {
      place[0] = a.starts[s];
      place[1] = n;
      place[2] = (int)before;
    }
    done += sum;
  }
  __syncthreads();
  if (place[1] == 0) return;
  const int k0 = (int)(tile - place[2]) * kKeys, live = min(kKeys, place[1] - k0);
  unsigned char* image = a.images + (tile * a.n_kv_heads + kvh) * C::kImage + (is_v ? C::kOperand : 0);

  // a thread's float4s of one row sit kSplitThreads / kF4 rows apart
  const int c4 = tid % kF4, r0 = tid / kF4;
  const int64_t ld = is_v ? a.ldv : a.ldk;
  const float* base = (is_v ? a.v : a.k) + (int64_t)(place[0] + k0) * ld + (int64_t)kvh * D;
  float4 x[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = r0 + i * (kSplitThreads / kF4);
    x[i] = r < live && 4 * c4 < D ? ldg_f4_stream(base + r * ld + 4 * c4)
                                  : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  // sizes compare as integers; an infinity or a NaN is larger than any number
  int channels[4] = {0, 0, 0, 0};  // of this thread's rows
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int size[4] = {__float_as_int(fabsf(x[i].x)), __float_as_int(fabsf(x[i].y)),
                         __float_as_int(fabsf(x[i].z)), __float_as_int(fabsf(x[i].w))};
#pragma unroll
    for (int e = 0; e < 4; ++e) channels[e] = max(channels[e], size[e]);
    int top = max(max(size[0], size[1]), max(size[2], size[3]));
#pragma unroll
    for (int o = 1; o < (kF4 < 32 ? kF4 : 32); o <<= 1)
      top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (c4 == 0 && top > 0) {
      atomicMax(&top_bits, top);
      atomicMin(&low_row, top);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) atomicMax(&channel_bits[e * kF4 + c4], channels[e]);
  __syncthreads();
  int low_channel = INT_MAX;  // by every warp
#pragma unroll
  for (int i = 0; i < DP; i += 32) {
    const int size = channel_bits[i + (tid & 31)];
    low_channel = min(low_channel, size ? size : INT_MAX);
  }
  low_channel = __reduce_min_sync(0xffffffffu, low_channel);
  const int top = top_bits;
  const int spread = 2 * (top >> 23) - (low_row >> 23) - (low_channel >> 23);
  const bool marked = top >= 0x7f800000 || (top > 0 && spread > kMostSpread);
  const int e = pow2_ex(__int_as_float(top));
  const float down = pow2f(-e);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    float4& f = x[i];
    f.x *= down, f.y *= down, f.z *= down, f.w *= down;
    if (marked) f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // the products must add nothing
  }
  if (!is_v) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = r0 + i * (kSplitThreads / kF4);
      uint2 hi, lo;
      split2(x[i].x, x[i].y, hi.x, lo.x);
      split2(x[i].z, x[i].w, hi.y, lo.y);
      // columns 64 h ..: plane half h, 8-byte half (c4 & 1) of chunk (c4 % 16) / 2
      unsigned char* dst = image + (c4 / 16) * (kKeys * 128) + tc::sw128(r, (c4 % 16) >> 1) + (c4 & 1) * 8;
      *reinterpret_cast<uint2*>(dst) = hi;
      *reinterpret_cast<uint2*>(dst + C::kPlane) = lo;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      float* to = &vt[r0 + i * (kSplitThreads / kF4)][4 * c4];
      to[0] = x[i].x, to[1] = x[i].y, to[2] = x[i].z, to[3] = x[i].w;
    }
    __syncthreads();
    // operand row d holds the 64 keys; a thread writes 16-byte chunks of 8 keys
#pragma unroll
    for (int i = tid; i < DP * 8; i += kSplitThreads) {
      const int d = i / 8, c = i % 8;
      uint4 hi, lo;
      split2(vt[8 * c][d], vt[8 * c + 1][d], hi.x, lo.x);
      split2(vt[8 * c + 2][d], vt[8 * c + 3][d], hi.y, lo.y);
      split2(vt[8 * c + 4][d], vt[8 * c + 5][d], hi.z, lo.z);
      split2(vt[8 * c + 6][d], vt[8 * c + 7][d], hi.w, lo.w);
      unsigned char* dst = image + tc::sw128(d, c);
      *reinterpret_cast<uint4*>(dst) = hi;
      *reinterpret_cast<uint4*>(dst + C::kPlane) = lo;
    }
  }
  if (tid == 0)
    reinterpret_cast<float2*>(a.meta + tile * a.n_kv_heads + kvh)[is_v] = make_float2(pow2f(e), marked ? 1.0f : 0.0f);
}

// ------------------------------------------------------------ second kernel
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
               "r"(tc::su32(src)), "r"(bytes)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// The warps w, w + 4, .. that share 32 rows: a barrier, and the AND of a predicate.
template <int N>
__device__ __forceinline__ void rows_sync(int quarter) {
  asm volatile("bar.sync %0, %1;" ::"r"(quarter + 1), "n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ bool rows_and(int quarter, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "bar.red.and.pred q, %1, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(quarter + 1), "r"((uint32_t)x), "n"(N)
      : "memory");
  return r != 0;
}
// 32 columns of this warp's 32 rows to registers; 8 from registers.
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// 16 rows of 8 columns: lane l has columns 2 (l % 4) + {0, 1} of row l / 4 in
// r[0], r[1] and of row l / 4 + 8 in r[2], r[3].
__device__ __forceinline__ void tmem_st_rows16(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x1.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]));
}

// An item as the roles of a CTA see it; kvh < 0: no more.
struct Work {
  Item it;
  int kvh, tiles, first_tok, first_head;  // of the item's first row
};
// x / d for 0 <= x < 2^21, inv = 1 / d: (x + 1/2) / d is at least 1 / 2d from a
// whole number, more than the roundings move it.
__device__ __forceinline__ int small_div(int x, float inv) { return (int)(((float)x + 0.5f) * inv); }

// WITHHOLD: a test hook, the copies of the keys of tile `withheld` are never made.
template <int DP, int CTAS, bool WITHHOLD>
__global__ void __launch_bounds__(Cfg<DP, CTAS>::kThreads, CTAS)
    attention_prompt_kernel(const PromptArgs a, const int withheld) {
  using C = Cfg<DP, CTAS>;
  constexpr int ST = C::kStages, NB = C::kBufs, kSoftWarps = C::kSoftWarps;
  constexpr int P = C::kParts, kShare = 32 * P;  // threads that share 32 rows
  constexpr int W = DP / P, K = kKeys / P;       // output columns and keys of a thread
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t kfull[ST], kempty[ST], vfull[ST], vempty[ST];
  __shared__ __align__(8) uint64_t s_done[NB], p_ready[NB], o_done, o_free, q_ready, fin;
  __shared__ __align__(8) uint64_t work_full[2], work_empty[2];
  __shared__ Work work[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  __shared__ float red[2][P][kRows], red_q[kRows], red_l[P][kRows];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* stage = smem + ST * C::kImage;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      tc::bar_init(&kfull[i], 1);
      tc::bar_init(&kempty[i], 1);
      tc::bar_init(&vfull[i], 1);
      tc::bar_init(&vempty[i], 1);
    }
    for (int i = 0; i < NB; ++i) {
      tc::bar_init(&s_done[i], 1);
      tc::bar_init(&p_ready[i], 32 * kSoftWarps);
    }
    for (int i = 0; i < 2; ++i) {
      tc::bar_init(&work_full[i], 1);
      tc::bar_init(&work_empty[i], 1 + 32 * kSoftWarps);
    }
    tc::bar_init(&o_done, 1);
    tc::bar_init(&o_free, 32 * kSoftWarps);
    tc::bar_init(&q_ready, 32 * kSoftWarps);
    tc::bar_init(&fin, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kSoftWarps + 1) tc::tmem_alloc(&tmem_slot, C::kTmem);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  auto wait = [&](uint64_t* b, int phase) {
    return tc::bar_wait(b, (uint32_t)(phase & 1), &abort_flag, &g_prompt_error);
  };
  pdl_wait();  // the first kernel's list, images and sizes

  // Tiles are counted through all items of the CTA (T, from 0): tile T uses
  // stage T % ST and score buffer T % NB; items are counted by w.
  if (warp == kSoftWarps) {
    // ---- the items and their tiles
    asm volatile("fence.proxy.async.global;" ::: "memory");
    const int total = __ldcg(a.heads) * a.n_kv_heads;  // at most INT_MAX: the host's check
    int nk = 0, nv = 0;  // copies issued, by lane 0
    // The next item, posted for the other roles once the item before last's
    // place is free; its queries start towards L2.
    auto post = [&](int w, Work& x) {
      int id = blockIdx.x;  // the first one; then from the counter
      if (w > 0) {
        if (lane == 0) id = gridDim.x + atomicAdd(a.heads + 1, 1);
        id = __shfl_sync(0xffffffffu, id, 0);
      }
      x.kvh = -1;
      if (id < total) {
        x.it = a.items[id / a.n_kv_heads];
        x.kvh = id % a.n_kv_heads;
        x.tiles = item_tiles(a, x.it.n, x.it.row);
        const int first = x.it.row / a.group;
        x.first_tok = first;
        x.first_head = x.it.row - first * a.group;
        const int behind = min(x.it.n, (x.it.row + kRows - 1) / a.group + 1);
        const uint32_t bytes = (uint32_t)min(a.group * a.head_dim, 1 << 16) * 4;
        for (int t = first + lane; t < behind; t += 32)
          asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(
                           a.q + (int64_t)(x.it.first + t) * a.ldq + (int64_t)x.kvh * a.group * a.head_dim),
                       "r"(bytes));
      }
      const bool ok = __all_sync(0xffffffffu, w < 2 || wait(&work_empty[w & 1], (w >> 1) - 1));
      if (ok && lane == 0) {
        work[w & 1] = x;
        tc::bar_arrive(&work_full[w & 1]);
      }
      return ok;
    };
    Work x = {}, ahead = {};
    bool ok = post(0, x);
    for (int w = 0; ok && x.kvh >= 0; ++w, x = ahead) {
      ok = post(w + 1, ahead);
      if (lane == 0 && ok) {
        const unsigned char* src = a.images + ((int64_t)x.it.key_tiles * a.n_kv_heads + x.kvh) * C::kImage;
        for (int j = 0; j < x.tiles; ++j, src += (size_t)a.n_kv_heads * C::kImage) {
          const int st = nk % ST;
          unsigned char* dst = smem + st * C::kImage;
          if (nk >= ST && !wait(&kempty[st], nk / ST - 1)) break;
          if (!WITHHOLD || x.it.key_tiles + j != withheld) {
            tc::bar_expect_tx(&kfull[st], C::kOperand);
            tc::bulk_load(dst, src, C::kOperand, &kfull[st]);
          }
          ++nk;
          if (nv >= ST && !wait(&vempty[st], nv / ST - 1)) break;
          tc::bar_expect_tx(&vfull[st], C::kOperand);
          tc::bulk_load(dst + C::kOperand, src + C::kOperand, C::kOperand, &vfull[st]);
          ++nv;
        }
      }
      ok = !__any_sync(0xffffffffu, abort_flag);
    }
    if (lane == 0 && abort_flag) {  // copies in flight land before the CTA ends
      const unsigned long long begin = tc::now_ns();
      auto landed = [&](uint64_t* b, int n) {
        while (!tc::bar_try(b, (uint32_t)n & 1) && tc::now_ns() - begin < tc::kWaitNs) {
        }
      };
      for (int j = max(0, nk - ST); j < nk; ++j) landed(&kfull[j % ST], j / ST);
      for (int j = max(0, nv - ST); j < nv; ++j) landed(&vfull[j % ST], j / ST);
    }
    __syncwarp();
  } else if (warp == kSoftWarps + 1) {
    // ---- the products, by one thread
    if (tc::elect_one()) {
      constexpr uint32_t kIdescS = tc::idesc_f16(kRows, kKeys), kIdescO = tc::idesc_f16(kRows, DP);
      auto scores = [&](int T) {
        const uint32_t d = tmem + C::kColS + 64u * (T % NB), q = tmem + C::kColQ;
        const uint32_t base = tc::su32(smem + (T % ST) * C::kImage);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          // a K = 16 slice: 8 TMEM columns of A, 32 bytes (+2) of the descriptor
          const uint32_t off = (k / 4) * (kKeys * 128);
          const uint64_t hi = tc::smem_desc(base + off) + 2u * (k % 4);
          const uint64_t lo = tc::smem_desc(base + off + C::kPlane) + 2u * (k % 4);
          tc::mma_f16_ts(d, q + 8u * k, hi, kIdescS, k > 0 ? 1u : 0u);
          tc::mma_f16_ts(d, q + 8u * k, lo, kIdescS, 1u);
          tc::mma_f16_ts(d, q + DP / 2 + 8u * k, hi, kIdescS, 1u);
        }
        tc::mma_commit(&s_done[T % NB]);
        tc::mma_commit(&kempty[T % ST]);
      };
      bool ok = true;
      int T = 0;
      for (int w = 0; ok; ++w) {
        ok = wait(&work_full[w & 1], w >> 1);
        if (!ok) break;
        const int kvh = work[w & 1].kvh, nt = work[w & 1].tiles;
        tc::bar_arrive(&work_empty[w & 1]);
        if (kvh < 0) break;
        // the item's first scores: their buffer's last P went into a product that
        // is over, for o_free of the one after it was waited for
        ok = wait(&q_ready, w) && wait(&kfull[T % ST], T / ST);
        tc::tc_fence_after();
        if (ok) scores(T);
        for (int j = 0; ok && j < nt; ++j, ++T) {
          if (j + 1 < nt) {
            ok = wait(&kfull[(T + 1) % ST], (T + 1) / ST);
            // S(T+1) goes over P(T+1-NB), which O'(T+1-NB) has to have read: with
            // three buffers o_free of that product was waited for before O'(T-1)
            if (ok && NB == 2 && T > 0) ok = wait(&o_done, T - 1);
            if (!ok) break;
            tc::tc_fence_after();
            scores(T + 1);
          }
          ok = wait(&vfull[T % ST], T / ST) && wait(&p_ready[T % NB], T / NB) &&
               (T == 0 || wait(&o_free, T - 1));
          if (!ok) break;
          tc::tc_fence_after();
          const uint32_t p = tmem + C::kColS + 64u * (T % NB), d = tmem + C::kColO;
          const uint32_t base = tc::su32(smem + (T % ST) * C::kImage + C::kOperand);
          const uint64_t hi = tc::smem_desc(base), lo = tc::smem_desc(base + C::kPlane);
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k) {
            tc::mma_f16_ts(d, p + 8u * k, hi + 2u * k, kIdescO, k > 0 ? 1u : 0u);
            tc::mma_f16_ts(d, p + 8u * k, lo + 2u * k, kIdescO, 1u);
            tc::mma_f16_ts(d, p + 32 + 8u * k, hi + 2u * k, kIdescO, 1u);
          }
          tc::mma_commit(&o_done);
          tc::mma_commit(&vempty[T % ST]);
        }
      }
      tc::mma_commit(&fin);
    }
    __syncwarp();
  } else {
    // ---- the softmax.  After a wait that ran out the warps go on to the item's
    // end without waiting (their pairs meet at barriers) and store nothing.
    const int quarter = warp & 3, part = warp >> 2;
    const int row = 32 * quarter + lane;
    const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
    const float inv_group = 1.0f / (float)a.group;

    struct Rows {  // this thread's row of an item
      int first_tok, tok, first, kvh, tiles, key_tiles, head;
      float fq;  // scores in base 2: S' fq 2^ek
      float4 meta;  // of the item's first key tile
    };
    // Token (counted from the sequence's) and head of row r of an item.
    auto place = [&](const Work& k, int r, int& head) {
      const int i = k.first_head + r, t = small_div(i, inv_group);
      head = k.kvh * a.group + i - t * a.group;
      return k.first_tok + t;
    };
    // Item w's queries on their way to the stage, once item w - 2's outputs have
    // left it: a warp takes the 16 rows whose outputs it sent, whole rows a copy
    // instruction.  false: no more items.
    auto fetch_item = [&](int w) {
      const bool got = wait(&work_full[w & 1], w >> 1);
      const Work& k = work[w & 1];
      if (!rows_and<kShare>(quarter, got && k.kvh >= 0)) return false;
      asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      __syncwarp();
      int head;
      const int r0 = 32 * quarter + 16 * part, tok = place(k, r0 + (lane & 15), head);
      const int64_t mine = tok < k.it.n ? (int64_t)(k.it.first + tok) * a.ldq + (int64_t)head * a.head_dim : -1;
      constexpr int kLanes = DP / 4;  // 16 bytes a lane
      const int col = 4 * (lane % kLanes);
#pragma unroll 4
      for (int i = 0; i < 16; i += 32 / kLanes) {
        const int r = i + lane / kLanes;
        const int64_t at = __shfl_sync(0xffffffffu, mine, r);
        const int bytes = at >= 0 && col < a.head_dim ? 16 : 0;  // zeros where there is nothing
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                         tc::su32(stage + (r0 + r) * C::kRowBytes + 4 * col)),
                     "l"(a.q + (bytes ? at + col : 0)), "r"(bytes)
                     : "memory");
      }
      return true;
    };
    // The fetched item's row, and its queries scaled, split and stored to TMEM,
    // once the last scores of the item before are over; 4 lanes a row.
    auto take_item = [&](int w, Rows& x) {
      const Work k = work[w & 1];
      tc::bar_arrive(&work_empty[w & 1]);
      x.meta = __ldcg(a.meta + (int64_t)k.it.key_tiles * a.n_kv_heads + k.kvh);
      x.first_tok = k.first_tok;
      x.tok = place(k, row, x.head);
      if (x.tok >= k.it.n) x.tok = -1;
      x.first = k.it.first, x.kvh = k.kvh, x.tiles = k.tiles, x.key_tiles = k.it.key_tiles;

      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      const int r0 = 32 * quarter + 16 * part + (lane >> 2);
      const uint32_t at = tmem + ((uint32_t)(32 * quarter + 16 * part) << 16) + C::kColQ;
      const float4* from[2] = {reinterpret_cast<const float4*>(stage + r0 * C::kRowBytes) + (lane & 3),
                               reinterpret_cast<const float4*>(stage + (r0 + 8) * C::kRowBytes) + (lane & 3)};
      float top[2];
      // queries whose largest value is of ordinary size are split under one scale,
      // 2^10, which leaves elements off by at most 2^-22 of themselves or 2^-34 of
      // that value (so that keys may outweigh them by channel); with others among
      // the 32 rows all are split again, those under a scale of their row, 2^-39
      // (33 ragged prompts 227 us, 237 with every row split again)
      constexpr int kUsual = -10;
      auto usual = [](float t) { return !(t > 0.0f) || (t >= 0.5f && t < 32.0f); };
      float up[2] = {pow2f(-kUsual), pow2f(-kUsual)};
      auto pass = [&] {
        top[0] = top[1] = 0.0f;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float4 v = from[i][4 * c];
            top[i] = fmaxf(top[i], fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
            split2(v.x * up[i], v.y * up[i], hi[2 * i], lo[2 * i]);
            split2(v.z * up[i], v.w * up[i], hi[2 * i + 1], lo[2 * i + 1]);
          }
          tmem_st_rows16(at + 8 * c, hi);
          tmem_st_rows16(at + DP / 2 + 8 * c, lo);
        }
      };
      pass();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        if ((lane & 3) == 0) red_q[r0 + 8 * i] = top[i];
      }
      // behind this barrier the stage's rows of the quarter are free, unless they
      // are read again
      const bool all_usual = rows_and<kShare>(quarter, usual(top[0]) && usual(top[1]));
      const float mine = red_q[row];
      if (!all_usual) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (!usual(top[i])) up[i] = pow2f(-pow2_ex(top[i]));
        pass();
        rows_sync<kShare>(quarter);
      }
      tc::tmem_wait_st();
      tc::tc_fence_before();
      tc::bar_arrive(&q_ready);
      x.fq = a.scale * pow2f(usual(mine) ? kUsual : pow2_ex(mine));
    };

    Rows cur, nxt;
    bool have = fetch_item(0);
    if (have) take_item(0, cur);
    int T = 0;
    for (int w = 0; have; ++w) {
      const int nt = cur.tiles;
      const float4* meta = a.meta + (int64_t)cur.key_tiles * a.n_kv_heads + cur.kvh;
      float o[W];
#pragma unroll
      for (int d = 0; d < W; ++d) o[d] = 0.0f;
      float m = -INFINITY, l = 0.0f, corr = 1.0f, vscale = 0.0f;
      // O'(T): o = o corr(T) + O'(T) 2^ev(T)
      auto take_output = [&](int at) {
        wait(&o_done, at);
        tc::tc_fence_after();
        if (__any_sync(0xffffffffu, corr != 1.0f)) {
#pragma unroll
          for (int d = 0; d < W; ++d) o[d] *= corr;
        }
#pragma unroll
        for (int c = 0; c < W; c += 32) {
          uint32_t r[32];
          tc::tmem_ld32(tmem + lanes + C::kColO + part * W + c, r);
          tc::tmem_wait_ld();
          if (c + 32 == W) {
            tc::tc_fence_before();
            tc::bar_arrive(&o_free);
          }
#pragma unroll
          for (int d = 0; d < 32; ++d) o[c + d] = fmaf(__uint_as_float(r[d]), vscale, o[c + d]);
        }
      };
      float4 next = cur.meta;
      for (int j = 0; j < nt; ++j, ++T) {
        const float4 mt = next;
        if (j + 1 < nt) next = __ldcg(meta + (int64_t)(j + 1) * a.n_kv_heads);
        const int kt = j * kKeys;
        const uint32_t buf = tmem + lanes + C::kColS + 64u * (T % NB);
        wait(&s_done[T % NB], T / NB);
        tc::tc_fence_after();
        uint32_t r[K];
        tc::tmem_ld32(buf + K * part, r);
        tc::tmem_wait_ld();
        const bool slow = mt.y + mt.w != 0.0f;  // the whole CTA's
        float tmax = -INFINITY;
        if (kt + kKeys - 1 <= cur.first_tok) {  // every key is visible to every row
#pragma unroll
          for (int i = 0; i < K; ++i) tmax = fmaxf(tmax, __uint_as_float(r[i]));
        } else {
#pragma unroll
          for (int i = 0; i < K; ++i) {
            if (kt + K * part + i > cur.tok) r[i] = 0xff800000u;  // -inf
            tmax = fmaxf(tmax, __uint_as_float(r[i]));
          }
        }
        red[T & 1][part][row] = tmax;
        rows_sync<kShare>(quarter);
#pragma unroll
        for (int i = 0; i < P; ++i) tmax = fmaxf(tmax, red[T & 1][i][row]);
        // held to a float's normal range: the scales' product may leave it where
        // scores do not, and times 0 or infinity a masked key or a score of 0 is NaN
        const float fs = slow ? 1.0f : fminf(fmaxf(cur.fq * mt.x, 0x1p-126f), 0x1.fffffep127f);
        const float mnew = slow ? m : fmaxf(m, tmax * fs);
        const float ref = mnew == -INFINITY ? 0.0f : mnew;
        const float c = ex2(m - ref);
        m = mnew;
        const float from = slow ? INFINITY : ref - 14.0f;  // a marked tile's weights are 0 here
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int g = 0; g < K; g += 16) {  // 16 keys at a time: few registers
          uint32_t ph[8], pl[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float p0 = ex2(fmaf(__uint_as_float(r[g + 2 * i]), fs, -from));
            const float p1 = ex2(fmaf(__uint_as_float(r[g + 2 * i + 1]), fs, -from));
            sum[0] += p0;
            sum[1] += p1;
            split2(p0, p1, ph[i], pl[i]);
          }
          tmem_st8(buf + K / 2 * part + g / 2, ph);
          tmem_st8(buf + 32 + K / 2 * part + g / 2, pl);
        }
        if (!slow) l = fmaf(l, c, sum[0] + sum[1]);
        tc::tmem_wait_st();
        tc::tc_fence_before();
        tc::bar_arrive(&p_ready[T % NB]);
        if (j == max(nt - 2, 0)) have = fetch_item(w + 1);
        if (j > 0) take_output(T - 1);
        corr = slow ? 1.0f : c;
        vscale = mt.z;
        if (slow && cur.tok >= 0) {
          // the marked tile in f32 from the inputs, o at m's scale; two keys at a time,
          // as a query load takes a line a lane.  With one marked tile in sight of every
          // row, 602 tokens of 14 / 2 heads of 64 take 135 us for 19.5, 2048 of 28 / 4
          // of 128 990 for 85 (190 and 1390 key by key).  8 keys at a time (104, 750)
          // slow the loop that serves the other tiles (4096 tokens of 14 / 2 heads of
          // 64: 120 -> 130 us), as do scores and weights through tensor memory
          // (54, 271; 33 ragged prompts 229 -> 240).
          const float* qr = a.q + (int64_t)(cur.first + cur.tok) * a.ldq + (int64_t)cur.head * a.head_dim;
          const int last = min(cur.tok, kt + kKeys - 1);
#pragma unroll 1
          for (int key = kt; key <= last; key += 2) {
            const float* kr = a.k + (int64_t)(cur.first + key) * a.ldk + (int64_t)cur.kvh * a.head_dim;
            const float* vr = a.v + (int64_t)(cur.first + key) * a.ldv + (int64_t)cur.kvh * a.head_dim + part * W;
            const bool two = key < last;  // no key that the row does not see is read
            const int64_t k_next = two ? a.ldk : 0, v_next = two ? a.ldv : 0;
            float s0 = 0.0f, s1 = 0.0f;
#pragma unroll 4
            for (int d = 0; d < a.head_dim; d += 4) {
              const float4 x = *reinterpret_cast<const float4*>(qr + d);
              const float4 y = *reinterpret_cast<const float4*>(kr + d);
              const float4 z = *reinterpret_cast<const float4*>(kr + k_next + d);
              s0 = fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, fmaf(x.x, y.x, s0))));
              s1 = fmaf(x.w, z.w, fmaf(x.z, z.z, fmaf(x.y, z.y, fmaf(x.x, z.x, s1))));
            }
            s0 *= a.scale;
            s1 = two ? s1 * a.scale : -INFINITY;
            const float top = fmaxf(fmaxf(m, s0), s1), at = top == -INFINITY ? 0.0f : top;
            const float down = ex2(m - at), p0 = ex2(s0 - at + 14.0f), p1 = ex2(s1 - at + 14.0f);
            l *= down;
            if (part == 0) l += p0 + p1;
            m = top;
#pragma unroll
            for (int d = 0; d < W; d += 4) {
              const bool in = part * W + d < a.head_dim;
              const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              const float4 y = in ? *reinterpret_cast<const float4*>(vr + d) : none;
              const float4 z = in && two ? *reinterpret_cast<const float4*>(vr + v_next + d) : none;
              o[d] = fmaf(p1, z.x, fmaf(p0, y.x, o[d] * down));
              o[d + 1] = fmaf(p1, z.y, fmaf(p0, y.y, o[d + 1] * down));
              o[d + 2] = fmaf(p1, z.z, fmaf(p0, y.z, o[d + 2] * down));
              o[d + 3] = fmaf(p1, z.w, fmaf(p0, y.w, o[d + 3] * down));
            }
          }
        }
      }
      if (have) take_item(w + 1, nxt);
      take_output(T - 1);
      red_l[part][row] = l;
      // without a next item the last one's outputs may still be in the stage
      if (!have) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      rows_sync<kShare>(quarter);
      l = red_l[0][row];
#pragma unroll
      for (int i = 1; i < P; ++i) l += red_l[i][row];
      const float inv = __frcp_rn(l);
      float4* to = reinterpret_cast<float4*>(stage + row * C::kRowBytes) + part * (W / 4);
#pragma unroll
      for (int i = 0; i < W / 4; ++i)
        to[i] = make_float4(o[4 * i] * inv, o[4 * i + 1] * inv, o[4 * i + 2] * inv, o[4 * i + 3] * inv);
      tc::fence_proxy_async_smem();
      rows_sync<kShare>(quarter);
      // a copy takes 60 cycles to issue: 32 / P rows a warp
      constexpr int kEach = 32 / P;
      const int src = kEach * part + lane % kEach;
      const int tok = __shfl_sync(0xffffffffu, cur.tok, src), head = __shfl_sync(0xffffffffu, cur.head, src);
      if (lane < kEach && tok >= 0 && !abort_flag)
        bulk_store(a.out + (int64_t)(cur.first + tok) * a.ldo + (int64_t)head * a.head_dim,
                   stage + (32 * quarter + src) * C::kRowBytes, (uint32_t)a.head_dim * 4);
      cur = nxt;
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == kSoftWarps + 1) {
    // every product has completed before its tensor memory is freed
    const unsigned long long begin = tc::now_ns();
    while (!tc::bar_try(&fin, 0u)) {
      if (tc::now_ns() - begin > tc::kWaitNs) {
        atomicOr(&g_prompt_error, kErrTimeout);
        break;
      }
    }
    __syncwarp();
    tc::tmem_free(tmem, C::kTmem);
  }
}

// Key tiles that n_tokens tokens in n_seqs sequences can have.
int64_t most_tiles(int n_tokens, int n_seqs) {
  const int64_t t = (int64_t)n_tokens / kKeys + n_seqs;
  return t < n_tokens ? t : n_tokens;
}

template <int DP, int CTAS, bool WITHHOLD>
cudaError_t launch_items(const PromptArgs& a, int withheld, cudaStream_t st) {
  using C = Cfg<DP, CTAS>;
  static DeviceOnce once;
  const cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(attention_prompt_kernel<DP, CTAS, WITHHOLD>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  if (e != cudaSuccess) return e;
  const int64_t items = (int64_t)a.max_items * a.n_kv_heads, most = (int64_t)CTAS * sm_count();
  return launch(attention_prompt_kernel<DP, CTAS, WITHHOLD>, dim3((unsigned)(items < most ? items : most)),
                dim3(C::kThreads), C::kSmem, st, use_pdl(), a, withheld);
}

template <int DP, bool WITHHOLD>
cudaError_t launch_prompt(const PromptArgs& a, int withheld, cudaStream_t st) {
  const cudaError_t e = launch(prompt_split_kernel<DP>, dim3(a.max_tiles + 1, 2 * a.n_kv_heads),
                               dim3(kSplitThreads), 0, st, false, a);
  if (e != cudaSuccess) return e;
  // At 64 two CTAs fit an SM, with 96 registers each for 168.  Two hide an item's
  // ends, one is faster while a CTA has few items, the longest of which ends last.
  // One / two, us, items an SM: 1 x 4096 tokens of 14 / 2 heads 120 / 133 (3.0), 1 x
  // 5120 176 / 180 (3.8), 1 x 8192 of 8 / 8 263 / 315 (3.5), 1 x 10240 392 / 398 (4.3);
  // 1 x 6144 of 14 / 2 239 / 234 (4.5), 1 x 8192 403 / 390 (6), 1 x 12288 of 8 / 8 550 /
  // 537 (5.2), 12 x 1024 of 14 / 2 115 / 110 (4.5), 37 x 1024 320 / 300 (14).  Packs of
  // short prompts lose by two: 148 x 64 of 14 / 2 49.5 / 52 (8), 300 x 16 52 / 55.5 (4);
  // the host does not know the lengths.
  if constexpr (DP == 64)
    if ((int64_t)a.max_items * a.n_kv_heads > 4 * sm_count()) return launch_items<DP, 2, WITHHOLD>(a, withheld, st);
  return launch_items<DP, 1, WITHHOLD>(a, withheld, st);
}

bool prompt_shape_ok(int n_heads, int n_kv_heads, int head_dim) {
  return n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && head_dim > 0;
}
// Row tiles: a sequence's last one may be short, at most one more for each.
int64_t most_items(int n_tokens, int n_seqs, int group) {
  return (int64_t)n_tokens * group / kRows + (n_seqs < n_tokens ? n_seqs : n_tokens);
}
// The workspace: list heads, list, tile sizes, images.
size_t up256(size_t b) { return (b + 255) / 256 * 256; }
size_t items_bytes(int64_t items) { return 256 + up256((size_t)items * sizeof(Item)); }
size_t meta_bytes(int64_t tiles, int n_kv_heads) {
  return up256((size_t)tiles * n_kv_heads * sizeof(float4));
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

extern "C" size_t dqmk_attention_prompt_workspace(int n_tokens, int n_seqs, int n_heads,
                                                  int n_kv_heads, int head_dim) {
  if (n_tokens <= 0 || n_seqs <= 0 || !prompt_shape_ok(n_heads, n_kv_heads, head_dim) ||
      head_dim > kMaxDim)
    return 0;
  const int64_t tiles = most_tiles(n_tokens, n_seqs);
  const size_t image = head_dim > 64 ? Cfg<128>::kImage : Cfg<64>::kImage;
  return items_bytes(most_items(n_tokens, n_seqs, n_heads / n_kv_heads)) +
         meta_bytes(tiles, n_kv_heads) + (size_t)tiles * n_kv_heads * image;
}

namespace {

int prompt_call(const float* q, int64_t ldq, const float* k, int64_t ldk, const float* v, int64_t ldv,
                const int* starts, int n_seqs, int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                float* out, int64_t ldo, void* workspace, size_t workspace_bytes, int withheld,
                void* stream) {
  const std::string api = "AttentionPrompt";
  if (n_tokens < 0 || n_seqs < 0) return fail(DQMK_ERR_INVALID, api + ": counts must not be negative");
  if (!prompt_shape_ok(n_heads, n_kv_heads, head_dim))
    return fail(DQMK_ERR_INVALID, api + ": invalid head configuration");
  if (head_dim % 4 != 0 || head_dim > kMaxDim)
    return fail(DQMK_ERR_UNSUPPORTED, api + ": head_dim must be a multiple of 4 of at most 128");
  if (n_heads / n_kv_heads > kMaxGroup)
    return fail(DQMK_ERR_UNSUPPORTED, api + ": too many query heads for a key/value head");
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
  if (out == q || out == k || out == v)
    return fail(DQMK_ERR_INVALID, api + ": out must not be an input");
  PromptArgs a = {};
  a.q = q, a.k = k, a.v = v, a.ldq = ldq, a.ldk = ldk, a.ldv = ldv;
  a.starts = starts, a.n_seqs = n_seqs, a.n_tokens = n_tokens;
  a.n_heads = n_heads, a.n_kv_heads = n_kv_heads, a.group = n_heads / n_kv_heads;
  a.head_dim = head_dim, a.out = out, a.ldo = ldo;
  a.scale = kLog2e / sqrtf((float)head_dim);
  a.max_tiles = (int)most_tiles(n_tokens, n_seqs);
  const int64_t items = most_items(n_tokens, n_seqs, a.group);
  if (items * n_kv_heads > INT_MAX / 2 || n_kv_heads > 32767 || (int64_t)n_tokens * a.group > INT_MAX - kRows)
    return fail(DQMK_ERR_UNSUPPORTED, api + ": too many rows");
  a.max_items = (int)items;
  unsigned char* work = static_cast<unsigned char*>(workspace);
  a.heads = reinterpret_cast<int*>(work);
  a.items = reinterpret_cast<Item*>(work + 256);
  work += items_bytes(items);
  a.meta = reinterpret_cast<float4*>(work);
  a.images = work + meta_bytes(a.max_tiles, n_kv_heads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&](auto hook) {
    constexpr bool W = decltype(hook)::value;
    return head_dim > 64 ? launch_prompt<128, W>(a, withheld, st) : launch_prompt<64, W>(a, withheld, st);
  };
  DQMK_CUDA_RET(api.c_str(), withheld < 0 ? run(std::false_type()) : run(std::true_type()));
  return DQMK_OK;
}

}  // namespace

extern "C" int dqmk_attention_prompt(const float* q, int64_t ldq, const float* k, int64_t ldk,
                                     const float* v, int64_t ldv, const int* starts, int n_seqs,
                                     int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                                     float* out, int64_t ldo, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  return prompt_call(q, ldq, k, ldk, v, ldv, starts, n_seqs, n_tokens, n_heads, n_kv_heads, head_dim,
                     out, ldo, workspace, workspace_bytes, -1, stream);
}

extern "C" int dqmk_attention_prompt_withhold_tile(
    const float* q, int64_t ldq, const float* k, int64_t ldk, const float* v, int64_t ldv,
    const int* starts, int n_seqs, int n_tokens, int n_heads, int n_kv_heads, int head_dim, float* out,
    int64_t ldo, void* workspace, size_t workspace_bytes, int tile, void* stream) {
  return prompt_call(q, ldq, k, ldk, v, ldv, starts, n_seqs, n_tokens, n_heads, n_kv_heads, head_dim,
                     out, ldo, workspace, workspace_bytes, tile, stream);
}
