// kv_q40.cu -- a KV cache held in 4 bits: write, read back, attention.
//
// Rows are quantized to Q4_0 blocks exactly as dqmk_quantize_q40 does (a
// block of 32 values: fp16 scale d = absmax / 7, codes n = round(v / d + 8) in
// 0..15, value d (n - 8)).  Each of the two buffers (keys, values) holds, for
// every layer, slot and KV head, its positions in tiles of 32, one after the
// other; a tile is the quants of its 32 rows, then their scales:
//
//   [layer][slot][kv_head][tile]  quants [32][D/2 bytes], scales [16][D/32][2 fp16]
//
// so the positions that a query reads are one contiguous run a head and a tile
// is one copy.  A block's scales of two neighbouring rows make one pair of
// halves.  The bytes of the blocks (byte j: value j low, value j + 16 high) are
// interleaved so that one thread's share of a matrix operand is contiguous:
//   keys    a row: 4-byte words [t][block], word t = bytes 4t .. 4t+3 of the block
//   values  two neighbouring rows: [g][block][row] units of 2 bytes, unit g =
//           bytes 2g, 2g+1 of the block; the 8 parts g of row pair r are turned
//           by 2r, so that 4 pairs lie in different shared-memory banks
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "tc_dev.cuh"

namespace dqmk {
namespace {

__device__ unsigned int g_kv_error;  // kErrTimeout / kErrBadIndex

constexpr int kMaxBlocks = 4;  // 32-value blocks of a row: head_dim at most 128
constexpr int kTile = 32;      // positions of a tile

__host__ __device__ __forceinline__ int64_t tiles_of(int max_seq) {
  return ((int64_t)max_seq + kTile - 1) / kTile;
}
// Bytes of a tile: 18 for a block.
__host__ __device__ constexpr int tile_bytes(int nb) { return kTile * 18 * nb; }

// One layer of the cache.
struct Plane {
  unsigned char *k, *v;
  int n_slots, max_seq, n_kv_heads, nb;
  int64_t tiles;  // of one head
};

__device__ __forceinline__ int64_t first_tile(const Plane& c, int slot, int head) {
  return ((int64_t)slot * c.n_kv_heads + head) * c.tiles;
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

// Offset in its buffer of word t (0..3) of block b of a key row, of unit g
// (0..7) of block b of a value row, and of a block's scale.
__device__ __forceinline__ int64_t key_at(int64_t row, int t, int b, int nb) {
  return (row / kTile) * tile_bytes(nb) + (row % kTile) * (16 * nb) + (t * nb + b) * 4;
}
__host__ __device__ __forceinline__ int value_part(int pair, int g) { return (g + 2 * pair) & 7; }
__device__ __forceinline__ int64_t value_at(int64_t row, int g, int b, int nb) {
  const int r = (int)(row % kTile), pair = r >> 1;
  return (row / kTile) * tile_bytes(nb) + pair * (32 * nb) + (value_part(pair, g) * nb + b) * 4 + (r & 1) * 2;
}
__device__ __forceinline__ int64_t scale_at(int64_t row, int b, int nb) {
  return (row / kTile) * tile_bytes(nb) + kTile * 16 * nb + ((row % kTile / 2) * nb + b) * 4 + (row & 1) * 2;
}

// The cache row a token names, or -1: a padding token (position -1), or a slot
// or position outside the cache, which is recorded.
__device__ __forceinline__ int64_t token_row(const RowsArgs& a, int token, int head) {
  const int pos = a.positions[token], slot = a.slots ? a.slots[token] : token;
  if (pos == -1) return -1;
  if (pos < 0 || pos >= a.c.max_seq || slot < 0 || slot >= a.c.n_slots) {
    atomicOr(&g_kv_error, kErrBadIndex);
    return -1;
  }
  return first_tile(a.c, slot, head) * kTile + pos;
}

// 8 lanes take one block of a token's rows (K's heads, then V's), 4 values each,
// the same block of TOK tokens, whose loads are in flight together.  With 8
// tokens lane j also works out token j's row and scale for the other lanes: the
// divisions and the rounding of the scale take more instructions than a block's
// values, and with each lane repeating them the kernel was bound by its
// instructions (21 us for 8191 tokens of 4 heads of 128 against a floor of 6).
// VEC: 16-byte accesses to the f32 rows.
constexpr int kRowThreads = 256;
constexpr int kWriteTokens = 8, kReadTokens = 4;

__device__ __forceinline__ int64_t shfl8(int64_t x, int lane) {
  const int lo = __shfl_sync(0xffffffffu, (int)x, lane, 8), hi = __shfl_sync(0xffffffffu, (int)(x >> 32), lane, 8);
  return (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
}
// Element `i` of an array in registers.
template <int N>
__device__ __forceinline__ float pick(const float (&x)[N], int i) {
  float y = x[0];
#pragma unroll
  for (int n = 1; n < N; ++n) y = i == n ? x[n] : y;
  return y;
}

template <int NB, int TOK, bool VEC>
__global__ void __launch_bounds__(kRowThreads) kv_q40_write_kernel(const RowsArgs a) {
  const int i8 = threadIdx.x & 7, blocks = a.c.n_kv_heads * NB;
  const int64_t token0 = (int64_t)blockIdx.x * TOK;
  const int tokens = (int)min((int64_t)TOK, a.n_tokens - token0);
  // whole warps stay in the loop: the shuffles name every lane
  for (int u0 = (threadIdx.x & ~31) >> 3; u0 < 2 * blocks; u0 += kRowThreads / 8) {
    const int u = min(u0 + (int)((threadIdx.x & 31) >> 3), 2 * blocks - 1);
    const bool live = u == u0 + (int)((threadIdx.x & 31) >> 3), is_v = u >= blocks;
    const int r = is_v ? u - blocks : u, head = r / NB, b = r % NB;
    const int64_t ld = is_v ? a.ldv : a.ldk;
    const float* src = (is_v ? a.v : a.k) + token0 * ld + r * 32 + 4 * i8;
    float x[TOK][4], top[TOK];
#pragma unroll
    for (int n = 0; n < TOK; ++n) {
      const float* p = src + n * ld;
      if constexpr (VEC) {
        const float4 f = n < tokens ? ldg_f4_stream(p) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        x[n][0] = f.x, x[n][1] = f.y, x[n][2] = f.z, x[n][3] = f.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[n][e] = n < tokens ? p[e] : 0.0f;
      }
    }
    const int own = i8 % TOK;  // the token this lane works out
    const int64_t own_row = live && own < tokens ? token_row(a, (int)(token0 + own), head) : -1;
#pragma unroll
    for (int n = 0; n < TOK; ++n) {
      top[n] = fmaxf(fmaxf(fabsf(x[n][0]), fabsf(x[n][1])), fmaxf(fabsf(x[n][2]), fabsf(x[n][3])));
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], o));
    }
    const float own_top = pick(top, own);
    float own_inv = 0.0f;
    if (own_top > 0.0f) {
      const uint16_t d = f2h_ref(__fdiv_rn(own_top, 7.0f));
      const float stored = h2f(d);
      own_inv = stored == 0.0f ? 0.0f : __fdiv_rn(1.0f, stored);
      if (own_row >= 0 && i8 < TOK)
        *reinterpret_cast<uint16_t*>((is_v ? a.c.v : a.c.k) + scale_at(own_row, b, NB)) = d;
    } else if (own_row >= 0 && i8 < TOK) {
      *reinterpret_cast<uint16_t*>((is_v ? a.c.v : a.c.k) + scale_at(own_row, b, NB)) = 0;
    }
#pragma unroll
    for (int n = 0; n < TOK; ++n) {
      const float inv = TOK > 1 ? __shfl_sync(0xffffffffu, own_inv, n, 8) : own_inv;
      const int64_t row = TOK > 1 ? shfl8(own_row, n) : own_row;
      // round(x inv + 8) held to 0 .. 15: with y = x inv + 8 a multiple of 2^-21
      // below 8, y + 1/2 is exact where it could reach the next whole number, so
      // its floor is y rounded with halves up; adding 2^23 rounded down leaves
      // it in the low bits.  A NaN (inf times 0) is held at 0.
      uint32_t q[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = __fadd_rn(__fmul_rn(x[n][e], inv), 8.0f);
        const float z = fminf(fmaxf(__fadd_rn(y, 0.5f), 0.0f), 15.5f);
        q[e] = __float_as_uint(__fadd_rd(z, 8388608.0f));
      }
      uint32_t codes = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
      if (!(top[n] > 0.0f)) codes = 0;  // a block without a value above 0 (or of NaN): codes and scale 0
      // lanes 0-3 hold values 0..15 of the block, lanes 4-7 values 16..31
      const uint32_t word = codes | __shfl_down_sync(0xffffffffu, codes, 4, 8) << 4;
      if (row < 0 || i8 >= 4) continue;
      if (is_v) {
        *reinterpret_cast<uint16_t*>(a.c.v + value_at(row, 2 * i8, b, NB)) = (uint16_t)word;
        *reinterpret_cast<uint16_t*>(a.c.v + value_at(row, 2 * i8 + 1, b, NB)) = (uint16_t)(word >> 16);
      } else {
        *reinterpret_cast<uint32_t*>(a.c.k + key_at(row, i8, b, NB)) = word;
      }
    }
  }
}

template <int NB, int TOK, bool VEC>
__global__ void __launch_bounds__(kRowThreads) kv_q40_read_kernel(const RowsArgs a) {
  const int i8 = threadIdx.x & 7, t = i8 & 3, blocks = a.c.n_kv_heads * NB;
  const int64_t token0 = (int64_t)blockIdx.x * TOK;
  const int tokens = (int)min((int64_t)TOK, a.n_tokens - token0);
  for (int u0 = (threadIdx.x & ~31) >> 3; u0 < 2 * blocks; u0 += kRowThreads / 8) {
    const int u = min(u0 + (int)((threadIdx.x & 31) >> 3), 2 * blocks - 1);
    const bool live = u == u0 + (int)((threadIdx.x & 31) >> 3), is_v = u >= blocks;
    const int r = is_v ? u - blocks : u, head = r / NB, b = r % NB;
    const unsigned char* base = is_v ? a.c.v : a.c.k;
    const int own = i8 % TOK;
    const int64_t own_row = live && own < tokens ? token_row(a, (int)(token0 + own), head) : -1;
    const float own_d =
        own_row >= 0 ? h2f(*reinterpret_cast<const uint16_t*>(base + scale_at(own_row, b, NB))) : 0.0f;
    uint32_t word[TOK];
    bool in[TOK];
#pragma unroll
    for (int n = 0; n < TOK; ++n) {
      const int64_t row = TOK > 1 ? shfl8(own_row, n) : own_row;
      in[n] = row >= 0;
      word[n] = 0;
      if (!in[n]) continue;
      if (is_v)
        word[n] = *reinterpret_cast<const uint16_t*>(base + value_at(row, 2 * t, b, NB)) |
                  (uint32_t)*reinterpret_cast<const uint16_t*>(base + value_at(row, 2 * t + 1, b, NB)) << 16;
      else
        word[n] = *reinterpret_cast<const uint32_t*>(base + key_at(row, t, b, NB));
    }
    const int64_t ld = is_v ? a.ldv : a.ldk;
    float* dst0 = (is_v ? a.vo : a.ko) + token0 * ld + r * 32 + 4 * i8;
#pragma unroll
    for (int n = 0; n < TOK; ++n) {
      const float d = TOK > 1 ? __shfl_sync(0xffffffffu, own_d, n, 8) : own_d;
      if (!in[n]) continue;
      const uint32_t w = (i8 >= 4 ? word[n] >> 4 : word[n]) & 0x0f0f0f0fu;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = __fmul_rn(d, magic_byte(w, e) - 8388616.0f);  // 2^23 + 8
      float* dst = dst0 + n * ld;
      if constexpr (VEC) {
        *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) dst[e] = y[e];
      }
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
//   output   A = w = p d_b 2^X, B = codes n - 8 (columns of V):
//            O[c] = 2^-X sum_j w_j (n_jc - 8), a block's channels at a time
// X keeps w in fp16's range: E is a running bound of the exponents of V's
// scales, kept like the running maximum of the scores, and p takes 2^15 (less
// where d is above 1) and d a power of two where it is below 2^-6.  The terms
// of w come from p = ph + pl and d in fp16 arithmetic: hi = ph d, lo = (ph d -
// hi) + pl d, whose first part a fused multiply-add leaves exact.  Terms end at
// 2^-24, so a w that is small beside the largest p times the largest d (at least 2^8)
// is off by 2^-32 of that rather than by 2^-22 of itself.  Blocks' scales far apart
// (2^10) would need a power of two for each block; that was built and took 16 columns
// of 65536 positions from 167 to 170 us, for values that f32 rows seldom hold.
//
// A code becomes a half by one AND/OR, (w & 0x000f) | 0x6400 = 1024 + n, and
// one addition that centres it: n - 8 (16 (n - 8) from a high nibble; for a key
// its channel of q takes 1/16).  The code's own bits are n 2^-24 as a subnormal
// half and would need neither, but results were then off by 2.4e-6 (3e-7 with
// centred codes).  Long chains in the accumulators cost bits as well (1.4e-6 over
// 65536 positions): a tile's products start from zero and are added in f32.
//
// Bound: 18 bytes for 32 values, each used by every head of the group; at the
// memory rate a scheduler has 3.1 lane slots a value of the cache, 1.5 for half2
// and integer instructions, which issue at half rate, and f32 arithmetic adds its
// time to the products'.  So it is bound by its instructions: 167 us for 16 columns
// of 65536 positions, 28 / 4 heads of 128 (3.6 TB/s, 56% of the measured copy rate;
// 180 us at 1860 MHz in a run of seconds, at the power limit); 64 ragged columns up
// to 2048 21 us (23 with the cache not in L2), 1 x 32768 14.7 us (16).  3 CTAs an SM
// with 168 registers: 4 with 128 took 184 us for 168.
//
// Work: the positions of all columns and heads form one list of units, kExtra
// for each (column, group), what its start and end cost, and one for each of
// its chunks of kChunk positions.  The list is cut into equal runs for the CTAs,
// whatever the lengths; a CTA that holds only part of a group's chunks leaves
// its partial sums in the workspace for a second kernel.  Each warp streams its
// own tiles of 32 positions through a ring of bulk copies.
constexpr int kWarps = 4, kThreads = 32 * kWarps, kChunk = kTile * kWarps;
constexpr int kStages = 2, kGroup = 8, kCtasPerSm = 3, kExtra = 1;
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
  int2* spans;                       // [column][sub]: first and last CTA
};

template <int NB>
struct Shape {
  static constexpr int kD = 32 * NB;
  static constexpr int kTileBytes = tile_bytes(NB), kQuantBytes = kTile * 16 * NB;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kPartFloats = kGroup * (kD + 2);
};

// Visible positions of a column: 0 for a length or slot outside the cache.
__device__ __forceinline__ int visible(const AttnQ40Args& a, int n, int slot) {
  return n > 0 && n <= a.c.max_seq && slot >= 0 && slot < a.c.n_slots ? n : 0;
}
__device__ __forceinline__ int slot_of(const AttnQ40Args& a, int col) {
  return a.slots ? a.slots[col] : col;
}
__device__ __forceinline__ int chunks_of(int len) { return (len + kChunk - 1) / kChunk; }
__device__ __forceinline__ int64_t units_of(int len) { return len ? chunks_of(len) + kExtra : 0; }
// The CTA whose run of the `total` units holds unit u: run i is
// [i total / n, (i + 1) total / n).
__device__ __forceinline__ int cta_of(int64_t u, int64_t total, int n) {
  return (int)(((u + 1) * n - 1) / total);
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// The same without an addend.
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ uint32_t bits(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
template <uint32_t MASK>
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t with) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "n"(MASK), "r"(with));
  return r;
}
__device__ __forceinline__ uint32_t codes_low(uint32_t w) {
  return bits(__hadd2(as_h2(and_or<0x000f000fu>(w, 0x64006400u)), as_h2(0xe408e408u)));  // -1032
}
__device__ __forceinline__ uint32_t codes_high(uint32_t w) {
  return bits(__hadd2(as_h2(and_or<0x00f000f0u>(w, 0x64006400u)), as_h2(0xe480e480u)));  // -1152
}
// V's scales that are all below 2^kSmall are raised by this power of two.
constexpr int kSmall = -6;
__device__ __forceinline__ int small_scales(int ev) { return max(0, kSmall - ev); }

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

// One CTA's share of one (column, group): chunks ch0 .. ch0 + take - 1.
struct Piece {
  int col, len, slot, sub, ch0, take;
};

// WITHHOLD: a test hook, the copies of one tile {column, tile} are never made.  It
// and the join's count of CTAs are arguments of their own: as members of AttnQ40Args
// they moved the registers that are spilled (16 x 65536 167 -> 179 us).
template <int NB, bool WITHHOLD>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    kv_q40_attention_kernel(const AttnQ40Args a, const int2 withheld) {
  using S = Shape<NB>;
  constexpr int D = S::kD;
  extern __shared__ __align__(128) unsigned char smem[];  // rings, then the warps' sums
  __shared__ __align__(8) uint64_t bars[kWarps][kStages];
  __shared__ uint4 qfrag[NB][2][32];
  __shared__ float qscale[kGroup];
  __shared__ float red_m[kWarps][kGroup], red_l[kWarps][kGroup];
  __shared__ int red_e[kWarps];
  __shared__ int64_t warp_sums[kWarps];
  __shared__ int64_t s_first;
  __shared__ int s_col, s_len, s_slot;
  __shared__ volatile int abort_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;

  pdl_trigger();  // the join kernel waits for this grid's end
  if (tid < kWarps * kStages) tc::bar_init(&bars[tid / kStages][tid % kStages], 1);
  if (tid == 0) {
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }

  // ---- this CTA's run of the chunk list: the list's length, then the column
  // that holds the run's first unit
  int64_t total = 0, before = 0, mine_units = 0;
  int my_len = 0, my_slot = 0;
  auto count = [&](int c0) {  // columns c0 + tid: units of those before, sum
    const int col = c0 + tid;
    my_slot = 0, my_len = 0;
    if (col < a.n_cols) {
      const int n = a.lengths[col];
      my_slot = slot_of(a, col);
      my_len = visible(a, n, my_slot);
      if (my_len != n && blockIdx.x == 0) atomicOr(&g_kv_error, kErrBadIndex);
    }
    mine_units = units_of(my_len) * a.subs;
    return block_scan(mine_units, &before, warp_sums);
  };
  for (int c0 = 0; c0 < a.n_cols; c0 += kThreads) total += count(c0);
  // columns that see nothing have no units; their rows are zero
  auto zero_rows = [&] {
    for (int c = blockIdx.x; c < a.n_cols; c += gridDim.x)
      if (visible(a, a.lengths[c], slot_of(a, c)) == 0)
        for (int i = tid; i < a.n_heads * D; i += kThreads) a.out[c * a.ldo + i] = 0.0f;
  };
  const int n_ctas = (int)min((int64_t)gridDim.x, total);
  if ((int)blockIdx.x >= n_ctas) {
    zero_rows();
    return;
  }
  const int64_t u0 = blockIdx.x * total / n_ctas, u1 = (blockIdx.x + 1) * total / n_ctas;
  {
    int64_t run = 0;
    for (int c0 = 0; run <= u0; c0 += kThreads) {
      // up to kThreads columns the counts are still there
      const int64_t sum = a.n_cols > kThreads ? count(c0) : total;
      if (run + before <= u0 && u0 < run + before + mine_units) {
        s_col = c0 + tid;
        s_len = my_len;
        s_slot = my_slot;
        s_first = run + before;
      }
      run += sum;
    }
  }
  __syncthreads();

  unsigned char* ring = smem + (size_t)warp * kStages * S::kStageBytes;
  float* sums = reinterpret_cast<float*>(smem + (size_t)kWarps * kStages * S::kStageBytes);
  uint32_t used = 0;  // tiles this warp has waited for: stage used % kStages
  uint32_t issued = 0;
  bool ok = true;

  // the run's part of a group from its unit r on; the units it takes
  auto cut = [&](Piece& x, int64_t r, int64_t u) {
    const int64_t n = min(units_of(x.len) - r, u1 - u);
    x.ch0 = (int)max(r - kExtra, (int64_t)0);
    x.take = (int)max(r + n - kExtra, (int64_t)0) - x.ch0;
    return n;
  };
  Piece p;
  p.col = s_col, p.len = s_len, p.slot = s_slot;
  int64_t group0 = s_first;  // the group's first unit
  {
    const int64_t each = units_of(p.len);
    p.sub = (int)((u0 - s_first) / each);
    group0 += p.sub * each;
  }
  int64_t u = u0 + cut(p, u0 - group0, u0);  // behind the piece
  if (p.take == 0) {  // the whole run lies before a group's first chunk
    zero_rows();
    return;
  }
  auto first_of = [&](const Piece& x) { return x.ch0 * kWarps + warp; };  // this warp's first tile
  auto tiles_end = [&](const Piece& x) {
    return min((x.ch0 + x.take) * kWarps, (x.len + kTile - 1) / kTile);
  };
  auto tiles_mine = [&](const Piece& x) {
    const int n = tiles_end(x) - first_of(x);
    return n > 0 ? (n + kWarps - 1) / kWarps : 0;
  };
  auto issue = [&](const Piece& x, int i) {  // lane 0: this warp's tile i of the piece
    unsigned char* st = ring + (issued % kStages) * S::kStageBytes;
    uint64_t* bar = &bars[warp][issued % kStages];
    if constexpr (WITHHOLD)
      if (x.col == withheld.x && first_of(x) + i * kWarps == withheld.y) return;
    const int64_t at = (first_tile(a.c, x.slot, x.sub % a.c.n_kv_heads) + first_of(x) + i * kWarps) * S::kTileBytes;
    tc::bar_expect_tx(bar, S::kStageBytes);
    tc::bulk_load(st, a.c.k + at, S::kTileBytes, bar);
    tc::bulk_load(st + S::kTileBytes, a.c.v + at, S::kTileBytes, bar);
  };
  auto start = [&](const Piece& x) {  // its first tiles
    for (int i = 0; i < min(tiles_mine(x), kStages); ++i) {
      if (lane == 0) issue(x, i);
      ++issued;
    }
  };
  float qx[2][NB];  // this warp's two heads of the coming piece's queries
  auto load_q = [&](const Piece& x) {
    const int kvh = x.sub % a.c.n_kv_heads, h0 = (x.sub / a.c.n_kv_heads) * kGroup;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int hh = warp * 2 + i;
        const int64_t head = (int64_t)kvh * a.group + h0 + hh;
        qx[i][b] = h0 + hh < a.group ? a.q[x.col * a.ldq + head * D + 32 * b + lane] : 0.0f;
      }
  };
  start(p);
  load_q(p);
  // The spans of the groups that start here, before the first wait: the join then
  // finds them also where one runs out.
  if (tid == kThreads - 1) {
    Piece x = p;
    for (int64_t at = group0, r = u;;) {
      const int chunks = chunks_of(x.len);
      if (x.ch0 == 0)  // only the last one can go on in other runs
        a.spans[(int64_t)x.col * a.subs + x.sub] =
            make_int2(blockIdx.x, x.take == chunks ? blockIdx.x : cta_of(at + kExtra + chunks - 1, total, n_ctas));
      if (r >= u1) break;
      if (++x.sub == a.subs) {
        x.sub = 0;
        do {
          ++x.col;
          x.len = visible(a, a.lengths[x.col], slot_of(a, x.col));
        } while (x.len == 0);
      }
      at = r;
      r += cut(x, 0, r);
      if (x.take == 0) break;
    }
  }

  while (true) {
    const int kvh = p.sub % a.c.n_kv_heads, h0 = (p.sub / a.c.n_kv_heads) * kGroup;
    const int n_here = min(kGroup, a.group - h0);  // heads of this group
    const int mine = tiles_mine(p), tile0 = first_of(p), len = p.len;
    // the next piece begins a group: of this column, or of the next with any
    Piece nx = p;
    int64_t behind = u;
    nx.take = 0;
    if (u < u1) {
      if (++nx.sub == a.subs) {
        nx.sub = 0;
        do {
          ++nx.col;
          nx.slot = slot_of(a, nx.col);
          nx.len = visible(a, a.lengths[nx.col], nx.slot);
        } while (nx.len == 0);
      }
      behind += cut(nx, 0, u);
    }
    const bool more = nx.take > 0;

    // ---- the group's queries as A operands (high and low terms), two heads a warp
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int hh = warp * 2 + i;
      float top = 0.0f;
#pragma unroll
      for (int b = 0; b < NB; ++b) top = fmaxf(top, fabsf(qx[i][b]));
      top = warp_max(top);
      // 2^-e brings the row's largest value into [2^14, 2^15)
      const int e = top > 0.0f ? min(max(((__float_as_int(top) >> 23) & 0xff) - 141, -120), 120) : 0;
      const bool high = lane >= 16;
      const int jj = lane & 15, tq = jj >> 2, el = jj & 3;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        // a high nibble stands for 16 (n - 8): its channel takes 1/16
        const float v = qx[i][b] * pow2f(-e) * (high ? 0.0625f : 1.0f);
        const __half hi = __float2half_rn(v);
        const __half lo = __float2half_rn(v - __half2float(hi));
        __half* dst = reinterpret_cast<__half*>(&qfrag[b][el & 1][hh * 4 + tq]) + (high ? 4 : 0) + (el >> 1);
        dst[0] = hi;
        dst[2] = lo;
      }
      if (lane == 0) qscale[hh] = pow2f(e) * a.scale;
    }
    __syncthreads();

    // running sums of head g: channels 4t + {0, 2}, {1, 3} of a block's halves
    float o[NB][4][2];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int s = 0; s < 4; ++s) o[b][s][0] = o[b][s][1] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    float ref = -INFINITY;  // weights are 2^(score - ref)
    int ev = -14;           // V's scales so far are below 2^ev
    const float qs = qscale[g];

    for (int i = 0; i < mine; ++i) {
      const uint32_t stage = used % kStages;
      uint64_t* bar = &bars[warp][stage];
      const uint32_t phase = (used / kStages) & 1;
      if (__any_sync(0xffffffffu, !tc::bar_try(bar, phase))) {
        ok = __all_sync(0xffffffffu, tc::bar_wait(bar, phase, &abort_flag, &g_kv_error));
        if (!ok) break;
      }
      ++used;
      unsigned char* st = ring + stage * S::kStageBytes;
      const unsigned char* kq = st;
      const unsigned char* vq = st + S::kTileBytes;
      uint32_t* kd = reinterpret_cast<uint32_t*>(st + S::kQuantBytes);
      uint32_t* vd = reinterpret_cast<uint32_t*>(st + S::kTileBytes + S::kQuantBytes);
      const int left = len - (tile0 + i * kWarps) * kTile;  // live positions of the tile
      if (left < kTile) {
        // rows past the end may hold anything: zero scales take them out
        if (lane >= left) {
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const int at = ((lane >> 1) * NB + b) * 2 + (lane & 1);
            reinterpret_cast<uint16_t*>(kd)[at] = reinterpret_cast<uint16_t*>(vd)[at] = 0;
          }
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
          lds_words<NB>(dk[j], kd + (4 * j + t) * NB);
          s[j][0] = s[j][1] = 0.0f;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint4 a0 = qfrag[b][0][lane], a1 = qfrag[b][1][lane];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t w = kw[j][b], w8 = w >> 8;
            float c[4];
            mma16816_first(c, a0, codes_low(w), codes_high(w));
            mma16816(c, a1, codes_low(w8), codes_high(w8));
            const float2 d = __half22float2(as_h2(dk[j][b]));
            s[j][0] = fmaf(d.x, c[0] + c[2], s[j][0]);
            s[j][1] = fmaf(d.y, c[1] + c[3], s[j][1]);
          }
        }
      }
      if (left < kTile) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (8 * j + 2 * t + e >= left) s[j][e] = -INFINITY;
      }
      float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])),
                       fmaxf(fmaxf(s[2][0], s[2][1]), fmaxf(s[3][0], s[3][1])));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      m = fmaxf(m, fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * qs);
      uint32_t dtop = 0;
#pragma unroll
      for (int w = 0; w < (NB + 1) / 2; ++w)
        if (lane + 32 * w < kTile / 2 * NB) dtop = __vmaxu2(dtop, vd[lane + 32 * w]);
      dtop = __reduce_max_sync(0xffffffffu, max(dtop >> 16, dtop & 0xffffu));
      const int eold = ev;
      ev = max(ev, (int)(dtop >> 10) - 14);
      const float rnew = (m == -INFINITY ? 0.0f : m) + (float)(max(ev, 0) - 15);
      const float corr = ex2(ref - rnew);
      const float down = corr * pow2f(small_scales(ev) - small_scales(eold));
      ref = rnew;
      __half2 ph[4], pl[4];
      float psum = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p0 = ex2(fmaf(s[j][0], qs, -rnew)), p1 = ex2(fmaf(s[j][1], qs, -rnew));
        psum += p0;
        psum += p1;
        split2(p0, p1, ph[j], pl[j]);
      }
      l = fmaf(l, corr, psum);

      // ---- output, a block's 32 channels at a time: keys 16 h + {2t, 2t+1, 2t+8,
      // 2t+9} of unit g
      uint32_t vw[4][NB], dv[4][NB];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        lds_words<NB>(vw[j], vq + (4 * j + t) * (32 * NB) + value_part(t, g) * (4 * NB));
        lds_words<NB>(dv[j], vd + (4 * j + t) * NB);
      }
      if (ev < kSmall) {
        const __half2 up = __float2half2_rn(pow2f(small_scales(ev)));
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int b = 0; b < NB; ++b) dv[j][b] = bits(__hmul2(as_h2(dv[j][b]), up));
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __half2 d = as_h2(dv[j][b]);
          const __half2 x = __hmul2(ph[j], d);
          hi[j] = bits(x);
          lo[j] = bits(__hfma2(pl[j], d, __hfma2(ph[j], d, __hneg2(x))));
        }
        float c[4][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 w4 = make_uint4(hi[2 * h], lo[2 * h], hi[2 * h + 1], lo[2 * h + 1]);
#pragma unroll
          for (int byte = 0; byte < 2; ++byte) {
            const uint32_t x0 = vw[2 * h][b] >> (8 * byte), x1 = vw[2 * h + 1][b] >> (8 * byte);
            // channels 2g + byte (low nibbles) and 2g + byte + 16 (high)
            if (h == 0) {
              mma16816_first(c[byte], w4, codes_low(x0), codes_low(x1));
              mma16816_first(c[2 + byte], w4, codes_high(x0), codes_high(x1));
            } else {
              mma16816(c[byte], w4, codes_low(x0), codes_low(x1));
              mma16816(c[2 + byte], w4, codes_high(x0), codes_high(x1));
            }
          }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          o[b][n][0] = fmaf(o[b][n][0], down, c[n][0] + c[n][2]);
          o[b][n][1] = fmaf(o[b][n][1], down, c[n][1] + c[n][3]);
        }
      }
      __syncwarp();
      if (i + kStages < mine) {
        if (lane == 0) issue(p, i + kStages);
        ++issued;
      }
    }
    // the next piece's copies and loads run while this one's sums are joined
    if (more && ok) {
      start(nx);
      load_q(nx);
    }

    // ---- join the warps' sums, in warp order
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) {
      red_m[warp][g] = ref;
      red_l[warp][g] = l;
    }
    if (lane == 0) red_e[warp] = small_scales(ev);
    const int warps_used = min(kWarps, tiles_end(p) - p.ch0 * kWarps);
    if (mine) {
      float* ro = sums + warp * (kGroup * D);  // [head][channel]
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // column 2t + e of the products: channels 2 (2t + e) + byte, + 16
          float2* to = reinterpret_cast<float2*>(ro + g * D + 32 * b + 4 * t + 2 * e);
          to[0] = make_float2(o[b][0][e], o[b][1][e]);
          to[8] = make_float2(o[b][2][e] * 0.0625f, o[b][3][e] * 0.0625f);
        }
    }
    ok = __syncthreads_and(ok);
    if (!ok) break;
    // 16 threads a head, D / 16 channels each
    const int h = tid / 16, chunks = chunks_of(len);
    if (h < n_here) {
      constexpr int C = D / 16;
      float mm = -INFINITY, ll = 0.0f, acc[C];
      for (int w = 0; w < warps_used; ++w) mm = fmaxf(mm, red_m[w][h]);
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] = 0.0f;
      for (int w = 0; w < warps_used; ++w) {
        const float f = ex2(red_m[w][h] - mm), fo = f * pow2f(-red_e[w]);
        ll = fmaf(red_l[w][h], f, ll);
        const float* from = sums + w * (kGroup * D) + h * D + tid % 16;
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] = fmaf(from[16 * c], fo, acc[c]);
      }
      if (p.take == chunks) {
        float* y = a.out + p.col * a.ldo + ((int64_t)kvh * a.group + h0 + h) * D + tid % 16;
#pragma unroll
        for (int c = 0; c < C; ++c) y[16 * c] = __fdiv_rn(acc[c], ll);
      } else {
        float* part = a.part + ((int64_t)blockIdx.x * 2 + (p.ch0 == 0 ? 1 : 0)) * S::kPartFloats;
#pragma unroll
        for (int c = 0; c < C; ++c) part[h * D + tid % 16 + 16 * c] = acc[c];
        if (tid % 16 == 0) {
          part[kGroup * D + h] = mm;
          part[kGroup * D + kGroup + h] = ll;
        }
      }
    }
    if (!more) break;
    u = behind;
    p = nx;
  }
  if (!ok) {
    // A wait ran out: the sums of weights among this run's partial sums become NaN,
    // so that nothing the workspace held before enters a result.
    if (tid < 2 * kGroup)
      a.part[((int64_t)blockIdx.x * 2 + tid / kGroup) * S::kPartFloats + kGroup * (D + 1) + tid % kGroup] =
          __int_as_float(0x7fc00000);
    // leave once this warp's own copies have landed or given up
    for (; used < issued; ++used) {
      const unsigned long long t0 = tc::now_ns();
      while (!tc::bar_try(&bars[warp][used % kStages], (used / kStages) & 1))
        if (tc::now_ns() - t0 > tc::kWaitNs) break;
    }
  }
  zero_rows();
}

// Joins the partial sums of a (column, group) whose chunks lie in more than
// one CTA's run.  A warp sums every kSlots-th partial of one head, then the
// warps' sums are joined in order.  HEADS heads a CTA: 1 where there are few
// groups and many partials of each, 8 where there are many groups.
template <int NB, int HEADS>
__global__ void __launch_bounds__(HEADS == 1 ? 1024 : 512)
    kv_q40_join_kernel(const AttnQ40Args a, const int n_ctas) {
  using S = Shape<NB>;
  constexpr int kJoinThreads = HEADS == 1 ? 1024 : 512, kJoinWarps = kJoinThreads / 32;
  constexpr int D = S::kD, kSlots = kJoinWarps / HEADS;
  __shared__ float acc_s[kJoinWarps][D], m_s[kJoinWarps], l_s[kJoinWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int col = blockIdx.x / a.subs, sub = blockIdx.x % a.subs;
  const int kvh = sub % a.c.n_kv_heads, h0 = (sub / a.c.n_kv_heads) * kGroup;
  const int len = visible(a, a.lengths[col], slot_of(a, col));
  pdl_wait();  // every CTA waits, so that this grid's end is also the first kernel's
  if (chunks_of(len) == 0) return;
  // whole in one CTA; the partial sums' indices stay within the workspace
  // whatever it holds
  const int2 span = __ldcg(a.spans + blockIdx.x);
  if (span.x < 0 || span.x >= span.y || span.y >= n_ctas) return;
  const int h = blockIdx.y * HEADS + warp % HEADS, slot = warp / HEADS;
  float m = -INFINITY, l = 0.0f, acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = 0.0f;
  if (h0 + h < a.group) {
#pragma unroll 4
    for (int i = span.x + slot; i <= span.y; i += kSlots) {
      // the first run ends with this group's start, the others begin inside it
      const float* p = a.part + ((int64_t)i * 2 + (i == span.x ? 1 : 0)) * S::kPartFloats;
      const float mi = __ldcg(p + kGroup * D + h), li = __ldcg(p + kGroup * D + kGroup + h);
      float x[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) x[b] = __ldcg(p + h * D + 32 * b + lane);
      const float top = fmaxf(m, mi), ref = top == -INFINITY ? 0.0f : top;
      const float f = ex2(m - ref), fi = ex2(mi - ref);
      m = top;
      l = fmaf(li, fi, l * f);
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[b] = fmaf(x[b], fi, acc[b] * f);
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) acc_s[warp][32 * b + lane] = acc[b];
  if (lane == 0) {
    m_s[warp] = m;
    l_s[warp] = l;
  }
  __syncthreads();
  for (int i = tid; i < HEADS * D; i += kJoinThreads) {
    const int hh = i / D, d = i % D, head = h0 + blockIdx.y * HEADS + hh;
    if (head >= a.group) continue;
    float mm = -INFINITY, ll = 0.0f, x = 0.0f;
    for (int s = 0; s < kSlots; ++s) mm = fmaxf(mm, m_s[s * HEADS + hh]);
    const float ref = mm == -INFINITY ? 0.0f : mm;
    for (int s = 0; s < kSlots; ++s) {
      const float f = ex2(m_s[s * HEADS + hh] - ref);
      ll = fmaf(l_s[s * HEADS + hh], f, ll);
      x = fmaf(acc_s[s * HEADS + hh][d], f, x);
    }
    a.out[col * a.ldo + ((int64_t)kvh * a.group + head) * D + d] = __fdiv_rn(x, ll);
  }
}

template <int NB>
constexpr size_t attention_smem() {
  return (size_t)kWarps * (kStages * Shape<NB>::kStageBytes + kGroup * Shape<NB>::kD * sizeof(float));
}

template <int NB, bool WITHHOLD>
cudaError_t launch_attention_q40(const AttnQ40Args& args, int n_ctas, int2 withheld, bool join,
                                 cudaStream_t st) {
  static DeviceOnce once;
  cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(kv_q40_attention_kernel<NB, WITHHOLD>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)attention_smem<NB>());
  });
  if (e != cudaSuccess) return e;
  e = launch(kv_q40_attention_kernel<NB, WITHHOLD>, dim3(n_ctas), dim3(kThreads),
             attention_smem<NB>(), st, false, args, withheld);
  if (e != cudaSuccess || !join) return e;
  // One head a CTA of the join where a group has many partial sums, 8 where there are
  // many groups.  Us of both kernels, one / 8, and partial sums a group, 28 / 4 heads
  // of 128: 1 column of 32768 14.5 / 36.5 (111), 1 of 4096 9.0 / 15.3 (32), 8 of 8192
  // 22.3 / 22.4 (14), 12 of 8192 28.4 / 27.3 (9), 8 of 1024 13.1 / 11.8 (8), 64 of 1024
  // 41.0 / 22.1 (2); 14 / 2 of 64: 16 of 8192 17.1 / 16.8 (14), 24 of 2048 12.8 / 11.8
  // (9), 8 of 1024 8.2 / 8.5 (8); 40 / 8 of 128: 4 of 8192 20.9 / 21.7 (14); 5 / 1 of
  // 64: 16 of 8192 10.8 / 16.0 (28).
  const unsigned groups = (unsigned)(args.n_cols * args.subs);
  if ((unsigned)n_ctas / 12 >= groups)
    return launch(kv_q40_join_kernel<NB, 1>, dim3(groups, kGroup), dim3(1024), 0, st, use_pdl(),
                  args, n_ctas);
  return launch(kv_q40_join_kernel<NB, kGroup>, dim3(groups), dim3(512), 0, st, use_pdl(), args,
                n_ctas);
}

// CTAs of the attention kernel: what the SMs hold at once, or the most chunks
// there can be.
int attention_ctas(int n_cols, int subs, int max_seq) {
  const int64_t units = (int64_t)n_cols * subs * ((max_seq + kChunk - 1) / kChunk);
  const int64_t most = (int64_t)kCtasPerSm * sm_count();
  return (int)(units < most ? units : most);
}
// The workspace: partial sums, then the groups' spans.
size_t part_bytes(int n_cols, int subs, int max_seq, int head_dim) {
  return (size_t)attention_ctas(n_cols, subs, max_seq) * 2 * kGroup * (head_dim + 2) * sizeof(float);
}
size_t workspace_need(int n_cols, int subs, int max_seq, int head_dim) {
  return part_bytes(n_cols, subs, max_seq, head_dim) + (size_t)n_cols * subs * sizeof(int2);
}

bool shape_ok(int n_layers, int n_slots, int max_seq, int n_kv_heads, int head_dim) {
  return n_layers > 0 && n_slots > 0 && max_seq > 0 && max_seq <= INT_MAX - 256 && n_kv_heads > 0 &&
         head_dim > 0 && head_dim % 32 == 0 && head_dim <= 32 * kMaxBlocks;
}

// A buffer's bytes fit 62 bits, so that no offset wraps.
bool size_ok(int n_layers, int n_slots, int max_seq, int n_kv_heads, int head_dim) {
  const unsigned __int128 tiles = (unsigned __int128)((uint64_t)n_layers * (uint64_t)n_slots) *
                                  (uint64_t)n_kv_heads * (uint64_t)tiles_of(max_seq);
  return tiles < ((uint64_t)1 << 62) / tile_bytes(head_dim / 32);
}

// The status of a cache argument; on success its layer `layer`.
int check_cache(const std::string& api, const dqmk_kv_q40* kv, int layer, Plane* out) {
  if (!kv || !kv->keys_dev || !kv->values_dev) return fail(DQMK_ERR_INVALID, api + ": null pointer");
  if (kv->n_layers <= 0 || kv->n_slots <= 0 || kv->max_seq <= 0 || kv->n_kv_heads <= 0)
    return fail(DQMK_ERR_INVALID, api + ": invalid cache shape");
  if (!shape_ok(kv->n_layers, kv->n_slots, kv->max_seq, kv->n_kv_heads, kv->head_dim))
    return fail(DQMK_ERR_UNSUPPORTED, api + ": head_dim must be a multiple of 32 of at most 128");
  if (!size_ok(kv->n_layers, kv->n_slots, kv->max_seq, kv->n_kv_heads, kv->head_dim))
    return fail(DQMK_ERR_UNSUPPORTED, api + ": cache too large");
  if ((reinterpret_cast<uintptr_t>(kv->keys_dev) | reinterpret_cast<uintptr_t>(kv->values_dev)) & 15u)
    return fail(DQMK_ERR_INVALID, api + ": KV cache must be 16-byte aligned");
  if (layer < 0 || layer >= kv->n_layers) return fail(DQMK_ERR_RANGE, api + ": layer out of range");
  const int64_t tiles = tiles_of(kv->max_seq);
  const int nb = kv->head_dim / 32;
  const int64_t at = (int64_t)layer * kv->n_slots * kv->n_kv_heads * tiles * tile_bytes(nb);
  out->k = static_cast<unsigned char*>(kv->keys_dev) + at;
  out->v = static_cast<unsigned char*>(kv->values_dev) + at;
  out->n_slots = kv->n_slots, out->max_seq = kv->max_seq, out->n_kv_heads = kv->n_kv_heads;
  out->nb = nb, out->tiles = tiles;
  return DQMK_OK;
}

template <int NB, int TOK, bool VEC>
cudaError_t launch_rows(bool write, const RowsArgs& a, cudaStream_t st) {
  constexpr int RT = TOK > 1 ? kReadTokens : 1, WT = TOK > 1 ? kWriteTokens : 1;
  const int64_t n = a.n_tokens;
  const dim3 block(kRowThreads);
  return write ? launch(kv_q40_write_kernel<NB, WT, VEC>, dim3((unsigned)((n + WT - 1) / WT)), block, 0, st, false, a)
               : launch(kv_q40_read_kernel<NB, RT, VEC>, dim3((unsigned)((n + RT - 1) / RT)), block, 0, st, false, a);
}
template <int NB>
cudaError_t launch_rows(bool write, bool vec, const RowsArgs& a, cudaStream_t st) {
  // Several tokens a CTA once they fill the SMs.  Write and read, 4 heads of 128,
  // one / several, us, rows in L2: 148 tokens 4.3 / 7.0, 888 6.3 / 7.3, 1184 7.7 / 7.8,
  // 1480 9.3 / 8.6, 8191 32.5 / 21.0 (29 with rows from memory)
  if (a.n_tokens >= 8 * sm_count())
    return vec ? launch_rows<NB, 8, true>(write, a, st) : launch_rows<NB, 8, false>(write, a, st);
  return vec ? launch_rows<NB, 1, true>(write, a, st) : launch_rows<NB, 1, false>(write, a, st);
}
cudaError_t launch_rows(bool write, bool vec, const RowsArgs& a, cudaStream_t st) {
  switch (a.c.nb) {
    case 1: return launch_rows<1>(write, vec, a, st);
    case 2: return launch_rows<2>(write, vec, a, st);
    case 3: return launch_rows<3>(write, vec, a, st);
    default: return launch_rows<4>(write, vec, a, st);
  }
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
  if (!shape_ok(n_layers, n_slots, max_seq, n_kv_heads, head_dim) ||
      !size_ok(n_layers, n_slots, max_seq, n_kv_heads, head_dim))
    return 0;
  return (size_t)n_layers * n_slots * n_kv_heads * tiles_of(max_seq) * tile_bytes(head_dim / 32);
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
  DQMK_CUDA_RET(api.c_str(), launch_rows(true, vec_rows(k, v, ldk, ldv), a, static_cast<cudaStream_t>(stream)));
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
  DQMK_CUDA_RET(api.c_str(), launch_rows(false, vec_rows(k, v, ldk, ldv), a, static_cast<cudaStream_t>(stream)));
  return DQMK_OK;
}

extern "C" size_t dqmk_kv_q40_attention_workspace(const dqmk_kv_q40* kv, int n_cols, int n_heads) {
  if (!kv || !shape_ok(kv->n_layers, kv->n_slots, kv->max_seq, kv->n_kv_heads, kv->head_dim) ||
      n_cols <= 0 || n_heads <= 0 || n_heads % kv->n_kv_heads != 0)
    return 0;
  const int subs = kv->n_kv_heads * ((n_heads / kv->n_kv_heads + kGroup - 1) / kGroup);
  return workspace_need(n_cols, subs, kv->max_seq, kv->head_dim);
}

namespace {

int attention_call(const dqmk_kv_q40* kv, int layer, const float* q, int64_t ldq, const int* slots,
                   const int* lengths, int n_cols, int n_heads, float* out, int64_t ldo,
                   void* workspace, size_t workspace_bytes, int withhold_col, int withhold_tile,
                   void* stream) {
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
  if (width > INT_MAX - kThreads) return fail(DQMK_ERR_UNSUPPORTED, api + ": too many heads");
  if (subs * n_cols > INT_MAX) return fail(DQMK_ERR_UNSUPPORTED, api + ": too many columns");
  a.subs = (int)subs;
  const size_t need = workspace_need(n_cols, a.subs, kv->max_seq, kv->head_dim);
  if (workspace_bytes < need)
    return fail(DQMK_ERR_INVALID, api + ": workspace of " + std::to_string(workspace_bytes) +
                                      " bytes, needs " + std::to_string(need));
  a.q = q, a.ldq = ldq, a.out = out, a.ldo = ldo;
  a.lengths = lengths, a.slots = slots, a.n_cols = n_cols, a.n_heads = n_heads;
  a.scale = kLog2e / sqrtf((float)kv->head_dim);
  a.part = static_cast<float*>(workspace);
  a.spans = reinterpret_cast<int2*>(static_cast<char*>(workspace) +
                                    part_bytes(n_cols, a.subs, kv->max_seq, kv->head_dim));
  const int n_ctas = attention_ctas(n_cols, a.subs, kv->max_seq);
  const bool join = kv->max_seq > kChunk;  // else every run ends with a whole group
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  const int2 withheld = make_int2(withhold_col, withhold_tile);
  auto run = [&](auto nb) {
    constexpr int NB = decltype(nb)::value;
    return withhold_col < 0 ? launch_attention_q40<NB, false>(a, n_ctas, withheld, join, st)
                            : launch_attention_q40<NB, true>(a, n_ctas, withheld, join, st);
  };
  switch (a.c.nb) {
    case 1: e = run(std::integral_constant<int, 1>()); break;
    case 2: e = run(std::integral_constant<int, 2>()); break;
    case 3: e = run(std::integral_constant<int, 3>()); break;
    default: e = run(std::integral_constant<int, 4>()); break;
  }
  DQMK_CUDA_RET(api.c_str(), e);
  return DQMK_OK;
}

}  // namespace

extern "C" int dqmk_kv_q40_attention(const dqmk_kv_q40* kv, int layer, const float* q, int64_t ldq,
                                     const int* slots, const int* lengths, int n_cols, int n_heads,
                                     float* out, int64_t ldo, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  return attention_call(kv, layer, q, ldq, slots, lengths, n_cols, n_heads, out, ldo, workspace,
                        workspace_bytes, -1, -1, stream);
}

extern "C" int dqmk_kv_q40_attention_withhold_tile(const dqmk_kv_q40* kv, int layer, const float* q,
                                                   int64_t ldq, const int* slots, const int* lengths,
                                                   int n_cols, int n_heads, float* out, int64_t ldo,
                                                   void* workspace, size_t workspace_bytes, int column,
                                                   int tile, void* stream) {
  return attention_call(kv, layer, q, ldq, slots, lengths, n_cols, n_heads, out, ldo, workspace,
                        workspace_bytes, column, tile, stream);
}
