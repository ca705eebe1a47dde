// Attention of few queries a key head over long keys: one new token of a sequence over its cache, or of an image's text over the
// encoder's states.
//
//   s_ij = scale * q_i . k_j over the keys j that query i sees,   o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i)
//
// A unit is a tile of up to 16 (query, head) rows of a sequence that share a key head, with all the keys they see, in steps of 32 keys (16
// in 16 bits).  The steps of all units lie on one line that is cut into equal pieces, one a block, and those again, one a warp, whatever the
// lengths are: long sequences are spread over the GPU as evenly as many short ones.  A warp keeps the running maximum and sum and the
// 16 x 64 accumulator in registers; it writes a unit that lies in its piece whole, and of one that does not (at most the first and the last)
// its part.  Parts of a block's warps are added up in the block, those of several blocks by the join kernel behind it, both in the order of the
// keys.  With short contexts the line is cut between blocks at the units' ends and there is no second kernel; where units are many or short it
// is cut so between warps too, and nothing is joined.
//
// Each warp has a ring of steps in shared memory of its own, filled by asynchronous copies two steps ahead (no barriers).  Packed rows are
// copied as they are, and two codes become two levels in fp16 on the way into the tensor instructions with one read: their byte (or 4 or 6 bits) is
// moved into bits 8-15 of a table address by one byte permute or shift, the table lying at shared address 64 KB with copies a lane, so that reads
// have no bank conflicts.  Scale and center never touch the levels:
//   q . k_j = scale_j (q . level_j) + center_j sum(q),    sum_j p_j v_j = sum_j (p_j scale_j) level_j + sum_j p_j center_j
// Rounded to fp16 a level is off by the same amount wherever its code stands, which would add up over a long context; its copies are rounded up or
// down in the share of its position between the two, and lanes serve different keys, so that it averages out (error against 64 bits over 65 521
// keys of 3 bits, relative to the output: 3.9e-4 with all copies rounded alike, 2.1e-4 so, which is the output's own rounding).  p_j scale_j is
// rounded to fp16 as p_j is without scales.  Pairs of keys' values are a byte as it is stored; of values, which have to be paired along the
// keys, the codes of two keys are interleaved.  The order of a head's values in a product is free, and so is that of keys: each lane takes values
// that lie side by side.
//
// 1 token over 64 contexts of up to 4096, 12 heads over 4 key heads, 4 bits: 29.3 us, 25 % of the copy bandwidth (47 MB); over two of 65 521 in 3
// bits, 12 heads: 52.7 us.  Two things take that time, in about equal parts for the first: launches, set-up and the join, during which little is
// issued (0.42 a scheduler and cycle over the whole call), and 660 instructions a step and warp (32 keys, 16 rows or fewer; counted over the call, by
// pipe 214 integer, 240 fp32, 103 loads and stores).  Table reads, their addresses, row reads and the interleaving of values are a quarter of
// them; of the fp32 pipe's, scores, exponents and scales account for some 90.
// Few steps: set-up and latency, 1 token over 333: 9.0 us.
#pragma once
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>
#include "ptx.cuh"
#include "f32x2.cuh"
#include "attention.cuh"
#include "kv_cache.cuh"

namespace arcq {

struct AttendView {                     // keys or values
  const uint8_t* rows;
  const __half2* stats;                 // [pages, heads, page]; null in 16 bits
  long long block_stride, token_stride, head_stride;     // bytes; a block is a page, or an image's states
};
struct AttendParams {
  AttendView k, v;
  const float* codebooks;               // [2, 2^bits]: keys, values
  const int* table;                     // [batch, table_width]; null: block = sequence
  int table_width, page_shift, pages;
  const int* lengths;                   // keys of a sequence; null: max_keys each
  const uint8_t* mask;                  // [batch, max_keys], 0: not seen; null: all are
  long long mask_stride;
  int max_keys;
  const void* q;
  long long q_batch, q_token, q_head;   // values; q_batch is not used with starts
  long long q_rows;                     // tokens of q (with starts)
  const int* starts;                    // [batch + 1]; null: max_new queries each
  int max_new;
  int causal;
  int q_bf16;
  float scale_log2;                     // scale / ln 2
  void* out;                            // [tokens, heads, 64]
  int heads, kv_heads, group, tiles, splits, batch;
  void* workspace;                      // split_attention_kernel
  int part_rows;                        // of a part: 16, or all rows that there can be
  int whole_units;                      // 1: each block has whole units, 2: each warp
  uint32_t poll_limit;                  // tile_attention.cuh
  int* status;
};

// What a block has to know of its sequence
struct AttendSequence {
  int keys, first_row, queries;         // queries that are there: at most max_new
  int all_queries;                      // the sequence's own count, which the causal mask goes by
};
__device__ __forceinline__ AttendSequence attend_sequence(const AttendParams& p, int b) {
  AttendSequence s;
  s.keys = p.lengths != nullptr ? min(max(p.lengths[b], 0), p.max_keys) : p.max_keys;
  if (p.starts != nullptr) {
    const int from = p.starts[b], to = p.starts[b + 1];
    s.first_row = from;
    s.all_queries = max(to - from, 0);
    s.queries = from < 0 ? 0 : static_cast<int>(min(static_cast<long long>(min(s.all_queries, p.max_new)), max(p.q_rows - from, 0ll)));
  } else {
    s.first_row = b * p.max_new;
    s.all_queries = s.queries = p.max_new;
  }
  return s;
}
__device__ __forceinline__ const uint16_t* attend_query(const AttendParams& p, const AttendSequence& s, int b, int i, int head) {
  const long long at = p.starts != nullptr ? (static_cast<long long>(s.first_row) + i) * p.q_token : b * p.q_batch + i * p.q_token;
  return static_cast<const uint16_t*>(p.q) + at + head * p.q_head;
}

template <typename E> __device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the same without an accumulator
template <typename E> __device__ __forceinline__ void mma_16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16816_first<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
template <> __device__ __forceinline__ void mma_16816_first<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t half2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// A row of bf16 queries (or a lane's part of it, with `top` the whole row's largest magnitude) as fp16: times the power of two that brings
// the largest value to 2^13..2^14, so that fp16 holds all that counts exactly.  Returns the factor that undoes it.
__device__ __forceinline__ float bf16_top(const uint32_t* w, int n) {
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < n; ++j) {
    float x, y;
    unpack2(sixteen_to_pair<__nv_bfloat16>(w[j]), x, y);
    top = fmaxf(top, fmaxf(fabsf(x), fabsf(y)));
  }
  return top;
}
__device__ __forceinline__ float bf16_to_half(uint32_t* w, int n, float top) {
  const int e = (__float_as_int(top) >> 23) - 127;
  const int up = top > 0.0f && e < 128 ? min(13 - e, 126) : 0;                     // -114 at least; f and the factor are normal numbers
  const float f = __int_as_float((up + 127) << 23);
#pragma unroll
  for (int j = 0; j < n; ++j) w[j] = pair_to_sixteen<__half>(mul2(sixteen_to_pair<__nv_bfloat16>(w[j]), pack2(f, f)));
  return __int_as_float((127 - up) << 23);
}

constexpr int kSplitWarps = 12, kSplitThreads = kSplitWarps * 32, kSplitRows = 16, kSplitStages = 3;
constexpr uint32_t kPairTableBytes = 256 * 32 * 4;                  // [byte][lane]

// [byte][lane]: the levels of the byte's two codes, low nibble first
__device__ __forceinline__ void fill_pair_table(uint32_t table, const float* levels, int count, int tid, int threads) {
  for (int i = tid; i < 256 * 8; i += threads) {
    const int byte = i >> 3;
    const __half2 h = __halves2half2(__float2half_rn(__ldg(levels + min(byte & 15, count - 1))), __float2half_rn(__ldg(levels + min(byte >> 4, count - 1))));
    const uint32_t w = *reinterpret_cast<const uint32_t*>(&h);
    sts128(table + byte * 128 + (i & 7) * 16, w, w, w, w);
  }
}
// pairs of levels of the four bytes of w; `table` includes the lane's column
__device__ __forceinline__ void pair_levels(uint32_t table, uint32_t w, uint32_t (&pairs)[4]) {
  pairs[0] = lds_const_u32(table + ((w << 7) & 0x7F80u));
  pairs[1] = lds_const_u32(table + ((w >> 1) & 0x7F80u));
  pairs[2] = lds_const_u32(table + ((w >> 9) & 0x7F80u));
  pairs[3] = lds_const_u32(table + ((w >> 17) & 0x7F80u));
}

// The same in fp32, for values: [byte][lane & 15], `table` with the lane's column.  Rounded to fp16 a level is off by the same amount in every
// key that has its code, which adds up over a long context; one rounding of center + scale * level does not.
__device__ __forceinline__ void fill_pair_table_f32(uint32_t table, const float* levels, int count, int tid, int threads) {
  for (int i = tid; i < 256 * 8; i += threads) {
    const int byte = i >> 3;
    const uint32_t lo = __float_as_uint(__ldg(levels + min(byte & 15, count - 1))), hi = __float_as_uint(__ldg(levels + min(byte >> 4, count - 1)));
    sts128(table + byte * 128 + (i & 7) * 16, lo, hi, lo, hi);
  }
}
__device__ __forceinline__ f32x2 lds_const_pair(uint32_t addr) {
  f32x2 v;
  asm("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void pair_levels_f32(uint32_t table, uint32_t w, f32x2 (&pairs)[4]) {
  pairs[0] = lds_const_pair(table + ((w << 7) & 0x7F80u));
  pairs[1] = lds_const_pair(table + ((w >> 1) & 0x7F80u));
  pairs[2] = lds_const_pair(table + ((w >> 9) & 0x7F80u));
  pairs[3] = lds_const_pair(table + ((w >> 17) & 0x7F80u));
}

// ---------------------------------------------------------------- shared memory of split_attention_kernel
// Packed: a table at shared address 64 KB, 256 bytes for each pair of codes: 32 copies of its levels for keys, 32 for values (fp16); the warps'
// rings below and above.
constexpr uint32_t kSplitTable = 0x10000, kSplitTableEnd = 0x20000;
template <int BITS> struct SplitStep {
  static constexpr int kKeys = BITS == 16 ? 16 : 32;
  static constexpr uint32_t kRow = BITS == 16 ? 128 : 8 * BITS;
  static constexpr uint32_t kPad = BITS == 16 ? 0 : 32;                           // behind each 8 rows, so that reads have no bank conflicts
  static constexpr uint32_t kRows = kKeys * kRow + kKeys / 8 * kPad;              // keys, or values
  static constexpr uint32_t kStats = BITS == 16 ? 0 : 4 * kKeys;                  // likewise
  static constexpr uint32_t kBytes = 2 * (kRows + kStats);
  static constexpr uint32_t kRing = kSplitStages * kBytes;
};
// `base`: where the block's shared memory starts; rings of warps that do not fit below the table lie above it
template <int BITS> __host__ __device__ constexpr uint32_t split_ring(uint32_t base, int warp) {
  const uint32_t ring = SplitStep<BITS>::kRing;
  if (BITS == 16) return base + warp * ring;
  const int below = static_cast<int>((kSplitTable - base) / ring);
  return warp < below ? base + warp * ring : kSplitTableEnd + (warp - below) * ring;
}
// where the rings and the table end for a base of at most kSplitBase (16 bits: relative to it); the warps' parts lie behind
constexpr uint32_t kSplitBase = 8192;
template <int BITS> __host__ __device__ constexpr uint32_t split_parts() {
  const uint32_t end = split_ring<BITS>(kSplitBase, kSplitWarps);
  return BITS == 16 ? kSplitWarps * SplitStep<16>::kRing : end < kSplitTableEnd ? kSplitTableEnd : end;
}
// A level in fp16, rounded up in a share of the copies that is the position between its neighbours: the copies of lanes 4g + c, low and high,
// serve different keys (values) or parts of a head (keys), over which the roundings then average out.
// `sixteenths` of the way from one neighbour to the next is where rounding up begins.  Low and high of c = 0 .. 3 have 7 and 9, 5 and 11, 3 and 13, 1 and
// 15: a pair is off to neither side on average, and the first keys of a context, which have c = 0, are rounded almost to the nearest.  Error against
// 64 bits in 4 bits and fp16, relative to the output, over 1, 8, 32 and 333 keys:
// 2.8, 3.3, 3.2, 2.4e-4 (the output's rounding alone: 2.1e-4); with shares rising from 1 for c = 0 to 15 for c = 3 6.1, 5.6, 3.4, 2.3e-4.
__device__ __forceinline__ __half dithered_level(float x, int sixteenths) {
  const __half down = __float2half_rd(x), up = __float2half_ru(x);
  const float a = __half2float(down), b = __half2float(up);
  return (x - a) * 16.0f > (b - a) * sixteenths ? up : down;
}
// Entry i of the table: codes i & (levels - 1) and i >> BITS.
template <int BITS> __device__ __forceinline__ void fill_split_table(const float* codebooks, int tid, int threads) {
  constexpr int LEVELS = 1 << BITS;
  for (int i = tid; i < 2 * LEVELS * LEVELS; i += threads) {
    const int entry = i >> 1, values = i & 1;
    const float lo = __ldg(codebooks + values * LEVELS + (entry & (LEVELS - 1))), hi = __ldg(codebooks + values * LEVELS + (entry >> BITS));
    uint32_t w[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const __half2 h = __halves2half2(dithered_level(lo, 7 - 2 * c), dithered_level(hi, 9 + 2 * c));
      w[c] = *reinterpret_cast<const uint32_t*>(&h);
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) sts128(kSplitTable + entry * 256 + values * 128 + ((r + entry) & 7) * 16, w[0], w[1], w[2], w[3]);
  }
}
// Address of entry I of the four whose numbers lie side by side in x (2 * BITS bits each); `column` is in the low byte, and the table's.
template <int BITS, int I> __device__ __forceinline__ uint32_t table_address(uint32_t x, uint32_t column) {
  if (BITS == 4) return __byte_perm(x, column, 0x7604 | (I << 4));
  constexpr int at = 2 * BITS * I;
  constexpr uint32_t mask = ((1u << (2 * BITS)) - 1) << 8;
  return ((at <= 8 ? x << (at <= 8 ? 8 - at : 0) : x >> (at > 8 ? at - 8 : 0)) & mask) | column;
}

// ---------------------------------------------------------------- units and their line
// KEYS: of a step
struct SplitUnit {
  int b, kvh, tile;
  AttendSequence seq;
  int rows, keys, steps;
};
__device__ __forceinline__ int split_tiles(const AttendParams& p, const AttendSequence& s) {
  return static_cast<int>((static_cast<long long>(s.queries) * p.group + kSplitRows - 1) / kSplitRows);
}
__device__ __forceinline__ int split_rows(const AttendParams& p, const AttendSequence& s, int tile) {
  return static_cast<int>(min(static_cast<long long>(s.queries) * p.group - static_cast<long long>(tile) * kSplitRows, static_cast<long long>(kSplitRows)));
}
template <int KEYS> __device__ __forceinline__ void split_tile(const AttendParams& p, SplitUnit& u) {
  u.rows = split_rows(p, u.seq, u.tile);
  u.keys = u.seq.keys;
  if (p.causal) u.keys = min(u.keys, max(u.seq.keys - u.seq.all_queries + (u.tile * kSplitRows + u.rows - 1) / p.group + 1, 0));
  u.steps = max((u.keys + KEYS - 1) / KEYS, 1);                                    // without keys a step, in which nothing is seen
}
// steps of all units of a sequence and key head
template <int KEYS> __device__ __forceinline__ int split_head_steps(const AttendParams& p, const AttendSequence& seq) {
  SplitUnit u;
  u.seq = seq;
  const int tiles = split_tiles(p, u.seq);
  int n = 0;
  for (u.tile = 0; u.tile < tiles; ++u.tile) {
    split_tile<KEYS>(p, u);
    n += u.steps;
  }
  return n;
}
// The unit after (b, kvh, tile); behind the last one: b = batch.  What a kernel keeps of a unit while it works on it is little.
template <int KEYS> __device__ __forceinline__ SplitUnit split_next(const AttendParams& p, int b, int kvh, int tile) {
  SplitUnit u;
  u.b = b;
  u.kvh = kvh;
  u.tile = tile + 1;
  u.seq = attend_sequence(p, b);
  if (u.tile >= split_tiles(p, u.seq)) {
    u.tile = 0;
    if (++u.kvh == p.kv_heads) {
      u.kvh = 0;
      while (++u.b < p.batch) {
        u.seq = attend_sequence(p, u.b);
        if (u.seq.queries > 0) break;
      }
      if (u.b >= p.batch) return u;
    }
  }
  split_tile<KEYS>(p, u);
  return u;
}
// The line: each of a block's threads has a share of the sequences, `mine` steps, with `before` steps before them.  Where all sequences are alike
// `mine` is a sequence's.  (The host keeps the line below 2^30 steps.)
template <int KEYS> struct SplitLine {
  int share, total, mine, before;
  bool alike;
  // whole block; of_warps: shared memory for a number a warp
  __device__ __forceinline__ SplitLine(const AttendParams& p, int* of_warps) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    alike = p.lengths == nullptr && p.starts == nullptr;
    share = (p.batch + kSplitThreads - 1) / kSplitThreads;
    if (alike) {
      mine = split_head_steps<KEYS>(p, attend_sequence(p, 0)) * p.kv_heads;
      total = mine * p.batch;
      before = 0;
      return;
    }
    mine = 0;
    for (int b = tid * share; b < min((tid + 1) * share, p.batch); ++b) mine += split_head_steps<KEYS>(p, attend_sequence(p, b)) * p.kv_heads;
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 31) of_warps[warp] = sum;
    __syncthreads();
    total = 0;
    before = sum - mine;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) {
      const int n = of_warps[w];
      if (w < warp) before += n;
      total += n;
    }
  }
  // Whose share step x(i) is in, and the steps before that share; for locate, behind a barrier.
  template <typename X> __device__ __forceinline__ void find(int count, X x, int2* found) const {
    if (alike || mine == 0) return;
    for (int i = 0; i < count; ++i) {
      const int v = x(i) - before;
      if (v >= 0 && v < mine) found[i] = make_int2(threadIdx.x, before);
    }
  }
  // the unit that step x is in, and the unit's first step
  __device__ __forceinline__ SplitUnit locate(const AttendParams& p, int x, const int2* found, int& at) const {
    SplitUnit u;
    int of_head;
    if (alike) {
      u.b = x / mine;
      at = u.b * mine;
      u.seq = attend_sequence(p, u.b);
      of_head = mine / p.kv_heads;
    } else {
      u.b = found->x * share;
      at = found->y;
      for (;; ++u.b) {
        u.seq = attend_sequence(p, u.b);
        of_head = split_head_steps<KEYS>(p, u.seq);
        if (at + of_head * p.kv_heads > x) break;
        at += of_head * p.kv_heads;
      }
    }
    u.kvh = (x - at) / max(of_head, 1);
    at += u.kvh * of_head;
    for (u.tile = 0;; ++u.tile) {
      split_tile<KEYS>(p, u);
      if (at + u.steps > x) break;
      at += u.steps;
    }
    return u;
  }
};

// A part of a unit: for each of its rows 64 outputs, maximum and sum.  A warp has two of them (of a unit that began before its piece, and of one
// that goes on behind it), in shared memory where they fit, and so has a block, in the workspace: a header, a record for each unit, the blocks'
// parts, and the warps' where shared memory is too small.
struct SplitHeader {
  int piece, unused[3];                                                           // steps of a block
};
struct SplitRecord {
  int start, steps, whole, unused;
};
constexpr int kSplitPartRow = 68, kSplitSharedRows = 8;                            // rows of parts in shared memory
constexpr uint32_t kSplitSharedParts = 2 * kSplitWarps * kSplitSharedRows * kSplitPartRow * 4;
__host__ __device__ inline long long split_units(const AttendParams& p) { return static_cast<long long>(p.batch) * p.kv_heads * p.tiles; }
__host__ __device__ inline long long split_workspace(const AttendParams& p, int blocks) {
  const long long part = static_cast<long long>(p.part_rows) * kSplitPartRow * 4;
  return static_cast<long long>(sizeof(SplitHeader)) + split_units(p) * sizeof(SplitRecord) +
         2ll * blocks * part * (p.part_rows > kSplitSharedRows ? 1 + kSplitWarps : 1);
}
__device__ __forceinline__ SplitRecord* split_records(const AttendParams& p) {
  return reinterpret_cast<SplitRecord*>(static_cast<uint8_t*>(p.workspace) + sizeof(SplitHeader));
}
__device__ __forceinline__ float* split_part(const AttendParams& p, long long slot) {
  return reinterpret_cast<float*>(split_records(p) + split_units(p)) + slot * p.part_rows * kSplitPartRow;
}
// The parts of one unit added up in the order of the keys, four values of a row a thread (the first rows * 16 threads).  next(i): part i.
template <typename Next> __device__ __forceinline__ float4 add_parts(int count, int row, int column, float& top, float& sum, Next next) {
  top = __int_as_float(0xff800000);
#pragma unroll 4
  for (int i = 0; i < count; ++i) top = fmaxf(top, next(i)[row * kSplitPartRow + 64]);
  const float base = top == __int_as_float(0xff800000) ? 0.0f : top;
  sum = 0.0f;
  float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 4
  for (int i = 0; i < count; ++i) {
    const float* const part = next(i) + row * kSplitPartRow;
    const float2 ts = *reinterpret_cast<const float2*>(part + 64);
    const float4 x = *reinterpret_cast<const float4*>(part + 4 * column);
    const float f = exp2_approx(ts.x - base);
    sum += ts.y * f;
    o = make_float4(o.x + x.x * f, o.y + x.y * f, o.z + x.z * f, o.w + x.w * f);
  }
  return o;
}
// a query that sees no key: zeros; NaN stays NaN
__device__ __forceinline__ float inverse_sum(float sum) { return sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum); }
__device__ __forceinline__ void write_four(const AttendParams& p, long long first_row, int kvh, int row, int column, float4 o, float f) {
  const long long token = first_row + row / p.group;
  const long long dst = (token * p.heads + kvh * p.group + row % p.group) * 64 + 4 * column;
  const f32x2 lo = pack2(o.x * f, o.y * f), hi = pack2(o.z * f, o.w * f);
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + dst) =
      p.q_bf16 ? make_uint2(pair_to_sixteen<__nv_bfloat16>(lo), pair_to_sixteen<__nv_bfloat16>(hi)) : make_uint2(pair_to_sixteen<__half>(lo), pair_to_sixteen<__half>(hi));
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(addr) : "memory");
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool is) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(is ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int BITS, typename E>
__global__ void __launch_bounds__(kSplitThreads, 1) split_attention_kernel(const __grid_constant__ AttendParams p) {
  pdl_launch_dependents();
  constexpr bool PACKED = BITS != 16;
  using Step = SplitStep<BITS>;
  constexpr int KEYS = Step::kKeys, NT = KEYS / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_scan[kSplitWarps], s_ends[kSplitWarps + 1];
  __shared__ int2 s_found[kSplitWarps];
  __shared__ struct {
    int at, b, kvh, tile, rows, steps, first_row;
  } s_groups[kSplitWarps + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  if constexpr (PACKED) fill_split_table<BITS>(p.codebooks, tid, kSplitThreads);
  pdl_wait();

  const SplitLine<KEYS> line(p, s_scan);
  // ---- the block's piece of the line, and the warp's
  const int piece = max(static_cast<int>((static_cast<unsigned>(line.total) + gridDim.x - 1) / gridDim.x), 1);
  int from = static_cast<int>(min(static_cast<long long>(blockIdx.x) * piece, static_cast<long long>(line.total))), to = min(piece, line.total - from) + from;
  if (p.whole_units) {                                                             // the units that begin in the piece
    line.find(2, [&](int i) { return i == 0 ? from : to; }, s_found);
    __syncthreads();
    if (warp < 2) {
      const int x = warp == 0 ? from : to;
      int at = x;
      if (x < line.total) {
        const SplitUnit u = line.locate(p, x, s_found + warp, at);
        if (at < x) at += u.steps;
      }
      if (lane == 0) s_ends[warp] = at;
    }
    __syncthreads();
    from = s_ends[0];
    to = s_ends[1];
  } else if (blockIdx.x == 0 && tid == 0) {
    static_cast<SplitHeader*>(p.workspace)->piece = piece;
  }
  if (from >= to) return;
  const int per = (to - from + kSplitWarps - 1) / kSplitWarps;
  int start = min(from + warp * per, to), end = min(start + per, to);
  // parts of this block's warps; the units they are of, by the warp that has the first: 0 .. (begun there), kSplitWarps (before the block's piece)
  float* const parts = p.part_rows <= kSplitSharedRows ? reinterpret_cast<float*>(smem + split_parts<BITS>() - (PACKED ? smem_u32(smem) : 0))
                                                       : split_part(p, 2ll * gridDim.x + 2ll * kSplitWarps * blockIdx.x);
  const int part_size = p.part_rows * kSplitPartRow;
  if (tid <= kSplitWarps) s_groups[tid].rows = 0;
  line.find(kSplitWarps, [&](int w) { return from + w * per; }, s_found);
  __syncthreads();
  int at = start;
  SplitUnit u;
  if (start < to) u = line.locate(p, start, s_found + warp, at);
  if (p.whole_units == 2) {                                                        // the units that begin in the warp's piece
    if (at < start) {
      at += u.steps;
      if (at < to) u = split_next<KEYS>(p, u.b, u.kvh, u.tile);
    }
    start = at;
    if (lane == 0) s_ends[warp] = at;
    __syncthreads();
    end = warp + 1 < kSplitWarps ? s_ends[warp + 1] : to;
  }
  if (start < end) {

  const uint32_t ring = split_ring<BITS>(smem_u32(smem), warp);
  // ---- copies, two steps ahead of the computation, in halves of sixteen keys (16 bits: whole steps).  A run is what lies side by side: the rest
  // of a page, or of an image's states; the page after it is looked up when it begins.
  struct { int b, kvh, tile, keys, steps; } f = {u.b, u.kvh, u.tile, u.keys, u.steps};
  int f_step = start - at, f_left = end - start, f_slot = 0;
  int run = 0, next_page = 0;                                                      // sixteens of the run that are left
  bool valid = false, masked = true;
  const uint8_t *fk = p.k.rows, *fv = p.v.rows, *fs = reinterpret_cast<const uint8_t*>(p.k.stats);      // the lane's 16 bytes of the next sixteen
  auto look_up = [&](int key) {
    next_page = f.b;
    if (p.table != nullptr && key < f.keys) next_page = p.table[static_cast<long long>(f.b) * p.table_width + (key >> p.page_shift)];
  };
  auto mask_ahead = [&](int key) {
    if (!PACKED && p.mask != nullptr) masked = key + (lane & 15) < f.keys && p.mask[f.b * p.mask_stride + key + (lane & 15)] != 0;
  };
  auto begin_run = [&](int key) {
    const int page = next_page, size = p.table != nullptr ? 1 << p.page_shift : 0x7ffffff0, in = key & (size - 1);
    const int place = p.table != nullptr ? in : key, left = (f.keys - key + 15) >> 4;
    run = p.table != nullptr ? min((size - in) >> 4, left) : left;
    valid = p.table == nullptr || (page >= 0 && page < p.pages);
    if (PACKED) {
      const long long row = valid ? ((static_cast<long long>(page) * p.kv_heads + f.kvh) << p.page_shift) + place : 0;
      fk = p.k.rows + row * Step::kRow + lane * 16;
      fv = p.v.rows + row * Step::kRow + lane * 16;
      fs = reinterpret_cast<const uint8_t*>((lane & 4 ? p.v.stats : p.k.stats) + row) + (lane & 3) * 16 + (lane & 8) * 8;
    } else {
      const long long blk = valid ? page : 0, row = valid ? place + (lane >> 3) : 0;
      fk = p.k.rows + blk * p.k.block_stride + f.kvh * p.k.head_stride + row * p.k.token_stride + (lane & 7) * 16;
      fv = p.v.rows + blk * p.v.block_stride + f.kvh * p.v.head_stride + row * p.v.token_stride + (lane & 7) * 16;
    }
    look_up(key + run * 16);
  };
  look_up(f_step * KEYS);
  mask_ahead(f_step * KEYS);
  // returns which of the step's keys are seen
  auto copy_step = [&]() {
    uint32_t seen = 0;
    if (f_left > 0) {
      const uint32_t dst = ring + f_slot * Step::kBytes;
      if (PACKED && valid && run >= 2 && f_step * KEYS + KEYS <= f.keys) {          // both halves there, side by side
        constexpr int CHUNKS = 8 * BITS;
        const uint32_t to = dst + lane * 16 + (lane >= CHUNKS / 2 ? Step::kPad : 0);
        constexpr uint32_t half = 16 * Step::kRow;
        if (lane < CHUNKS) {
          cp_async_16(to, fk);
          cp_async_16(to + half + 2 * Step::kPad, fk + half);
          cp_async_16(to + Step::kRows, fv);
          cp_async_16(to + Step::kRows + half + 2 * Step::kPad, fv + half);
        }
        if (lane < 16) cp_async_16(dst + 2 * Step::kRows + ((lane >> 2) & 1) * Step::kStats + (lane >> 3) * 64 + (lane & 3) * 16, fs);
        fk += 2 * half;
        fv += 2 * half;
        fs += 128;
        run -= 2;
        seen = 0xffffffffu;
      } else
#pragma unroll
      for (int h = 0; h < KEYS / 16; ++h) {
        const int key = f_step * KEYS + 16 * h, left = f.keys - key;
        if (run == 0 && left > 0) begin_run(key);
        const bool is = valid && left > 0;
        uint32_t half = !is ? 0u : left >= 16 ? 0xFFFFu : (1u << left) - 1u;
        if constexpr (PACKED) {
          constexpr int CHUNKS = 8 * BITS;                                         // of 16 bytes, in sixteen rows
          const uint32_t to = dst + h * (16 * Step::kRow + 2 * Step::kPad) + lane * 16 + (lane >= CHUNKS / 2 ? Step::kPad : 0);
          if (lane < CHUNKS) {
            cp_async_16(to, fk, is);
            cp_async_16(to + Step::kRows, fv, is);
          }
          if (lane < 8) cp_async_16(dst + 2 * Step::kRows + (lane >> 2) * Step::kStats + h * 64 + (lane & 3) * 16, fs, is);
          fk += 16 * Step::kRow;
          fv += 16 * Step::kRow;
          fs += 64;
        } else {
          if (p.mask != nullptr) half &= __ballot_sync(0xffffffffu, masked);
          const uint32_t to = dst + (lane >> 3) * 128;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t at = to + r * 512 + (((lane & 7) ^ ((4 * r + (lane >> 3)) & 7)) << 4);
            const bool sees = (half >> (4 * r + (lane >> 3))) & 1;
            cp_async_16(at, fk + r * 4 * p.k.token_stride, sees);
            cp_async_16(at + Step::kRows, fv + r * 4 * p.v.token_stride, sees);
          }
          fk += 16 * p.k.token_stride;
          fv += 16 * p.v.token_stride;
        }
        run -= left > 0 ? 1 : 0;
        seen |= half << (16 * h);
      }
      f_slot = f_slot + 1 == kSplitStages ? 0 : f_slot + 1;
      if (--f_left > 0) {
        if (++f_step == f.steps) {
          const SplitUnit n = split_next<KEYS>(p, f.b, f.kvh, f.tile);
          f = {n.b, n.kvh, n.tile, n.keys, n.steps};
          f_step = run = 0;
          look_up(0);
        }
        mask_ahead(f_step * KEYS);
      }
    }
    cp_async_commit();
    return seen;
  };
  // rows g and g + 8 of a unit's queries: values 16c .. 16c + 15 (packed), 8n + 2c and the next (16 bits); the first unit's before the copies
  uint32_t qw[2][8];
  auto load_queries = [&] {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool row = g + 8 * h < u.rows;
      const int r = u.tile * kSplitRows + (row ? g + 8 * h : 0);
      const uint16_t* const src = attend_query(p, u.seq, u.b, r / p.group, u.kvh * p.group + r % p.group);
      if constexpr (PACKED) {
        uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0;
        if (row) {
          u0 = reinterpret_cast<const uint4*>(src + 16 * c)[0];
          u1 = reinterpret_cast<const uint4*>(src + 16 * c)[1];
        }
        qw[h][0] = u0.x; qw[h][1] = u0.y; qw[h][2] = u0.z; qw[h][3] = u0.w; qw[h][4] = u1.x; qw[h][5] = u1.y; qw[h][6] = u1.z; qw[h][7] = u1.w;
      } else {
#pragma unroll
        for (int n = 0; n < 8; ++n) qw[h][n] = row ? *reinterpret_cast<const uint32_t*>(src + 8 * n + 2 * c) : 0u;
      }
    }
  };
  load_queries();
  uint32_t seen_now, seen_next = copy_step(), seen_after = copy_step();

  // ---- units
  // Which key the columns of the 8-wide products are: packed, column 2c + j of tile n is key 8c + (n & 1) + 2j + 4 (n >> 1), so that a lane's eight
  // keys lie side by side and reads of rows have no bank conflicts; 16 bits, 8n + 2c + j.
  const float ninf = __int_as_float(0xff800000);
  constexpr auto key_in_eight = [](int n, int j) { return (n & 1) + 2 * j + 4 * (n >> 1); };
  const uint32_t k_column = kSplitTable + lane * 4, v_column = k_column + 128;
  const uint32_t k_lane = (g >> 1) * (8 * Step::kRow + Step::kPad) + 2 * (g & 1) * Step::kRow;
  const uint32_t v_lane = Step::kRows + c * (8 * Step::kRow + Step::kPad);
  int step = 0, slot = 0;                                                          // of the piece
  const int steps = end - start;
  while (step < steps) {
    // rows g and g + 8 of the unit: queries, the keys that they see, the factor of their scores
    int limit[2];
    uint32_t qa[4][4];
    float row_scale[2] = {p.scale_log2, p.scale_log2}, q_sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = (u.tile * kSplitRows + (g + 8 * h < u.rows ? g + 8 * h : 0)) / p.group;
      limit[h] = p.causal ? min(u.seq.keys, max(u.seq.keys - u.seq.all_queries + i + 1, 0)) : u.seq.keys;
      uint32_t* const w = qw[h];
      if constexpr (PACKED) {
        if (p.q_bf16) {
          float top = bf16_top(w, 8);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          row_scale[h] *= bf16_to_half(w, 8, top);
        }
        f32x2 q2 = pack2(0.0f, 0.0f);
#pragma unroll
        for (int n = 0; n < 8; ++n) q2 = add2(q2, sixteen_to_pair<__half>(w[n]));
        float x, y;
        unpack2(q2, x, y);
        x += y;
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        q_sum[h] = x + __shfl_xor_sync(0xffffffffu, x, 2);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        qa[s][h] = w[2 * s];
        qa[s][2 + h] = w[2 * s + 1];
      }
    }
    float top[2] = {ninf, ninf}, sum[2] = {0.0f, 0.0f}, o[8][4] = {}, centers[2] = {0.0f, 0.0f};
    const int unit_last = min(at + u.steps, end) - start;
    const int key_base = (start - at) * KEYS;                    // key of step s: key_base + s * KEYS
    // the loop twice: with the upper eight rows and without, whose work would else be issued for nothing
    auto steps_of = [&](auto two) {
    constexpr bool both = decltype(two)::value;
#pragma unroll 1
    for (; step < unit_last; ++step) {
      seen_now = seen_next;
      seen_next = seen_after;
      seen_after = copy_step();
      cp_async_wait<2>();
      __syncwarp();
      const uint32_t src = ring + slot * Step::kBytes;
      uint32_t seen = seen_now;
      slot = slot + 1 == kSplitStages ? 0 : slot + 1;
      const int base = key_base + step * KEYS;
      const bool all = seen == (KEYS == 32 ? 0xffffffffu : 0xffffu);
      // ---- scores
      float s[NT][4];
      if constexpr (PACKED) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint32_t row = src + k_lane + key_in_eight(n, 0) * Step::kRow;
          uint32_t lo, hi;
          if constexpr (BITS == 4) {
            const uint2 w = lds64(row + 8 * c);
            lo = w.x; hi = w.y;
          } else if constexpr (BITS == 3) {
            const uint32_t first = row + ((6 * c) & ~3), w0 = lds32(first), w1 = lds32(first + 4);
            lo = __funnelshift_r(w0, w1, (c & 1) * 16);
            hi = __funnelshift_r(c & 1 ? w1 : w0, c & 1 ? 0u : w1, c & 1 ? 8 : 24);
          } else {
            lo = lds32(row + 4 * c);
            hi = lo >> 16;
          }
          const uint32_t b0 = lds_const_u32(table_address<BITS, 0>(lo, k_column)), b1 = lds_const_u32(table_address<BITS, 1>(lo, k_column));
          const uint32_t b2 = lds_const_u32(table_address<BITS, 2>(lo, k_column)), b3 = lds_const_u32(table_address<BITS, 3>(lo, k_column));
          const uint32_t b4 = lds_const_u32(table_address<BITS, 0>(hi, k_column)), b5 = lds_const_u32(table_address<BITS, 1>(hi, k_column));
          const uint32_t b6 = lds_const_u32(table_address<BITS, 2>(hi, k_column)), b7 = lds_const_u32(table_address<BITS, 3>(hi, k_column));
          mma_16816_first<E>(s[n], qa[0], b0, b1);
          mma_16816<E>(s[n], qa[1], b2, b3);
          mma_16816<E>(s[n], qa[2], b4, b5);
          mma_16816<E>(s[n], qa[3], b6, b7);
        }
        // q . k = scale * (q . level) + center * sum q
        const uint32_t stats = src + 2 * Step::kRows + c * 32;
        const uint4 k0 = lds128(stats), k1 = lds128(stats + 16);
        uint32_t kst[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
        if (!all) {                                                                // whatever lies behind the last key: 0
#pragma unroll
          for (int j = 0; j < 8; ++j) kst[j] = (seen >> (8 * c + j)) & 1 ? kst[j] : 0u;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 cs = __half22float2(*reinterpret_cast<const __half2*>(&kst[key_in_eight(n, j)]));
            s[n][j] = fmaf(s[n][j], cs.y, cs.x * q_sum[0]);
            if (both) s[n][2 + j] = fmaf(s[n][2 + j], cs.y, cs.x * q_sum[1]);
          }
      } else {
        // matrices of 8 keys x 8 values: lanes 0-7 keys 0-7, 8-15 the next eight values, 16-31 keys 8-15
        const int row = (lane & 7) + 8 * (lane >> 4), ch = (lane >> 3) & 1;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4(src + row * 128 + (((2 * t + ch) ^ (row & 7)) << 4), b0, b1, b2, b3);
          if (t == 0) {
            mma_16816_first<E>(s[0], qa[t], b0, b1);
            mma_16816_first<E>(s[1], qa[t], b2, b3);
          } else {
            mma_16816<E>(s[0], qa[t], b0, b1);
            mma_16816<E>(s[1], qa[t], b2, b3);
          }
        }
      }
      // ---- softmax: lane 4g + c has rows g and g + 8
      if (!__all_sync(0xffffffffu, all && base + KEYS <= limit[0] && base + KEYS <= limit[1])) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = PACKED ? 8 * c + key_in_eight(n, j & 1) : 8 * n + 2 * c + (j & 1);
            if (((seen >> key) & 1) == 0 || base + key >= limit[j >> 1]) s[n][j] = ninf;
          }
        if constexpr (PACKED) {
          // Values that are NaN, and only some of the rows see them: 0 * NaN would show in the others.  They are left out from here on, and the
          // sums of the rows that see one are NaN instead.
          const uint32_t own = lds32(src + 2 * Step::kRows + Step::kStats + lane * 4);
          const uint32_t bad = seen & __ballot_sync(0xffffffffu, (own & 0x7C00u) == 0x7C00u || (own & 0x7C000000u) == 0x7C000000u);
          if (bad != 0) {
            seen &= ~bad;
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (base + __ffs(bad) - 1 < limit[h]) sum[h] = __int_as_float(0x7fffffff);
          }
        }
      }
      // Packed: the values' scales go into the probabilities, sum p (scale * level + center) = sum (p scale) level + sum p center.  A row's
      // exponents are taken against the largest of a key's score plus its scale (log2, rounded down), so that p * scale stays in fp16's range;
      // what this multiplies all three sums by cancels in the end.  The largest score plus the largest scale bounds it and says whether there is
      // anything to renew.  The two may be different keys': taken for the maximum all the same, a large value that counts for little, or that the
      // row does not see, costs all others their bits, 2^-25 of it each.  Up to 2^6 that is below other roundings (2^-19); scales further apart are
      // added key by key.  Looking for them where there is something to renew: 64 contexts in 4 bits 29.2 -> 29.4 us, two long ones in 3 51.2 -> 52.2;
      // key by key in every step: 29.5 and 52.8.
      float v_log = 0.0f;
      if constexpr (PACKED) {
        const uint32_t own = (seen >> lane) & 1 ? (lds32(src + 2 * Step::kRows + Step::kStats + lane * 4) >> 26) & 31u : 0u;       // without the sign, which a NaN may have
        v_log = static_cast<float>(static_cast<int>(__reduce_max_sync(0xffffffffu, own)) - 15);
      }
      float m[2] = {ninf, ninf};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 1 && !both) continue;
        float x = fmaxf(s[0][2 * h], s[0][2 * h + 1]);
#pragma unroll
        for (int n = 1; n < NT; ++n) x = max3(x, s[n][2 * h], s[n][2 * h + 1]);
        x *= row_scale[h];                                                         // a positive factor
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        m[h] = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2)) + v_log;
      }
      // a maximum is renewed when it is passed by 2^8: sums are as exact, and it happens a few times a unit
      auto passed = [&](int h) { return m[h] > top[h] + 8.0f || (top[h] == ninf && m[h] > ninf); };
      bool renew[2] = {passed(0), passed(1)};
      if (__any_sync(0xffffffffu, renew[0] || renew[1])) {
        // scales more than 2^6 apart: with each key's own
        bool apart = false;
        if constexpr (PACKED) {
          const uint32_t own = (seen >> lane) & 1 ? (lds32(src + 2 * Step::kRows + Step::kStats + lane * 4) >> 26) & 31u : 31u;
          apart = static_cast<int>(__reduce_min_sync(0xffffffffu, own)) - 15 < static_cast<int>(v_log) - 6;
        }
        if (PACKED && apart) {
          m[0] = m[1] = ninf;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t scale = lds32(src + 2 * Step::kRows + Step::kStats + (8 * c + key_in_eight(n, j)) * 4);
              const float e = static_cast<float>(static_cast<int>((scale >> 26) & 31u) - 15);
              m[0] = fmaxf(m[0], fmaf(s[n][j], row_scale[0], e));
              if (both) m[1] = fmaxf(m[1], fmaf(s[n][2 + j], row_scale[1], e));
            }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            m[h] = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 1));
            m[h] = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 2));
            renew[h] = passed(h);
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float next = renew[h] ? m[h] : top[h];
          const float f = renew[h] ? exp2_approx(top[h] - next) : 1.0f;
          top[h] = next;
          sum[h] *= f;
          centers[h] *= f;
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            o[n][2 * h] *= f;
            o[n][2 * h + 1] *= f;
          }
        }
      }
      uint32_t pa[NT][2];
      uint32_t vst[8];                                                             // center and scale of the lane's eight values
      if constexpr (PACKED) {
        const uint32_t stats = src + 2 * Step::kRows + Step::kStats + c * 32;
        const uint4 v0 = lds128(stats), v1 = lds128(stats + 16);
        vst[0] = v0.x; vst[1] = v0.y; vst[2] = v0.z; vst[3] = v0.w; vst[4] = v1.x; vst[5] = v1.y; vst[6] = v1.z; vst[7] = v1.w;
        if (seen != 0xffffffffu) {
#pragma unroll
          for (int j = 0; j < 8; ++j) vst[j] = (seen >> (8 * c + j)) & 1 ? vst[j] : 0u;
        }
      }
      const float nm[2] = {top[0] == ninf ? 0.0f : -top[0], top[1] == ninf ? 0.0f : -top[1]};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float scale[2], center[2];
        if constexpr (PACKED) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 cs = __half22float2(*reinterpret_cast<const __half2*>(&vst[key_in_eight(n, j)]));
            center[j] = cs.x;
            scale[j] = cs.y;
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 1 && !both) {
            pa[n][1] = 0u;
            continue;
          }
          float e[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            e[j] = exp2_approx(fmaf(s[n][2 * h + j], row_scale[h], nm[h]));
            sum[h] += e[j];
            if constexpr (PACKED) {
              centers[h] = fmaf(e[j], center[j], centers[h]);
              e[j] *= scale[j];
            }
          }
          pa[n][h] = pair_to_sixteen<E>(pack2(e[0], e[1]));                        // rounded for the second product
        }
      }
      // ---- values
#pragma unroll
      for (int d = 0; d < KEYS / 16; ++d) {
        const uint32_t a[4] = {pa[2 * d][0], pa[2 * d][1], pa[2 * d + 1][0], pa[2 * d + 1][1]};
        if constexpr (PACKED) {
          uint32_t vb[2][8];                                                       // [first or second eight keys][value 8g + n]
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t w[2], even, odd;                                              // numbers of pairs of the two keys' codes
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const uint32_t row = src + v_lane + key_in_eight(2 * d + e, t) * Step::kRow;
              if constexpr (BITS == 4) {
                w[t] = lds32(row + 4 * g);
              } else if constexpr (BITS == 3) {
                const uint32_t first = row + ((3 * g) & ~3);
                w[t] = __funnelshift_r(lds32(first), lds32(row + min((3 * g & ~3) + 4, 20)), 8 * ((3 * g) & 3));
              } else {
                w[t] = lds16(row + 2 * g);
              }
            }
            constexpr uint32_t M = BITS == 4 ? 0x0F0F0F0Fu : BITS == 3 ? 0x001C71C7u : 0x3333u;      // codes 0, 2, 4, 6
            even = (w[0] & M) | ((w[1] << (BITS & 7)) & (M << (BITS & 7)));
            odd = ((w[0] >> (BITS & 7)) & M) | (w[1] & (M << (BITS & 7)));
            vb[e][0] = lds_const_u32(table_address<BITS, 0>(even, v_column));
            vb[e][2] = lds_const_u32(table_address<BITS, 1>(even, v_column));
            vb[e][4] = lds_const_u32(table_address<BITS, 2>(even, v_column));
            vb[e][6] = lds_const_u32(table_address<BITS, 3>(even, v_column));
            vb[e][1] = lds_const_u32(table_address<BITS, 0>(odd, v_column));
            vb[e][3] = lds_const_u32(table_address<BITS, 1>(odd, v_column));
            vb[e][5] = lds_const_u32(table_address<BITS, 2>(odd, v_column));
            vb[e][7] = lds_const_u32(table_address<BITS, 3>(odd, v_column));
          }
#pragma unroll
          for (int n = 0; n < 8; ++n) mma_16816<E>(o[n], a, vb[0][n], vb[1][n]);
        } else {
          // transposed: lanes 0-7 keys 0-7, 8-15 keys 8-15, 16-31 the next eight values
          const int row = lane & 15, ch = lane >> 4;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            uint32_t b0, b1, b2, b3;
            ldmatrix_x4_trans(src + Step::kRows + row * 128 + (((2 * t + ch) ^ (row & 7)) << 4), b0, b1, b2, b3);
            mma_16816<E>(o[2 * t], a, b0, b1);
            mma_16816<E>(o[2 * t + 1], a, b2, b3);
          }
        }
      }
      __syncwarp();                                                                // the slot may be copied over
    }
    };
    if (u.rows > 8) steps_of(std::true_type{});
    else steps_of(std::false_type{});
    // ---- the unit, or its part.  o[n][2h + j]: row g + 8h, value 16c + 8j + n (packed), 8n + 2c + j (16 bits)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
      if constexpr (PACKED) {
        centers[h] += __shfl_xor_sync(0xffffffffu, centers[h], 1);
        centers[h] += __shfl_xor_sync(0xffffffffu, centers[h], 2);
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) o[n][2 * h + j] += centers[h];
      }
    }
    const bool begins = at >= start, complete = begins && at + u.steps <= end;
    if (lane == 0) {
      if (complete && !p.whole_units) split_records(p)[(static_cast<long long>(u.b) * p.kv_heads + u.kvh) * p.tiles + u.tile] = {at, u.steps, 1, 0};
      if (!complete && (begins || warp == 0)) s_groups[begins ? warp : kSplitWarps] = {at, u.b, u.kvh, u.tile, u.rows, u.steps, u.seq.first_row};
    }
    float* const part = parts + (2 * warp + (begins ? 1 : 0)) * part_size;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (g + 8 * h >= u.rows) continue;
      const int r = u.tile * kSplitRows + g + 8 * h;
      if (complete) {
        const float f = inverse_sum(sum[h]);
        const long long token = u.seq.first_row + r / p.group;
        uint16_t* const dst = static_cast<uint16_t*>(p.out) + (token * p.heads + u.kvh * p.group + r % p.group) * 64;
        auto two = [&](float x, float y) { return p.q_bf16 ? pair_to_sixteen<__nv_bfloat16>(pack2(x * f, y * f)) : pair_to_sixteen<__half>(pack2(x * f, y * f)); };
        if constexpr (PACKED) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
            *reinterpret_cast<uint4*>(dst + 16 * c + 8 * j) = make_uint4(two(o[0][2 * h + j], o[1][2 * h + j]), two(o[2][2 * h + j], o[3][2 * h + j]),
                                                                         two(o[4][2 * h + j], o[5][2 * h + j]), two(o[6][2 * h + j], o[7][2 * h + j]));
        } else {
#pragma unroll
          for (int n = 0; n < 8; ++n) *reinterpret_cast<uint32_t*>(dst + 8 * n + 2 * c) = two(o[n][2 * h], o[n][2 * h + 1]);
        }
      } else {
        float* const dst = part + (g + 8 * h) * kSplitPartRow;
        if constexpr (PACKED) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            *reinterpret_cast<float4*>(dst + 16 * c + 8 * j) = make_float4(o[0][2 * h + j], o[1][2 * h + j], o[2][2 * h + j], o[3][2 * h + j]);
            *reinterpret_cast<float4*>(dst + 16 * c + 8 * j + 4) = make_float4(o[4][2 * h + j], o[5][2 * h + j], o[6][2 * h + j], o[7][2 * h + j]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < 8; ++n) *reinterpret_cast<float2*>(dst + 8 * n + 2 * c) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        }
        if (c == 0) *reinterpret_cast<float2*>(dst + 64) = make_float2(top[h], sum[h]);
      }
    }
    at += u.steps;
    if (step < steps) {
      u = split_next<KEYS>(p, u.b, u.kvh, u.tile);
      load_queries();
    }
  }
  cp_async_wait<0>();
  }
  // ---- units that lie in more than one warp's piece
  __syncthreads();
  for (int item = tid;; item += kSplitThreads) {                                  // four values of a row of some unit
    int i = 0, rest = item;
    while (i <= kSplitWarps && rest >= s_groups[i].rows * 16) rest -= s_groups[i++].rows * 16;
    if (i > kSplitWarps) break;
    const auto& u = s_groups[i];
    const int first = i < kSplitWarps ? i : 0, last = (min(u.at + u.steps, to) - 1 - from) / per, row = rest >> 4, column = rest & 15;
    float top, sum;
    const float4 o = add_parts(last - first + 1, row, column, top, sum, [&](int q) { return parts + (2 * (first + q) + (q == 0 && i < kSplitWarps ? 1 : 0)) * part_size; });
    const bool complete = u.at >= from && u.at + u.steps <= to;
    if (rest == 0 && u.at >= from && !p.whole_units)
      split_records(p)[(static_cast<long long>(u.b) * p.kv_heads + u.kvh) * p.tiles + u.tile] = {u.at, u.steps, complete ? 1 : 0, 0};
    if (complete) {
      write_four(p, u.first_row, u.kvh, u.tile * kSplitRows + row, column, o, inverse_sum(sum));
    } else {
      float* const dst = split_part(p, 2ll * blockIdx.x + (u.at >= from ? 1 : 0)) + row * kSplitPartRow;
      *reinterpret_cast<float4*>(dst + 4 * column) = o;
      if (column == 0) *reinterpret_cast<float2*>(dst + 64) = make_float2(top, sum);
    }
  }
}

// Adds up the blocks' parts of the units that lie in more than one block's piece: a block a unit, four values of a row a thread.
constexpr int kJoinThreads = 256;
static __global__ void __launch_bounds__(kJoinThreads) join_attention_kernel(const __grid_constant__ AttendParams p) {
  pdl_launch_dependents();
  const long long unit = blockIdx.x;
  const int tile = static_cast<int>(unit % p.tiles), kvh = static_cast<int>(unit / p.tiles % p.kv_heads), b = static_cast<int>(unit / p.tiles / p.kv_heads);
  pdl_wait();
  const SplitRecord rec = split_records(p)[unit];                                  // not written where there is no such tile
  const int piece = static_cast<SplitHeader*>(p.workspace)->piece;
  const AttendSequence seq = attend_sequence(p, b);
  if (tile >= split_tiles(p, seq) || rec.whole) return;
  const int rows = split_rows(p, seq, tile);
  const int first = rec.start / piece, last = (rec.start + rec.steps - 1) / piece;
  for (int e = threadIdx.x; e < rows * 16; e += kJoinThreads) {
    const int row = e >> 4, column = e & 15;
    float top, sum;
    const float4 o = add_parts(last - first + 1, row, column, top, sum,
                               [&](int q) { return split_part(p, 2ll * (first + q) + (rec.start >= (first + q) * piece ? 1 : 0)); });
    write_four(p, seq.first_row, kvh, tile * kSplitRows + row, column, o, inverse_sum(sum));
  }
}

}  // namespace arcq
