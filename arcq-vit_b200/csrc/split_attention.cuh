// Attention of few queries a key head over long keys: one new token of a sequence over its cache, or of an image's text over the
// encoder's states.  Keys and values are read once and never staged: registers straight from global memory to the tensor instructions.
//
//   s_ij = scale * q_i . k_j over the keys j that query i sees,   o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i)
//
// The rows of a tile are 16 (query, head) pairs that share a key head.  Its keys are split over the blocks of a cluster, and a block's
// over its warps, blocks of 16 or 32 keys in turn; each warp keeps a running maximum, sum and 16 x 64 accumulator, joined in shared
// memory of the block and then of the cluster.  No workspace, no second launch, a fixed order of every sum.
//
// Packed keys and values become fp16 in registers: a byte of two codes is an index into a table of pairs of levels (a copy a lane, so
// that a read has no bank conflicts), one half-precision fma makes center + scale * level.  Keys are paired along a head's values, which
// the packed byte already is; values along the keys, two bytes interleaved.  The order of a head's values within a product is free, so
// each lane takes 16 (keys) or 8 (values) that lie next to each other.
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
  const int up = top > 0.0f && e < 128 ? min(max(13 - e, -100), 100) : 0;
  const float f = __int_as_float((up + 127) << 23);
#pragma unroll
  for (int j = 0; j < n; ++j) w[j] = pair_to_sixteen<__half>(mul2(sixteen_to_pair<__nv_bfloat16>(w[j]), pack2(f, f)));
  return __int_as_float((127 - up) << 23);
}

constexpr int kSplitWarps = 8, kSplitThreads = kSplitWarps * 32, kSplitRows = 16;
constexpr int kSplitMaxBlocks = 8;                                  // of a cluster: the portable size
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

// The rows of one block of keys that a lane holds.  Lane 4g + c: of keys 8n + g the 16 values from 16c, of values 2c, 2c + 1 (+ 8 n) the 8 from 8g.
template <int BITS> struct KeyBlock;
template <int BITS> struct KeyBlock {
  static constexpr int kKeys = 32;
  uint32_t k[4][BITS == 4 ? 2 : BITS == 3 ? 2 : 1], v[4][2], k_stats[4], v_stats[4][2];
};
template <> struct KeyBlock<16> {
  static constexpr int kKeys = 16;
  uint4 k[2][2], v[2][2];
};

template <int BITS, typename E>
__global__ void __launch_bounds__(kSplitThreads, 2) split_attention_kernel(const __grid_constant__ AttendParams p) {
  pdl_launch_dependents();
  constexpr bool PACKED = BITS != 16;
  constexpr int KEYS = KeyBlock<BITS>::kKeys, NT = KEYS / 8;
  extern __shared__ __align__(128) uint8_t smem[];                  // tables of levels (keys, values), then accumulators over them
  __shared__ float s_max[kSplitWarps][kSplitRows], s_sum[kSplitWarps][kSplitRows];
  __shared__ float s_block_max[kSplitRows], s_block_sum[kSplitRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x % p.splits, unit = blockIdx.x / p.splits;
  const int tile = unit % p.tiles, kvh = unit / p.tiles % p.kv_heads, b = unit / p.tiles / p.kv_heads;
  const uint32_t k_table = smem_u32(smem) + lane * 4, v_table = smem_u32(smem) + kPairTableBytes + (lane & 15) * 8;
  if constexpr (PACKED) {
    fill_pair_table(smem_u32(smem), p.codebooks, 1 << BITS, tid, kSplitThreads);
    fill_pair_table_f32(smem_u32(smem) + kPairTableBytes, p.codebooks + (1 << BITS), 1 << BITS, tid, kSplitThreads);
  }
  pdl_wait();
  __syncthreads();
  const AttendSequence seq = attend_sequence(p, b);
  const int rows = min(seq.queries * p.group - tile * kSplitRows, kSplitRows);     // <= 0: an empty tile
  // keys that some row of the tile sees
  int limit[2], keys = 0;
  const uint16_t* q_row[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = min(g + 8 * h, max(rows, 1) - 1), at = tile * kSplitRows + r, i = at / p.group, head = kvh * p.group + at % p.group;
    limit[h] = p.causal ? min(seq.keys, max(seq.keys - seq.all_queries + i + 1, 0)) : seq.keys;
    q_row[h] = attend_query(p, seq, b, i, head);
  }
  if (rows > 0) {
    const int i = (tile * kSplitRows + rows - 1) / p.group;
    keys = p.causal ? min(seq.keys, max(seq.keys - seq.all_queries + i + 1, 0)) : seq.keys;
  }

  // ---- queries: fragments of the four steps of 16 values; bf16 against fp16 keys: a power of two makes the row's largest value 2^13..2^14
  uint32_t qa[4][4];
  float row_scale[2] = {p.scale_log2, p.scale_log2};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[8] = {};
    if (g + 8 * h < rows) {
      const uint4* const src = reinterpret_cast<const uint4*>(q_row[h] + 16 * c);
      const uint4 u0 = src[0], u1 = src[1];
      w[0] = u0.x; w[1] = u0.y; w[2] = u0.z; w[3] = u0.w; w[4] = u1.x; w[5] = u1.y; w[6] = u1.z; w[7] = u1.w;
    }
    if (PACKED && p.q_bf16) {
      float top = bf16_top(w, 8);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      row_scale[h] *= bf16_to_half(w, 8, top);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      qa[s][h] = w[2 * s];
      qa[s][2 + h] = w[2 * s + 1];
    }
  }

  const float ninf = __int_as_float(0xff800000);
  float top[2] = {ninf, ninf}, sum[2] = {0.0f, 0.0f}, o[8][4] = {};

  // ---- the block's share of the keys, in whole steps of 32
  const int steps = (keys + KEYS - 1) / KEYS;
  const int per = (steps + p.splits - 1) / p.splits;
  const int first = split * per, last = min(first + per, steps);

  auto load = [&](int step, KeyBlock<BITS>& blk, uint32_t& seen) {
    const int base = step * KEYS;
    // sixteen keys lie in one page
    long long k_at[KEYS / 16], v_at[KEYS / 16], st_at[KEYS / 16];
    bool there[KEYS / 16];
#pragma unroll
    for (int u = 0; u < KEYS / 16; ++u) {
      const int j = base + 16 * u;
      int block = b, place = j;
      there[u] = j < keys;
      if (p.table != nullptr && there[u]) {
        block = p.table[static_cast<long long>(b) * p.table_width + (j >> p.page_shift)];
        place = j & ((1 << p.page_shift) - 1);
        there[u] = block >= 0 && block < p.pages;
      }
      k_at[u] = block * p.k.block_stride + kvh * p.k.head_stride + place * p.k.token_stride;
      v_at[u] = block * p.v.block_stride + kvh * p.v.head_stride + place * p.v.token_stride;
      st_at[u] = PACKED ? ((static_cast<long long>(block) * p.kv_heads + kvh) << p.page_shift) + place : 0;
    }
    bool mine = lane < KEYS && base + lane < keys && there[KEYS / 16 - 1 < (lane >> 4) ? KEYS / 16 - 1 : (lane >> 4)];
    if (mine && p.mask != nullptr) mine = p.mask[b * p.mask_stride + base + lane] != 0;
    seen = __ballot_sync(0xffffffffu, mine);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool is = (seen >> (8 * n + g)) & 1;
      const uint8_t* const row = p.k.rows + k_at[n >> 1] + ((n & 1) * 8 + g) * p.k.token_stride;
      if constexpr (PACKED) {
        if constexpr (BITS == 4) {
          const uint2 u = is ? *reinterpret_cast<const uint2*>(row + 8 * c) : make_uint2(0, 0);
          blk.k[n][0] = u.x; blk.k[n][1] = u.y;
        } else if constexpr (BITS == 3) {
          const uint16_t* const h = reinterpret_cast<const uint16_t*>(row + 6 * c);
          const uint32_t a = is ? h[0] : 0, d = is ? h[1] : 0, e = is ? h[2] : 0;
          blk.k[n][0] = a | ((d & 0xFFu) << 16);
          blk.k[n][1] = (d >> 8) | (e << 8);
        } else {
          blk.k[n][0] = is ? *reinterpret_cast<const uint32_t*>(row + 4 * c) : 0;
        }
        blk.k_stats[n] = is ? *reinterpret_cast<const uint32_t*>(p.k.stats + st_at[n >> 1] + (n & 1) * 8 + g) : 0;
      } else {
        const uint4* const r = reinterpret_cast<const uint4*>(row + 32 * c);
        blk.k[n][0] = is ? r[0] : make_uint4(0, 0, 0, 0);
        blk.k[n][1] = is ? r[1] : make_uint4(0, 0, 0, 0);
      }
      const uint8_t* const vrow = p.v.rows + v_at[n >> 1] + ((n & 1) * 8 + 2 * c) * p.v.token_stride;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bool vis = (seen >> (8 * n + 2 * c + t)) & 1;
        const uint8_t* const r = vrow + t * p.v.token_stride;
        if constexpr (PACKED) {
          if constexpr (BITS == 4) {
            blk.v[n][t] = vis ? *reinterpret_cast<const uint32_t*>(r + 4 * g) : 0;
          } else if constexpr (BITS == 3) {
            const int q = (3 * g) >> 2;
            const uint32_t* const h = reinterpret_cast<const uint32_t*>(r);
            const uint32_t lo = vis ? h[q] : 0, hi = vis ? h[min(q + 1, 5)] : 0;
            blk.v[n][t] = __funnelshift_r(lo, hi, 8 * ((3 * g) & 3)) & 0xFFFFFFu;
          } else {
            blk.v[n][t] = vis ? *reinterpret_cast<const uint16_t*>(r + 2 * g) : 0;
          }
          blk.v_stats[n][t] = vis ? *reinterpret_cast<const uint32_t*>(p.v.stats + st_at[n >> 1] + (n & 1) * 8 + 2 * c + t) : 0;
        } else {
          blk.v[n][t] = vis ? *reinterpret_cast<const uint4*>(r + 16 * g) : make_uint4(0, 0, 0, 0);
        }
      }
    }
  };

  auto compute = [&](int step, const KeyBlock<BITS>& blk, uint32_t seen) {
    const int base = step * KEYS;
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[n][j] = 0.0f;
      uint32_t kb[8];
      if constexpr (PACKED) {
        uint32_t lo, hi;
        if constexpr (BITS == 2) {
          lo = spread_codes<2>(blk.k[n][0] & 0xFFFFu);
          hi = spread_codes<2>(blk.k[n][0] >> 16);
        } else {
          lo = spread_codes<BITS>(blk.k[n][0]);
          hi = spread_codes<BITS>(blk.k[n][1]);
        }
        uint32_t pl[4], ph[4];
        pair_levels(k_table, lo, pl);
        pair_levels(k_table, hi, ph);
        const uint32_t center = __byte_perm(blk.k_stats[n], 0, 0x1010), scale = __byte_perm(blk.k_stats[n], 0, 0x3232);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          kb[j] = half2_fma(scale, pl[j], center);
          kb[4 + j] = half2_fma(scale, ph[j], center);
        }
      } else {
        kb[0] = blk.k[n][0].x; kb[1] = blk.k[n][0].y; kb[2] = blk.k[n][0].z; kb[3] = blk.k[n][0].w;
        kb[4] = blk.k[n][1].x; kb[5] = blk.k[n][1].y; kb[6] = blk.k[n][1].z; kb[7] = blk.k[n][1].w;
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) mma_16816<E>(s[n], qa[t], kb[2 * t], kb[2 * t + 1]);
    }
    // ---- softmax: lane 4g + c has rows g and g + 8, keys 8n + 2c and the next
    const bool whole = seen == (KEYS == 32 ? 0xffffffffu : 0xffffu) && base + KEYS <= limit[0] && base + KEYS <= limit[1];
    if (!whole) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = 8 * n + 2 * c + (j & 1);
          if (((seen >> key) & 1) == 0 || base + key >= limit[j >> 1]) s[n][j] = ninf;
        }
    }
    float m[2] = {top[0], top[1]};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x = ninf;
#pragma unroll
      for (int n = 0; n < NT; ++n) x = fmaxf(x, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
      x *= row_scale[h];                                       // a positive factor
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
      m[h] = fmaxf(m[h], x);
    }
    if (__any_sync(0xffffffffu, m[0] > top[0] || m[1] > top[1])) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float f = m[h] == ninf ? 1.0f : exp2_approx(top[h] - m[h]);
        top[h] = m[h];
        sum[h] *= f;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          o[n][2 * h] *= f;
          o[n][2 * h + 1] *= f;
        }
      }
    }
    const float nm[2] = {top[0] == ninf ? 0.0f : -top[0], top[1] == ninf ? 0.0f : -top[1]};
    uint32_t pa[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = exp2_approx(fmaf(s[n][2 * h], row_scale[h], nm[h])), y = exp2_approx(fmaf(s[n][2 * h + 1], row_scale[h], nm[h]));
        sum[h] += x + y;
        pa[n][h] = pair_to_sixteen<E>(pack2(x, y));            // probabilities of at most 1, rounded for the second product
      }
    // ---- values
#pragma unroll
    for (int u = 0; u < KEYS / 16; ++u) {
      uint32_t vb[2][8];                                       // [first or second eight keys][value 8g + n]
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int n = 2 * u + e;
        if constexpr (PACKED) {
          const uint32_t w0 = spread_codes<BITS>(blk.v[n][0]), w1 = spread_codes<BITS>(blk.v[n][1]);
          f32x2 even[4], odd[4];
          pair_levels_f32(v_table, (w0 & 0x0F0F0F0Fu) | ((w1 << 4) & 0xF0F0F0F0u), even);
          pair_levels_f32(v_table, ((w0 >> 4) & 0x0F0F0F0Fu) | (w1 & 0xF0F0F0F0u), odd);
          const f32x2 center = sixteen_to_pair<__half>(__byte_perm(blk.v_stats[n][0], blk.v_stats[n][1], 0x5410));
          const f32x2 scale = sixteen_to_pair<__half>(__byte_perm(blk.v_stats[n][0], blk.v_stats[n][1], 0x7632));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            vb[e][2 * j] = pair_to_sixteen<__half>(fma2(scale, even[j], center));
            vb[e][2 * j + 1] = pair_to_sixteen<__half>(fma2(scale, odd[j], center));
          }
        } else {
          const uint4 a = blk.v[n][0], d = blk.v[n][1];
          const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            vb[e][2 * j] = __byte_perm(x[j], y[j], 0x5410);
            vb[e][2 * j + 1] = __byte_perm(x[j], y[j], 0x7632);
          }
        }
      }
      const uint32_t a[4] = {pa[2 * u][0], pa[2 * u][1], pa[2 * u + 1][0], pa[2 * u + 1][1]};
#pragma unroll
      for (int n = 0; n < 8; ++n) mma_16816<E>(o[n], a, vb[0][n], vb[1][n]);
    }
  };

  {
    KeyBlock<BITS> cur, next;
    uint32_t seen = 0, seen_next = 0;
    int step = first + warp;
    if (step < last) load(step, cur, seen);
    while (step < last) {
      const int after = step + kSplitWarps;
      if (after < last) load(after, next, seen_next);
      compute(step, cur, seen);
      cur = next;
      seen = seen_next;
      step = after;
    }
  }

  // ---- join the warps: o[n][j] is row g (+ 8), value 16c + n (j odd: + 8)
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
    if (c == 0) {
      s_max[warp][g + 8 * h] = top[h];
      s_sum[warp][g + 8 * h] = sum[h];
    }
  }
  __syncthreads();                                             // the tables are not read any more
  float* const s_out = reinterpret_cast<float*>(smem);         // [warp][row][64]
  float whole_max[2], whole_sum[2] = {0.0f, 0.0f};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float m = ninf;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) m = fmaxf(m, s_max[w][g + 8 * h]);
    whole_max[h] = m;
    const float base = m == ninf ? 0.0f : m;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) whole_sum[h] += s_sum[w][g + 8 * h] * exp2_approx(s_max[w][g + 8 * h] - base);
    const float f = exp2_approx(top[h] - base);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float4* const dst = reinterpret_cast<float4*>(s_out + (warp * kSplitRows + g + 8 * h) * 64 + 16 * c + 8 * j);
      dst[0] = make_float4(o[0][2 * h + j] * f, o[1][2 * h + j] * f, o[2][2 * h + j] * f, o[3][2 * h + j] * f);
      dst[1] = make_float4(o[4][2 * h + j] * f, o[5][2 * h + j] * f, o[6][2 * h + j] * f, o[7][2 * h + j] * f);
    }
    if (warp == 0 && c == 0) {
      s_block_max[g + 8 * h] = whole_max[h];
      s_block_sum[g + 8 * h] = whole_sum[h];
    }
  }
  __syncthreads();
  // the sum over the warps takes the first warp's place
  for (int i = tid; i < kSplitRows * 64; i += kSplitThreads) {
    float x = s_out[i];
#pragma unroll
    for (int w = 1; w < kSplitWarps; ++w) x += s_out[w * kSplitRows * 64 + i];
    s_out[i] = x;
  }
  // ---- join the blocks of the cluster: each writes its part of the rows
  const bool many = p.splits > 1;
  if (many) {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
  const int count = max(rows, 0) * 64, share = (count + p.splits - 1) / p.splits;
  auto remote = [&](uint32_t addr, int rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
  };
  for (int i = split * share + tid; i < min(count, (split + 1) * share); i += kSplitThreads) {
    const int r = i >> 6;
    float x, l;
    if (many) {
      float m = ninf;
      for (int s = 0; s < p.splits; ++s) m = fmaxf(m, remote(smem_u32(s_block_max + r), s));
      const float base = m == ninf ? 0.0f : m;
      x = l = 0.0f;
      for (int s = 0; s < p.splits; ++s) {
        const float f = exp2_approx(remote(smem_u32(s_block_max + r), s) - base);
        l += f * remote(smem_u32(s_block_sum + r), s);
        x += f * remote(smem_u32(s_out + i), s);
      }
    } else {
      x = s_out[i];
      l = s_block_sum[r];
    }
    x = l > 0.0f ? x / l : (l == 0.0f ? 0.0f : l);             // a query that sees no key: zeros; NaN stays NaN
    const int at = tile * kSplitRows + r;
    const long long token = seq.first_row + at / p.group;
    const long long to = (token * p.heads + kvh * p.group + at % p.group) * 64 + (i & 63);
    if (p.q_bf16) static_cast<__nv_bfloat16*>(p.out)[to] = __float2bfloat16_rn(x);
    else static_cast<__half*>(p.out)[to] = __float2half_rn(x);
  }
  if (many) asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

}  // namespace arcq
