// Attention of many queries a key head on the fifth-generation tensor cores: pieces of prompts over a cache, texts over an encoder's states.
// Same operator as split_attention.cuh; keys and values are staged in shared memory (packed ones rebuilt in fp16 there, once a block).
//
// A block takes up to 256 rows, (query, head) pairs that share a key head, in two streams of 128 (or one, see below) with scores and output of
// their own in tensor memory, a softmax thread a row:
//   more than 128 rows   the streams are the two halves of the rows; both use every tile of 128 keys
//   up to 128 rows       both streams have the same rows, one takes the even tiles of keys, the other the odd ones
// so that one stream's exponentials run while the other's products do.  The keys of a row tile are also split over the blocks of a
// cluster where there are too few row tiles for the SMs.  Partial results are joined in shared memory of the cluster, in a fixed order.
//
// Running maximum: a row's exponents are taken against a maximum that is renewed only when a score passes it by 2^8 (then the output in
// tensor memory is scaled): probabilities reach 256 instead of 1 at most, and sums and products are as exact either way.
//
// Warps: softmax, four a stream (a tensor-memory lane quarter each), then four for keys and values, then one a stream for its products; with two
// streams two more only keep step (registers are handed over by groups of four warps).
//
// One stream: up to 128 rows over few keys in 16 bits.  Such blocks take half of an SM, so that two run side by side: a block's set-up, first loads
// and join, together as long as its products, run beside the other block's (which kernel when: one_stream_is_ahead, with times).
#pragma once
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>
#include "ptx.cuh"
#include "f32x2.cuh"
#include "attention.cuh"
#include "split_attention.cuh"

namespace arcq {

constexpr int kStatusTileAttentionTimeout = 0x502;
constexpr int kTileRows = 128, kTileKeys = 128;
__host__ __device__ constexpr int tile_threads(int streams) { return streams == 1 ? 288 : 512; }
// tiles of keys, and of values, in shared memory: 16 bits have no tables there, and one stream's blocks share an SM
__host__ __device__ constexpr int tile_slots(bool packed, int streams) { return streams == 1 ? 2 : packed ? 3 : 5; }
constexpr int kTileSeen = 8;
constexpr int kTileRanked = 64;                                    // sequences that are put in order at most
// two streams' warps share out their registers
constexpr int kTileLaunchRegs = 128, kTileSoftmaxRegs = 184, kTileLoadRegs = 88, kTileIssueRegs = 56;
static_assert(2 * kTileSoftmaxRegs + kTileLoadRegs + kTileIssueRegs <= 4 * kTileLaunchRegs, "registers beyond the launch's never come");
constexpr uint32_t kTileBytes = 128 * 128;                        // 128 rows of 64 16-bit values
constexpr int kTileWeights = 2 * (kTileRows + 8);                  // rows of a block times parts: rounded up for 8 blocks and two streams
// tensor memory, 256 columns a stream: scores, probabilities (pairs), output
__host__ __device__ constexpr uint32_t tile_s_col(int t) { return 256u * t; }
__host__ __device__ constexpr uint32_t tile_p_col(int t) { return 256u * t + 128u; }
__host__ __device__ constexpr uint32_t tile_o_col(int t) { return 256u * t + 192u; }

struct TileSmem {
  uint32_t q, k, v, tables, seen, max, sum, weight, offset, bars, total;
};
__host__ __device__ constexpr TileSmem tile_smem_layout(bool packed, int streams) {
  TileSmem s = {};
  s.q = 0;
  s.k = s.q + streams * kTileBytes;
  s.v = s.k + tile_slots(packed, streams) * kTileBytes;
  s.tables = s.v + tile_slots(packed, streams) * kTileBytes;                       // [byte][lane] pairs of levels, keys then values
  s.seen = s.tables + (packed ? 2 * kPairTableBytes : 0);
  s.max = s.seen + kTileSeen * 16;
  s.sum = s.max + 2 * kTileRows * 4;
  s.weight = s.sum + 2 * kTileRows * 4;                           // of a part in a row's result
  s.offset = s.weight + kTileWeights * 4;                         // of a row in the result
  s.bars = s.offset + 2 * kTileRows * 8;
  s.total = s.bars + 32 * 8 + 1024;                               // and alignment
  return s;
}

template <typename E> __device__ __forceinline__ uint32_t tile_idesc(int M, int N) {
  return umma_idesc_f16(M, N) | (sizeof(E) == 2 && std::is_same<E, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u);
}
__device__ __forceinline__ float lds_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 lds128_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

template <int BITS, typename E, int STREAMS, bool RANKED>
__global__ void __launch_bounds__(tile_threads(STREAMS), 3 - STREAMS) tile_attention_kernel(const __grid_constant__ AttendParams p) {
  constexpr int kThreads = tile_threads(STREAMS), kBlockRows = STREAMS * kTileRows;
  constexpr int kLoad = 4 * STREAMS, kIssue = kLoad + 4;                         // first warps
  constexpr bool PACKED = BITS != 16;
  constexpr int SLOTS = tile_slots(PACKED, STREAMS);
  extern __shared__ uint8_t tile_smem_raw[];
  uint8_t* const smem = tile_smem_raw + ((1024u - (smem_u32(tile_smem_raw) & 1023u)) & 1023u);
  constexpr TileSmem L = tile_smem_layout(PACKED, STREAMS);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + L.bars);
  uint64_t *const k_full = bars, *const k_free = bars + 5, *const v_full = bars + 10, *const v_free = bars + 15;     // [slot]
  uint64_t *const q_full = bars + 20, *const s_full = bars + 22, *const s_read = bars + 24, *const p_full = bars + 26, *const o_done = bars + 28;   // [stream]
  uint64_t* const stopped = bars + 30;
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(bars + 31);
  int* const s_first_bad = reinterpret_cast<int*>(s_tmem + 1);                    // packed: the first key whose values are NaN
  uint32_t* const s_seen = reinterpret_cast<uint32_t*>(smem + L.seen);            // [tile % kTileSeen][warp]: written before the tile's keys are handed over
  float* const s_max = reinterpret_cast<float*>(smem + L.max);                    // [stream][row]
  float* const s_sum = reinterpret_cast<float*>(smem + L.sum);
  float* const s_weight = reinterpret_cast<float*>(smem + L.weight);
  long long* const s_offset = reinterpret_cast<long long*>(smem + L.offset);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t polls = p.poll_limit;

  const int split = blockIdx.x % p.splits, unit = blockIdx.x / p.splits;
  const int kvh = unit % p.kv_heads;
  int tile = p.tiles - 1 - unit / (p.kv_heads * p.batch), b = unit / p.kv_heads % p.batch;      // long rows of causal keys first

  pdl_wait();
  if constexpr (RANKED) {
    // The sequences with most work first, by the keys that their streams go through: blocks beyond the first round start as others end, and the
    // last to start should be short (when: launch_tile; a kernel of its own, since the choice alone takes 1 % of the others' time).
    __shared__ uint32_t s_work[kTileRanked];
    __shared__ int s_b;
    uint32_t work = 0;
    if (tid < p.batch) {
      const AttendSequence s = attend_sequence(p, tid);
      const long long rows = static_cast<long long>(s.queries) * p.group;
      work = rows == 0 ? 0u : static_cast<uint32_t>(s.keys) * (rows > kTileRows ? 2u : 1u);
      s_work[tid] = work;
    }
    __syncthreads();
    const int rank = unit / (p.kv_heads * p.tiles);
    if (tid < p.batch) {
      int before = 0;
      for (int i = 0; i < p.batch; ++i) before += s_work[i] > work || (s_work[i] == work && i < tid) ? 1 : 0;
      if (before == rank) s_b = tid;
    }
    __syncthreads();
    b = s_b;
    tile = p.tiles - 1 - unit / p.kv_heads % p.tiles;
  }
  const AttendSequence seq = attend_sequence(p, b);
  const int all_rows = seq.queries * p.group;                                     // the host sees to it that rows, and those of the last block, fit
  const bool halves = STREAMS == 1 || all_rows > kTileRows;                       // the streams are halves of the rows; or there is one
  const int row0 = tile * kBlockRows, rows = min(all_rows - row0, kBlockRows);
  // Tiles of rows that are not there: the whole cluster leaves.
  if (rows <= 0) {
    pdl_launch_dependents();
    return;
  }
  if (tid == (kIssue + STREAMS - 1) * 32) {
    const int users = halves ? STREAMS : 1;                                             // streams that read a tile of keys
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(k_full + i, 4); mbar_init(v_full + i, 4);
      mbar_init(k_free + i, users); mbar_init(v_free + i, users);
    }
    *s_first_bad = 0x7fffffff;
    for (int t = 0; t < STREAMS; ++t) {
      mbar_init(s_read + t, 4); mbar_init(p_full + t, 4);
      mbar_init(s_full + t, 1); mbar_init(o_done + t, 1);
      mbar_init(q_full + t, halves ? 4 : 8);
    }
    mbar_init(stopped, STREAMS);
    mbar_fence_init();
  }
  if (warp == kIssue) {
    __syncwarp();
    tmem_alloc(s_tmem, 256 * STREAMS);
    tmem_relinquish();
    tc_fence_before_sync();
  }
  // The block's set-up ends at this barrier, which each role reaches by itself: until then the loaders look up and fetch the first keys and the
  // softmax warps their queries, while all but the loaders fill the tables.  With rows of one block written from tensor memory: 2048 tokens over
  // 16 384 in 4 bits 191 -> 187 us, 1024 queries over 2309 states 162 -> 159.
  auto fill_tables = [&](int i) {                                                 // i of all but 128 threads
    if constexpr (PACKED) {
      fill_pair_table(smem_u32(smem) + L.tables, p.codebooks, 1 << BITS, i, kThreads - 128);
      fill_pair_table_f32(smem_u32(smem) + L.tables + kPairTableBytes, p.codebooks + (1 << BITS), 1 << BITS, i, kThreads - 128);
    }
  };
  auto set_up = [&] {
    asm volatile("bar.sync 0;" ::: "memory");
    pdl_launch_dependents();
    tc_fence_after_sync();
  };
  // keys that the last row sees, the block's share of their tiles
  int keys = seq.keys;
  if (p.causal) keys = min(keys, max(seq.keys - seq.all_queries + (row0 + rows - 1) / p.group + 1, 0));
  const int all_tiles = (keys + kTileKeys - 1) / kTileKeys, per = (all_tiles + p.splits - 1) / p.splits;
  const int first = min(split * per, all_tiles), count = min(first + per, all_tiles) - first;
  // tile j of the block is tile i of stream t: halves: j = i for both; else j = 2 i + t
  bool ok = true;

  if (warp >= kIssue) {
    // ------------------------------------------------------------------ products: a warp a stream
    if constexpr (STREAMS > 1) fewer_registers<kTileIssueRegs>();
    fill_tables(tid - 128);
    set_up();
    const uint32_t tmem = *s_tmem;
    const int t = warp - kIssue;
    const int mine = t >= STREAMS ? 0 : halves ? count : (count + 1 - t) / 2;
    if (t < STREAMS && mine > 0) {
      const uint32_t idesc_s = tile_idesc<E>(kTileRows, kTileKeys);
      const uint32_t idesc_o = tile_idesc<E>(kTileRows, 64) | (1u << 16);         // B with its rows (keys) along K
      auto desc_lo = [&](uint32_t off) { return ((smem_u32(smem + off) & 0x3FFFFu) >> 4) | (1u << 16); };
      const uint32_t q = desc_lo(L.q + (halves ? t : 0) * kTileBytes), k0 = desc_lo(L.k), v0 = desc_lo(L.v);
      auto at = [&](int i) { return halves ? i : 2 * i + t; };
      for (int i = 0; i <= mine; ++i) {
        if (i < mine) {
          const int j = at(i), slot = j % SLOTS;
          ok = ok && (i > 0 || mbar_wait(q_full + (halves ? t : 0), 0, polls)) && mbar_wait(k_full + slot, (j / SLOTS) & 1, polls) &&
               (i == 0 || mbar_wait(s_read + t, (i - 1) & 1, polls));
          tc_fence_after_sync();
          if (elect_one() && ok) {
            umma_f16_x4(tmem + tile_s_col(t), q, k0 + slot * (kTileBytes >> 4), idesc_s);
            umma_commit(s_full + t);
            umma_commit(k_free + slot);
          }
          __syncwarp();
        }
        if (i > 0) {
          const int j = at(i - 1), slot = j % SLOTS;
          ok = ok && mbar_wait(v_full + slot, (j / SLOTS) & 1, polls) && mbar_wait(p_full + t, (i - 1) & 1, polls);
          tc_fence_after_sync();
          if (elect_one() && ok) {
#pragma unroll
            for (int k = 0; k < kTileKeys; k += 16)
              umma_f16_tmem_a_lo(tmem + tile_o_col(t), tmem + tile_p_col(t) + (k >> 1), v0 + slot * (kTileBytes >> 4) + 8 * k, idesc_o,
                                 i > 1 || k > 0 ? 1u : 0u);
            umma_commit(o_done + t);
            umma_commit(v_free + slot);
          }
          __syncwarp();
        }
      }
    }
    __syncwarp();
  } else if (warp >= kLoad) {
    // ------------------------------------------------------------------ keys and values: a warp 32 keys of a tile
    if constexpr (STREAMS > 1) fewer_registers<kTileLoadRegs>();
    const int w = warp - kLoad;
    const uint32_t k_smem = smem_u32(smem) + L.k + w * 4096, v_smem = smem_u32(smem) + L.v + w * 4096;
    // where the two sixteens of keys of the warp lie, each in one page; looked up two tiles ahead, as are the masks
    int page[2] = {0, 0}, page_after[2] = {0, 0};
    bool masked = true, masked_after = true;
    auto look_up = [&](int j, int (&page)[2], bool& masked) {
      masked = true;
      const int base = (first + j) * kTileKeys + 32 * w;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        page[u] = b;
        if (p.table != nullptr && base + 16 * u < keys) page[u] = p.table[static_cast<long long>(b) * p.table_width + ((base + 16 * u) >> p.page_shift)];
      }
      if (!PACKED && p.mask != nullptr) masked = base + lane < keys && p.mask[b * p.mask_stride + base + lane] != 0;
    };
    struct Place {
      long long k[2], v[2], stats[2];
      uint32_t seen;
    };
    auto place = [&](int j) {
      Place pl;
      const int base = (first + j) * kTileKeys + 32 * w;
      bool there[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int in = p.table != nullptr ? (base + 16 * u) & ((1 << p.page_shift) - 1) : base + 16 * u;
        there[u] = base + 16 * u < keys && (p.table == nullptr || (page[u] >= 0 && page[u] < p.pages));
        if (PACKED) {
          pl.stats[u] = ((static_cast<long long>(page[u]) * p.kv_heads + kvh) << p.page_shift) + in;
        } else {
          pl.k[u] = page[u] * p.k.block_stride + kvh * p.k.head_stride + in * p.k.token_stride;
          pl.v[u] = page[u] * p.v.block_stride + kvh * p.v.head_stride + in * p.v.token_stride;
        }
      }
      pl.seen = __ballot_sync(0xffffffffu, base + lane < keys && (lane < 16 ? there[0] : there[1]) && masked);
      if (lane == 0) s_seen[j % kTileSeen * 4 + w] = pl.seen;
      page[0] = page_after[0];
      page[1] = page_after[1];
      masked = masked_after;
      if (j + 2 < count) look_up(j + 2, page_after, masked_after);
      return pl;
    };
    // a slot's phase that the products have to have ended
    auto wait_free = [&](uint64_t* bar, int j) {
      if (j >= SLOTS) ok = mbar_wait(bar + j % SLOTS, (j / SLOTS - 1) & 1, polls) && ok;
    };
    auto hand_over = [&](uint64_t* bar) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    if (count > 0) look_up(0, page, masked);
    if (count > 1) look_up(1, page_after, masked_after);
    if (count == 0) set_up();
    if constexpr (!PACKED) {
      // 16 bits: eight lanes a row, asynchronous copies.  A tile is handed over before a slot is waited for: the slot may be freed by a product
      // that is issued behind one with that tile.  Where the slots are free already, the copies go first.
      auto copy = [&](const AttendView& a, const long long (&from)[2], uint32_t seen, uint32_t dst) {
        const uint32_t row0 = lane >> 3, ch = lane & 7;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint8_t* const src = a.rows + from[u] + row0 * a.token_stride + 16 * ch;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t row = 16 * u + 4 * r + row0, to = dst + row * 128 + ((ch ^ (row & 7)) << 4);
            if (seen == 0xffffffffu) cp_async_16(to, src + r * 4 * a.token_stride);
            else cp_async_16(to, (seen >> row) & 1 ? src + r * 4 * a.token_stride : a.rows, (seen >> row) & 1);
          }
        }
        cp_async_commit();
      };
      for (int j = 0; j < count; ++j) {
        const Place pl = place(j);
        const int slot = j % SLOTS, before = (j + SLOTS - 1) % SLOTS;
        bool pending = j > 0;
        if (pending && j >= SLOTS &&
            !__all_sync(0xffffffffu, mbar_test_wait(k_free + slot, (j / SLOTS - 1) & 1) && mbar_test_wait(v_free + slot, (j / SLOTS - 1) & 1))) {
          cp_async_wait<1>();
          hand_over(k_full + before);
          cp_async_wait<0>();
          hand_over(v_full + before);
          pending = false;
        }
        wait_free(k_free, j);
        copy(p.k, pl.k, pl.seen, k_smem + slot * kTileBytes);
        wait_free(v_free, j);
        copy(p.v, pl.v, pl.seen, v_smem + slot * kTileBytes);
        if (j == 0) set_up();
        if (pending) {
          cp_async_wait<3>();
          hand_over(k_full + before);
          cp_async_wait<2>();
          hand_over(v_full + before);
        }
      }
      if (count > 0) {
        cp_async_wait<1>();
        hand_over(k_full + (count - 1) % SLOTS);
        cp_async_wait<0>();
        hand_over(v_full + (count - 1) % SLOTS);
      }
    } else {
      // packed: a lane has a key's row, eight values of it at a time
      const uint32_t k_table = smem_u32(smem) + L.tables + lane * 4, v_table = smem_u32(smem) + L.tables + kPairTableBytes + (lane & 15) * 8;
      const uint32_t row = lane * 128, x7 = lane & 7;
      struct Row {
        uint32_t w[2 * BITS], stats;
      };
      auto load_row = [&](const AttendView& a, long long at, bool is, Row& r) {
        const uint2* const src = reinterpret_cast<const uint2*>(a.rows + at * (8 * BITS));
#pragma unroll
        for (int i = 0; i < BITS; ++i) {
          const uint2 u = is ? src[i] : make_uint2(0, 0);
          r.w[2 * i] = u.x; r.w[2 * i + 1] = u.y;
        }
        r.stats = is ? *reinterpret_cast<const uint32_t*>(a.stats + at) : 0;
      };
      // the codes of values 8c .. 8c + 7, one per nibble
      auto codes = [](const Row& r, int c) {
        if (BITS == 4) return r.w[c];
        if (BITS == 2) return spread_codes<2>((c & 1) ? r.w[c >> 1] >> 16 : r.w[c >> 1] & 0xFFFFu);
        const uint32_t* const w = r.w + 3 * (c >> 2);                             // 24 bits each, four of them in three words
        switch (c & 3) {
          case 0: return spread_codes<3>(w[0] & 0xFFFFFFu);
          case 1: return spread_codes<3>(__funnelshift_r(w[0], w[1], 24) & 0xFFFFFFu);
          case 2: return spread_codes<3>(__funnelshift_r(w[1], w[2], 16) & 0xFFFFFFu);
          default: return spread_codes<3>(w[2] >> 8);
        }
      };
      auto write_keys = [&](uint32_t dst, const Row& r) {
        const uint32_t center = __byte_perm(r.stats, 0, 0x1010), scale = __byte_perm(r.stats, 0, 0x3232);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t l[4];
          pair_levels(k_table, codes(r, c), l);
          sts128(dst + ((static_cast<uint32_t>(c) ^ x7) << 4), half2_fma(scale, l[0], center), half2_fma(scale, l[1], center),
                 half2_fma(scale, l[2], center), half2_fma(scale, l[3], center));
        }
      };
      auto write_values = [&](uint32_t dst, const Row& r) {
        const f32x2 center = sixteen_to_pair<__half>(__byte_perm(r.stats, 0, 0x1010)), scale = sixteen_to_pair<__half>(__byte_perm(r.stats, 0, 0x3232));
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          f32x2 l[4];
          pair_levels_f32(v_table, codes(r, c), l);
          uint32_t w[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) w[n] = pair_to_sixteen<__half>(fma2(scale, l[n], center));
          sts128(dst + ((static_cast<uint32_t>(c) ^ x7) << 4), w[0], w[1], w[2], w[3]);
        }
      };
      Row kr, vr;
      auto fetch = [&](int j) {
        const Place pl = place(j);
        const long long at = pl.stats[lane >> 4] + (lane & 15);
        const bool is = (pl.seen >> lane) & 1;
        load_row(p.k, at, is, kr);
        load_row(p.v, at, is, vr);
      };
      if (count > 0) {
        fetch(0);
        set_up();
      }
      for (int j = 0; j < count; ++j) {
        const int slot = j % SLOTS;
        const Row k = kr, v = vr;
        if (j + 1 < count) fetch(j + 1);
        wait_free(k_free, j);
        write_keys(k_smem + slot * kTileBytes + row, k);
        hand_over(k_full + slot);
        wait_free(v_free, j);
        // Values that are NaN are left out of the products, where 0 * NaN would show in rows that do not see them; those that do get it below.
        Row used = v;
        if ((v.stats & 0x7C00u) == 0x7C00u || (v.stats & 0x7C000000u) == 0x7C000000u) {
          used.stats = 0;
          atomicMin(s_first_bad, (first + j) * kTileKeys + 32 * w + lane);
        }
        write_values(v_smem + slot * kTileBytes + row, used);
        hand_over(v_full + slot);
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax: a thread a row
    if constexpr (STREAMS > 1) more_registers<kTileSoftmaxRegs>();
    const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const int at = row0 + (halves ? t * kTileRows : 0) + r;                       // of the sequence's rows
    const bool live = at < row0 + rows;
    const int limit = !live ? 0 : p.causal ? min(seq.keys, max(seq.keys - seq.all_queries + at / p.group + 1, 0)) : seq.keys;
    // ---- the queries, eight lanes a row: a stream its own, without halves (the second stream's are the first's) both half of them; what their
    // products are scaled by goes through s_max
    {
      uint4 u[8];
      const int c = lane & 7, of = halves ? 8 : 4, first_row = halves ? t * kTileRows : t * 64;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int q = first_row + k * 16 + quarter * 4 + (lane >> 3), row = row0 + q;
        u[k] = make_uint4(0, 0, 0, 0);
        if (k < of && q < rows) u[k] = reinterpret_cast<const uint4*>(attend_query(p, seq, b, row / p.group, kvh * p.group + row % p.group))[c];
      }
      fill_tables(tid);
      set_up();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (k >= of) break;
        const int q = first_row + k * 16 + quarter * 4 + (lane >> 3);
        float factor = p.scale_log2;
        if (PACKED && p.q_bf16) {
          uint32_t w[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
          float largest = bf16_top(w, 4);
#pragma unroll
          for (int d = 1; d < 8; d <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, d));
          factor *= bf16_to_half(w, 4, largest);
          u[k] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        sts128(smem_u32(smem) + L.q + q * 128 + ((c ^ (q & 7)) << 4), u[k].x, u[k].y, u[k].z, u[k].w);
        if (c == 0) s_max[q] = factor;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full + (halves ? t : 0));
    }
    asm volatile("bar.sync 1, %0;" ::"n"(128 * STREAMS) : "memory");
    const float scale = s_max[halves ? t * kTileRows + r : r];
    const uint32_t tmem = *s_tmem;
    asm volatile("bar.sync 1, %0;" ::"n"(128 * STREAMS) : "memory");           // all have read theirs: s_max is free again
    const int mine = halves ? count : (count + 1 - t) / 2;
    const float ninf = __int_as_float(0xff800000);
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_at = tmem + tile_s_col(t) + lanes, p_at = tmem + tile_p_col(t) + lanes, o_at = tmem + tile_o_col(t) + lanes;
    const bool rows_here = __any_sync(0xffffffffu, live);
    float top = ninf;                                                             // in units of the exponent
    f32x2 sum0 = pack2(0.0f, 0.0f), sum1 = sum0;
    // The streams take turns at the exponentials (barrier 2 + t is stream t's turn): while one has their pipe to itself, the other waits for its
    // products, reads its scores and finds the maximum.  Left alone they fall into step, and the pipe idles during all of that: 3720 cycles
    // a tile of keys (both streams), in turns 3170, of which the exponentials of a stream take 1500.
    // A stream has as many turns as tiles; the second has as many as the first or one fewer.
    auto my_turn = [&] { if constexpr (STREAMS > 1) asm volatile("bar.sync %0, 256;" ::"r"(2 + t) : "memory"); };
    auto your_turn = [&] { if constexpr (STREAMS > 1) asm volatile("bar.arrive %0, 256;" ::"r"(3 - t) : "memory"); };
    if (t == 1) your_turn();
    for (int i = 0; i < mine; ++i) {
      const int j = halves ? i : 2 * i + t;
      ok = ok && mbar_wait_warp(s_full + t, i & 1, polls);
      tc_fence_after_sync();
      if (rows_here && ok) {
        const uint4 seen = lds128(smem_u32(s_seen + j % kTileSeen * 4));
        // One stream's threads, with 96 registers, hold a quarter of a row's scores at a time and read three of the quarters twice.
        constexpr int PART = STREAMS == 1 ? 1 : 4, PARTS = 4 / PART;
        uint32_t s[PART][32];
        auto read_scores = [&](int part, bool last) {
#pragma unroll
          for (int c = 0; c < PART; ++c) tmem_ld_32x32(s_at + 32 * (part * PART + c), s[c]);
          tmem_ld_wait();
          if (last) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_read + t);
          }
        };
        const int base = (first + j) * kTileKeys;
        bool all_seen = false;
        auto hide_unseen = [&](int part) {
          if (all_seen) return;
          const uint32_t words[4] = {seen.x, seen.y, seen.z, seen.w};
#pragma unroll
          for (int c = 0; c < PART; ++c) {
            const uint32_t of = PART == 4 ? words[c] : s_seen[j % kTileSeen * 4 + part * PART + c];
            const int left = limit - base - 32 * (part * PART + c);               // keys of the 32 that the row may see
            const uint32_t word = of & (left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u);
#pragma unroll
            for (int n = 0; n < 32; ++n) s[c][n] = (word >> n) & 1 ? s[c][n] : 0xff800000u;
          }
        };
        // ---- maximum
        float m0 = ninf, m1 = ninf, m2 = ninf, m3 = ninf;
#pragma unroll 1
        for (int part = 0; part < PARTS; ++part) {
          read_scores(part, PARTS == 1);
          if (part == 0) {
            __syncwarp();
            all_seen = __all_sync(0xffffffffu, (seen.x & seen.y & seen.z & seen.w) == 0xffffffffu && base + kTileKeys <= limit);
          }
          hide_unseen(part);
#pragma unroll
          for (int n = 0; n < 32; n += 2) {
            float& m = PART == 1 && (n & 2) ? m1 : m0;
            m = max3(m, __uint_as_float(s[0][n]), __uint_as_float(s[0][n + 1]));
            if constexpr (PART == 4) {
              m1 = max3(m1, __uint_as_float(s[1][n]), __uint_as_float(s[1][n + 1]));
              m2 = max3(m2, __uint_as_float(s[2][n]), __uint_as_float(s[2][n + 1]));
              m3 = max3(m3, __uint_as_float(s[3][n]), __uint_as_float(s[3][n + 1]));
            }
          }
        }
        const float m = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * scale;
        // the probabilities' columns are free, and the output may be scaled, once the last product has ended
        if (i > 0) ok = ok && mbar_wait_warp(o_done + t, (i - 1) & 1, polls);
        tc_fence_after_sync();
        const bool renew = m > top + 8.0f || (top == ninf && m > ninf);
        if (__any_sync(0xffffffffu, renew) && ok) {
          const float next = renew ? m : top;
          const float f = renew ? exp2_approx(top - next) : 1.0f;
          top = next;
          const f32x2 f2 = pack2(f, f);
          sum0 = mul2(sum0, f2);
          sum1 = mul2(sum1, f2);
          if (i > 0) {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              uint32_t o[16];
              tmem_ld_32x16(o_at + 16 * h, o);
              tmem_ld_wait();
#pragma unroll
              for (int n = 0; n < 16; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * f);
              tmem_st_32x16(o_at + 16 * h, o);
            }
          }
        }
        my_turn();
        const float nm = top == ninf ? 0.0f : -top;
        const f32x2 scale2 = pack2(scale, scale), nm2 = pack2(nm, nm);
#pragma unroll 1
        for (int part = PARTS - 1; part >= 0; --part) {
          if (part < PARTS - 1) {
            read_scores(part, part == 0);
            hide_unseen(part);
          }
#pragma unroll
          for (int c = 0; c < PART; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int n = 0; n < 16; ++n) {
              float x, y;
              unpack2(fma2(pack2(__uint_as_float(s[c][2 * n]), __uint_as_float(s[c][2 * n + 1])), scale2, nm2), x, y);
              const f32x2 e = pack2(exp2_approx(x), exp2_approx(y));
              if (n & 1) sum1 = add2(sum1, e); else sum0 = add2(sum0, e);
              w[n] = pair_to_sixteen<E>(e);
            }
            tmem_st_32x16(p_at + 16 * (part * PART + c), w);
          }
        }
        your_turn();
        tmem_st_wait();
      } else {
        __syncwarp();
        if (lane == 0) mbar_arrive(s_read + t);
        if (i > 0 && ok) ok = mbar_wait_warp(o_done + t, (i - 1) & 1, polls);
        my_turn();
        your_turn();
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + t);
    }
    // ---- the stream's part: maximum, sum and output, as they are
    if (mine > 0) ok = ok && mbar_wait_warp(o_done + t, (mine - 1) & 1, polls);
    tc_fence_after_sync();
    float x, y;
    unpack2(add2(sum0, sum1), x, y);
    s_max[t * kTileRows + r] = top;
    s_sum[t * kTileRows + r] = PACKED && *s_first_bad < limit ? __int_as_float(0x7fffffff) : x + y;
  }
  // ---------------------------------------------------------------------- join and write
  // All copies into the key and value slots have landed (their products have ended) or nobody waits for them any more.
  tc_fence_before_sync();
  const bool gave_up = __syncthreads_or(!ok) != 0;
  tc_fence_after_sync();
  const uint32_t tmem = *s_tmem;
  if (gave_up && tid == kIssue * 32) atomicExch(p.status, kStatusTileAttentionTimeout);
  float* const part = reinterpret_cast<float*>(smem + L.k);                       // [stream][row][64], over the slots, 16-byte chunks swizzled by row
  const bool many = p.splits > 1, direct = halves && !many;                       // a row's result is in one place
  if (warp < kLoad) {
    const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane, at = row0 + t * kTileRows + r;
    const int mine = halves ? count : (count + 1 - t) / 2;
    const float inv = direct ? inverse_sum(s_sum[t * kTileRows + r]) : 0.0f;
    uint16_t* const dst = static_cast<uint16_t*>(p.out) +
                          ((static_cast<long long>(seq.first_row) + at / p.group) * p.heads + kvh * p.group + at % p.group) * 64;
    const uint32_t o_at = tmem + tile_o_col(t) + (static_cast<uint32_t>(quarter * 32) << 16);
    const bool none = s_max[t * kTileRows + r] == __int_as_float(0xff800000);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t o[32];
      if (mine > 0 && !gave_up) {
        tmem_ld_32x32(o_at + 32 * h, o);
        tmem_ld_wait();
      }
#pragma unroll
      for (int n = 0; n < 32; n += 4) {
        uint4 u = make_uint4(o[n], o[n + 1], o[n + 2], o[n + 3]);
        if (mine <= 0 || gave_up || none) u = make_uint4(0, 0, 0, 0);
        o[n] = u.x; o[n + 1] = u.y; o[n + 2] = u.z; o[n + 3] = u.w;
        if (!direct) sts128(smem_u32(part) + (t * kTileRows + r) * 256 + (((h * 8 + (n >> 2)) ^ (r & 7)) << 4), u.x, u.y, u.z, u.w);
      }
      if (direct && at < row0 + rows) {
#pragma unroll
        for (int n = 0; n < 32; n += 8) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x2 x = pack2(__uint_as_float(o[n + 2 * i]) * inv, __uint_as_float(o[n + 2 * i + 1]) * inv);
            w[i] = p.q_bf16 ? pair_to_sixteen<__nv_bfloat16>(x) : pair_to_sixteen<__half>(x);
          }
          *reinterpret_cast<uint4*>(dst + 32 * h + n) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (gave_up && warp >= kIssue && warp < kIssue + STREAMS) {                                    // products that nobody waited for end before their memory is given back
    if (elect_one()) umma_commit(stopped);
    __syncwarp();
    mbar_wait(stopped, 0);
    __syncwarp();
  }
  if (warp == kIssue) tmem_dealloc(tmem, 256 * STREAMS);
  if (many) asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  // The rows are shared out over the blocks of the cluster: first what each part counts in a row and where the row goes, then four values a
  // thread.
  if (!direct) {
    const int share = (rows + p.splits - 1) / p.splits, from = min(split * share, rows), mine = min(share, rows - from);
    const int parts = (halves ? 1 : 2) * p.splits;
    auto address = [&](int q, int r, uint32_t offset, int row_bytes) {
      const int rank = halves ? q : q >> 1, t = halves ? r >> 7 : q & 1;
      uint32_t d;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_u32(smem) + offset + (t * kTileRows + (r & 127)) * row_bytes), "r"(rank));
      return d;
    };
    if (tid < mine) {
      const int r = from + tid, at = row0 + r;
      float m = __int_as_float(0xff800000), l = 0.0f;
#pragma unroll 1
      for (int q = 0; q < parts; ++q) m = fmaxf(m, lds_cluster(address(q, r, L.max, 4)));
      const float base = m == __int_as_float(0xff800000) ? 0.0f : m;
#pragma unroll 1
      for (int q = 0; q < parts; ++q) {
        const float f = exp2_approx(lds_cluster(address(q, r, L.max, 4)) - base);
        l += f * lds_cluster(address(q, r, L.sum, 4));
        s_weight[tid * parts + q] = f;
      }
      const float inv = inverse_sum(l);
#pragma unroll 1
      for (int q = 0; q < parts; ++q) s_weight[tid * parts + q] *= inv;
      s_offset[tid] = ((static_cast<long long>(seq.first_row) + at / p.group) * p.heads + kvh * p.group + at % p.group) * 64;
    }
    __syncthreads();
    for (int e = tid; e < mine * 16; e += kThreads) {
      const int i = e >> 4, r = from + i, c = e & 15;
      float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 2
      for (int q = 0; q < parts; ++q) {
        const float f = s_weight[i * parts + q];
        const float4 v = lds128_cluster(address(q, r, L.k, 256) + ((c ^ (r & 7)) << 4));
        o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
      }
      const f32x2 lo = pack2(o.x, o.y), hi = pack2(o.z, o.w);
      const uint2 u = p.q_bf16 ? make_uint2(pair_to_sixteen<__nv_bfloat16>(lo), pair_to_sixteen<__nv_bfloat16>(hi))
                               : make_uint2(pair_to_sixteen<__half>(lo), pair_to_sixteen<__half>(hi));
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + s_offset[i] + 4 * c) = u;
    }
  }
  __syncwarp();
  if (many) asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

}  // namespace arcq
