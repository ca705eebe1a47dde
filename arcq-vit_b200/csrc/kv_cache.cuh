// A key/value cache in pages, in the ARCQ format or in 16 bits: writing new tokens and reading tokens back by their slots.
//
// A page holds `page` tokens (a power of two, 16 or more) of every key/value head: keys and values apart, [pages, heads, page, row].
// A row is a head's 64 values of one token: 128 bytes in 16 bits, or one quantizer group of 2, 3 or 4 bits (8 * bits bytes of codes) with
// a pair (center, scale) beside it, [pages, heads, page, 2] fp16.  Heads before tokens: a query reads the tokens of one head, which then
// lie one after the other, a page at a time.
//   scale, codes  those of the activation quantizer, bit for bit
//   center        mean - scale * code_sum / 64
//   value         center + scale * level
// Center and scale are rounded to fp16: 2^-11 of a value, against quantization steps of 0.1 (4 bits) to 0.6 scale, for 36 instead of 40
// bytes a row; a center or scale beyond fp16's range is held at its end.  A group with a NaN or an infinity has a NaN for both (the mean is not
// finite, so the scale is NaN, and with it the center): all of its 64 values are read back as NaN.
// A slot is page * page_size + place in it; tokens whose slot is negative or beyond the cache are neither written nor read (zeros).
#pragma once
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>
#include <type_traits>
#include "ptx.cuh"
#include "f32x2.cuh"
#include "element_types.cuh"
#include "act_quant.cuh"
#include "group_quant.cuh"

namespace arcq {

struct KvPages {
  uint8_t* pages;          // keys or values
  __half2* stats;          // null in 16 bits
  const float* levels;     // 2^bits
  const float* thresholds; // writing only
  const void* x;           // writing: [tokens, heads, 64]
  void* out;               // reading: the same, contiguous
  long long token_stride, head_stride;   // of x, in values
};
struct KvCacheParams {
  KvPages kv[2];
  const long long* slots;
  long long tokens, slot_count;
  int heads, page_shift;
};

// Row of the cache that a token's head has: (page * heads + head) * page_size + place
__device__ __forceinline__ long long kv_row(long long slot, int head, int heads, int page_shift) {
  const long long page = slot >> page_shift;
  return ((page * heads + head) << page_shift) + (slot & ((1ll << page_shift) - 1));
}

// held to fp16's range; NaN stays NaN (fmaxf would drop it)
__device__ __forceinline__ __half kv_half(float v) { return __float2half_rn(v == v ? fminf(fmaxf(v, -65504.0f), 65504.0f) : v); }

// 8 codes of BITS bits, one per nibble
template <int BITS> __device__ __forceinline__ uint32_t spread_codes(uint32_t x) {
  if (BITS == 4) return x;
  if (BITS == 3) {
    x = (x & 0xFFFu) | ((x & 0xFFF000u) << 4);
    x = (x & 0x003F003Fu) | ((x & 0x0FC00FC0u) << 2);
    return (x & 0x07070707u) | ((x & 0x38383838u) << 1);
  }
  x = (x & 0xFFu) | ((x & 0xFF00u) << 8);
  x = (x & 0x000F000Fu) | ((x & 0x00F000F0u) << 4);
  return (x & 0x03030303u) | ((x & 0x0C0C0C0Cu) << 2);
}

// ---------------------------------------------------------------- codebooks and thresholds
// What a write needs may have been fitted by the kernel before.  kv_write_kernel reads it behind the wait, with its first rows.
// kv_write_tile_kernel makes its tables while that kernel may still run all the same; behind the wait the threads that read the values for them do
// so once more, past the first-level cache, and where one is different the block makes the tables anew: 16 384 tokens of 12 heads in 4 bits 24.2 ->
// 24.8 us, 25.5 with tables made behind the wait.  Reads of the cache and attention come behind a write, and read codebooks early.
__device__ __forceinline__ float load_settled(const float* at) {
  float v;
  asm volatile("ld.relaxed.gpu.global.f32 %0, [%1];" : "=f"(v) : "l"(at) : "memory");
  return v;
}
__device__ __forceinline__ bool other_bits(float a, float b) { return __float_as_uint(a) != __float_as_uint(b); }

// ---------------------------------------------------------------- writing
// Eight lanes a group, four groups a warp; blockIdx.y: keys or values.
template <typename T, int BITS>
__global__ void __launch_bounds__(256) kv_write_kernel(const __grid_constant__ KvCacheParams p) {
  pdl_launch_dependents();
  constexpr int L = 1 << BITS;
  __shared__ float s_th[16], s_cb[16];
  const KvPages& kv = p.kv[blockIdx.y];
  const int lane = threadIdx.x & 31, l = lane & 7, octet = lane & ~7;
  const long long groups = p.tokens * p.heads, warps = static_cast<long long>(gridDim.x) * 8;
  pdl_wait();
  float v[8], level[8];
  long long slot = -1;
  int head = 0;
  auto fetch = [&](long long task) {
    const long long g = min(task * 4 + (lane >> 3), groups - 1);             // octets without a group shadow the last one
    const long long token = g / p.heads;
    head = static_cast<int>(g - token * p.heads);
    slot = p.slots[token];
    const T* const x = static_cast<const T*>(kv.x) + token * kv.token_stride + head * kv.head_stride + l;
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] = load_f32<T>(x + 8 * c);
  };
  long long task = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  float th = __int_as_float(0x7f800000), cb = 0.0f;
  if (threadIdx.x < L - 1) th = kv.thresholds[threadIdx.x];
  if (threadIdx.x < L) cb = kv.levels[threadIdx.x];
  fetch(task);
  if (threadIdx.x < 16) {
    s_th[threadIdx.x] = th;
    s_cb[threadIdx.x] = cb;
  }
  __syncthreads();
  while (task * 4 < groups) {
    const bool valid = task * 4 + (lane >> 3) < groups && slot >= 0 && slot < p.slot_count;
    uint32_t w;
    const OctetStats st = octet_quantize<BITS>(v, s_th, s_cb, octet, level, w);
    w = octet_transpose_nibbles(w, l);
    const long long row = valid ? kv_row(slot, head, p.heads, p.page_shift) : 0;
    uint32_t* const codes = reinterpret_cast<uint32_t*>(kv.pages + row * (8 * BITS));
    if (BITS == 4) {
      if (valid) codes[l] = w;
    } else if (BITS == 3) {
      const uint32_t v24 = squeeze_nibbles_3(w);
      const int q = (4 * l) / 3, r = (4 * l) % 3;
      const uint32_t lo = __shfl_sync(0xffffffffu, v24, octet + (q & 7)), hi = __shfl_sync(0xffffffffu, v24, octet + ((q + 1) & 7));
      if (valid && l < 6) codes[l] = (lo >> (8 * r)) | (hi << (24 - 8 * r));
    } else {
      const uint32_t v16 = squeeze_nibbles_2(w);
      const uint32_t lo = __shfl_sync(0xffffffffu, v16, octet + ((2 * l) & 7)), hi = __shfl_sync(0xffffffffu, v16, octet + ((2 * l + 1) & 7));
      if (valid && l < 4) codes[l] = lo | (hi << 16);
    }
    if (valid && l == 0)
      kv.stats[row] = __halves2half2(kv_half(__fmaf_rn(-st.scale, __fmul_rn(st.code_sum, 0.015625f), st.mean)), kv_half(st.scale));
    task += warps;
    if (task * 4 < groups) fetch(task);
  }
}

// Many tokens, 16-bit values: a lane a group (group_quant.cuh), 32 groups a warp and step, the next step's rows on their way meanwhile.  Eight
// lanes copy a row, so a row may lie anywhere; codes and statistics leave from registers, a full 32-byte sector of codes a row in 4 bits.
// Bound by the quantizer's issue slots like the kernels that it shares them with: 16 384 tokens of 12 heads in 4 bits (50 MB in, 14 MB out)
// 24.8 us, 61 with the octets of kv_write_kernel.
constexpr int kWriteWarps = 4, kWriteThreads = kWriteWarps * 32;
constexpr uint32_t kWriteTables = kWriteWarps * 2 * 4096;
constexpr uint32_t kWriteSmem = 1024 + kWriteTables + (sizeof(GroupQuantTables) + 15) / 16 * 16;
template <typename T, int BITS>
__global__ void __launch_bounds__(kWriteThreads, 4) kv_write_tile_kernel(const __grid_constant__ KvCacheParams p) {
  pdl_launch_dependents();
  extern __shared__ uint8_t kv_smem_raw[];
  uint8_t* const smem = kv_smem_raw + ((1024u - (smem_u32(kv_smem_raw) & 1023u)) & 1023u);
  GroupQuantTables* const tables = reinterpret_cast<GroupQuantTables*>(smem + kWriteTables);
  const KvPages& kv = p.kv[blockIdx.y];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bufs = smem_u32(smem) + warp * 8192;
  const long long groups = p.tokens * p.heads, stride = static_cast<long long>(gridDim.x) * kWriteWarps * 32;
  const T* const x = static_cast<const T*>(kv.x);
  // what the lane has to know of its group, and the copies of the warp's 32 rows
  struct Group {
    long long slot;
    int head;
  };
  auto fetch = [&](long long first, uint32_t buf) {
    Group g;
    const long long i = min(first + lane, groups - 1), token = i / p.heads;        // lanes without a group shadow the last one
    g.head = static_cast<int>(i - token * p.heads);
    g.slot = first + lane < groups ? p.slots[token] : -1;
    const unsigned long long row = reinterpret_cast<unsigned long long>(x + token * kv.token_stride + g.head * kv.head_stride);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int of = 4 * r + (lane >> 3), c = lane & 7;
      const unsigned long long src = __shfl_sync(0xffffffffu, row, of) + 16 * c;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(buf + of * 128 + ((c ^ (of & 7)) << 4)), "l"(src) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    return g;
  };
  long long first = (static_cast<long long>(blockIdx.x) * kWriteWarps + warp) * 32;
  int buf = 0;
  constexpr int L = 1 << BITS;
  auto make_tables = [&] {
    return group_quant_tables<L, true>(tables, kv.thresholds, kv.levels, tid, kWriteThreads, [](bool b) { return __syncthreads_and(b) != 0; },
                                       [](const float* at) { return load_settled(at); });
  };
  GroupQuantParams gp = make_tables();
  pdl_wait();
  if (__syncthreads_or((tid < L - 1 && other_bits(load_settled(kv.thresholds + tid), tables->th[tid])) ||
                       (tid < L && other_bits(load_settled(kv.levels + tid), tables->cb[tid]))))
    gp = make_tables();
  if (first >= groups) return;
  Group now = fetch(first, bufs), next = now;
  for (; first < groups; first += stride) {
    const bool more = first + stride < groups;
    if (more) {
      next = fetch(first + stride, bufs + (buf ^ 1) * 4096);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    uint32_t w[32], words[8];
    f32x2 v[32];
    row_load<1>(w, bufs + buf * 4096 + lane * 128, lane & 7);
    __syncwarp();                                                                  // the rows have been read
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = sixteen_to_pair<T>(w[i]);
    const GroupStats st = group_quantize<BITS, true, 1>(v, tables, gp, words);
    if (now.slot >= 0 && now.slot < p.slot_count) {
      const long long row = kv_row(now.slot, now.head, p.heads, p.page_shift);
      uint8_t* const out = kv.pages + row * (8 * BITS);
      if constexpr (BITS == 4) {
        reinterpret_cast<uint4*>(out)[0] = make_uint4(words[0], words[1], words[2], words[3]);
        reinterpret_cast<uint4*>(out)[1] = make_uint4(words[4], words[5], words[6], words[7]);
      } else if constexpr (BITS == 3) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {                                              // four chunks of 24 bits: three words
          const uint32_t a = squeeze_nibbles_3(words[4 * h]), b = squeeze_nibbles_3(words[4 * h + 1]);
          const uint32_t c = squeeze_nibbles_3(words[4 * h + 2]), d = squeeze_nibbles_3(words[4 * h + 3]);
          const uint32_t o[3] = {a | (b << 24), (b >> 8) | (c << 16), (c >> 16) | (d << 8)};
          for (int j = 0; j < 3; ++j) reinterpret_cast<uint32_t*>(out)[3 * h + j] = o[j];
        }
      } else {
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = squeeze_nibbles_2(words[2 * j]) | (squeeze_nibbles_2(words[2 * j + 1]) << 16);
        *reinterpret_cast<uint4*>(out) = make_uint4(o[0], o[1], o[2], o[3]);
      }
      kv.stats[row] = __halves2half2(kv_half(__fmaf_rn(-st.scale, __fmul_rn(st.code_sum, 0.015625f), st.mean)), kv_half(st.scale));
    }
    now = next;
    buf ^= 1;
  }
}

// 16 bits: a copy, 16 bytes a thread.  16 384 tokens of 12 heads (50 MB in and out each) 20.2 us, 15.4 at the copy bandwidth.
__global__ void __launch_bounds__(256) kv_write_copy_kernel(const __grid_constant__ KvCacheParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const KvPages& kv = p.kv[blockIdx.y];
  const long long chunks = p.tokens * p.heads * 8, step = static_cast<long long>(gridDim.x) * 256;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < chunks; i += step) {
    const long long g = i >> 3, token = g / p.heads;
    const int head = static_cast<int>(g - token * p.heads), c = static_cast<int>(i & 7);
    const long long slot = p.slots[token];
    if (slot < 0 || slot >= p.slot_count) continue;
    const uint16_t* const x = static_cast<const uint16_t*>(kv.x) + token * kv.token_stride + head * kv.head_stride + 8 * c;
    *reinterpret_cast<uint4*>(kv.pages + kv_row(slot, head, p.heads, p.page_shift) * 128 + 16 * c) = __ldg(reinterpret_cast<const uint4*>(x));
  }
}

// ---------------------------------------------------------------- reading
__device__ __forceinline__ void store_32_bytes(void* out, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
               "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
template <typename O> __device__ __forceinline__ void store_sixteen(O* out, const float (&v)[16]) {
  uint32_t w[8];
  if constexpr (sizeof(O) == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(v[8 * h + j]);
      store_32_bytes(out + 8 * h, w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = pair_to_sixteen<O>(pack2(v[2 * j], v[2 * j + 1]));
    store_32_bytes(out, w);
  }
}

// Sixteen values a thread, a sector of the output in 16 bits.  BITS 16: pages of type T.  Levels come from a table of 16 in shared memory (as many
// banks, so no conflicts).  16 384 tokens of 12 heads in 4 bits (14 MB in, 50 MB out) one after the other 12.6 us, 16.5 with eight values a thread,
// where the addresses cost twice as much; all over the cache 14.0 us, in 16 bits (50 MB in) 19.1; 40 009 tokens of 3 heads in 3 bits, all over the
// cache, 9.2 us.
template <typename T, int BITS, typename O>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvCacheParams p) {
  pdl_launch_dependents();
  __shared__ float s_cb[16];
  const KvPages& kv = p.kv[blockIdx.y];
  if (BITS != 16 && threadIdx.x < 16) s_cb[threadIdx.x] = threadIdx.x < (1 << (BITS & 7)) ? kv.levels[threadIdx.x] : 0.0f;
  __syncthreads();
  pdl_wait();
  const long long pieces = p.tokens * p.heads * 4, step = static_cast<long long>(gridDim.x) * 256;
  const int c = threadIdx.x & 3;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < pieces; i += step) {
    const unsigned g = static_cast<unsigned>(i >> 2), token = g / static_cast<unsigned>(p.heads);
    const long long slot = p.slots[token];
    const bool is = slot >= 0 && slot < p.slot_count;
    const long long row = is ? kv_row(slot, static_cast<int>(g - token * p.heads), p.heads, p.page_shift) : 0;
    O* const out = static_cast<O*>(kv.out) + i * 16;
    float v[16] = {};
    if constexpr (BITS == 16) {
      const uint4* const src = reinterpret_cast<const uint4*>(kv.pages + row * 128 + 32 * c);
      const uint4 z = make_uint4(0, 0, 0, 0), a = is ? src[0] : z, b = is ? src[1] : z;
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      if constexpr (std::is_same<T, O>::value) {                                   // a copy, NaN's bits too
        store_32_bytes(out, w);
        continue;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) unpack2(sixteen_to_pair<T>(w[j]), v[2 * j], v[2 * j + 1]);
    } else if (is) {
      const uint8_t* const codes = kv.pages + row * (8 * BITS) + c * (2 * BITS);
      uint32_t lo, hi;
      if constexpr (BITS == 4) {
        const uint2 w = *reinterpret_cast<const uint2*>(codes);
        lo = w.x; hi = w.y;
      } else if constexpr (BITS == 3) {
        const uint16_t* const w = reinterpret_cast<const uint16_t*>(codes);
        const uint32_t x = w[0], y = w[1], z = w[2];
        lo = x | (y << 16);                                                        // 24 bits, and eight of the next
        hi = (y >> 8) | (z << 8);
      } else {
        lo = *reinterpret_cast<const uint32_t*>(codes);
        hi = lo >> 16;
      }
      const float2 st = __half22float2(kv.stats[row]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = __fmaf_rn(st.y, s_cb[(lo >> (BITS * j)) & ((1 << (BITS & 7)) - 1)], st.x);
        v[8 + j] = __fmaf_rn(st.y, s_cb[(hi >> (BITS * j)) & ((1 << (BITS & 7)) - 1)], st.x);
      }
    }
    store_sixteen(out, v);
  }
}

}  // namespace arcq
