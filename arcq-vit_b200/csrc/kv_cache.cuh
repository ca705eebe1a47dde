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
// bytes a row; a center or scale beyond fp16's range is held at its end.
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

__device__ __forceinline__ __half kv_half(float v) { return __float2half_rn(fminf(fmaxf(v, -65504.0f), 65504.0f)); }

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

// ---------------------------------------------------------------- writing
// Eight lanes a group, four groups a warp; blockIdx.y: keys or values.
template <typename T, int BITS>
__global__ void __launch_bounds__(256) kv_write_kernel(const __grid_constant__ KvCacheParams p) {
  pdl_launch_dependents();
  constexpr int L = 1 << BITS;
  __shared__ float s_th[16], s_cb[16];
  const KvPages& kv = p.kv[blockIdx.y];
  if (threadIdx.x < 16) {
    const int t = threadIdx.x;
    s_th[t] = t < L - 1 ? kv.thresholds[t] : __int_as_float(0x7f800000);
    s_cb[t] = t < L ? kv.levels[t] : 0.0f;
  }
  __syncthreads();
  pdl_wait();
  const int lane = threadIdx.x & 31, l = lane & 7, octet = lane & ~7;
  const long long groups = p.tokens * p.heads, warps = static_cast<long long>(gridDim.x) * 8;
  for (long long task = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); task * 4 < groups; task += warps) {
    const long long g = min(task * 4 + (lane >> 3), groups - 1);             // octets without a group shadow the last one
    const long long token = g / p.heads;
    const int head = static_cast<int>(g - token * p.heads);
    const long long slot = p.slots[token];
    const bool valid = task * 4 + (lane >> 3) < groups && slot >= 0 && slot < p.slot_count;
    const T* const x = static_cast<const T*>(kv.x) + token * kv.token_stride + head * kv.head_stride + l;
    float v[8], level[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] = load_f32<T>(x + 8 * c);
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
  }
}

// 16 bits: a copy, 16 bytes a thread
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
template <typename O> __device__ __forceinline__ void store_eight(O* out, const float (&v)[8]) {
  if (sizeof(O) == 4) {
    float4* const o = reinterpret_cast<float4*>(out);
    o[0] = make_float4(v[0], v[1], v[2], v[3]);
    o[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pair_to_sixteen<typename std::conditional<sizeof(O) == 4, __half, O>::type>(pack2(v[2 * j], v[2 * j + 1]));
    *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Eight values a thread.  BITS 16: pages of type T.
template <typename T, int BITS, typename O>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvCacheParams p) {
  pdl_launch_dependents();
  __shared__ float s_cb[16];
  const KvPages& kv = p.kv[blockIdx.y];
  if (BITS != 16 && threadIdx.x < 16) s_cb[threadIdx.x] = threadIdx.x < (1 << (BITS & 7)) ? kv.levels[threadIdx.x] : 0.0f;
  __syncthreads();
  pdl_wait();
  const long long chunks = p.tokens * p.heads * 8, step = static_cast<long long>(gridDim.x) * 256;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < chunks; i += step) {
    const long long g = i >> 3, token = g / p.heads;
    const int head = static_cast<int>(g - token * p.heads), c = static_cast<int>(i & 7);
    const long long slot = p.slots[token];
    float v[8] = {};
    if (slot >= 0 && slot < p.slot_count) {
      const long long row = kv_row(slot, head, p.heads, p.page_shift);
      if constexpr (BITS == 16) {
        const uint4 u = *reinterpret_cast<const uint4*>(kv.pages + row * 128 + 16 * c);
        if constexpr (std::is_same<T, O>::value) {                 // a copy, NaN's bits too
          *reinterpret_cast<uint4*>(static_cast<O*>(kv.out) + g * 64 + 8 * c) = u;
          continue;
        }
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) unpack2(sixteen_to_pair<T>(w[j]), v[2 * j], v[2 * j + 1]);
      } else {
        const uint8_t* const codes = kv.pages + row * (8 * BITS) + c * BITS;
        uint32_t w;
        if (BITS == 4) w = *reinterpret_cast<const uint32_t*>(codes);
        else if (BITS == 3) w = codes[0] | (static_cast<uint32_t>(codes[1]) << 8) | (static_cast<uint32_t>(codes[2]) << 16);
        else w = *reinterpret_cast<const uint16_t*>(codes);
        w = spread_codes<BITS>(w);
        const float2 st = __half22float2(kv.stats[row]);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fmaf_rn(st.y, s_cb[(w >> (4 * j)) & 15], st.x);
      }
    }
    store_eight(static_cast<O*>(kv.out) + g * 64 + 8 * c, v);
  }
}

}  // namespace arcq
