// C ABI of the key/value cache, attention over it and attention to an encoder's states: argument checks and launches.
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>
#include <stdarg.h>
#include <stdio.h>
#include <math.h>

#include "../../include/arcq_b200.h"
#include "launch.h"
#include "kv_cache.cuh"
#include "split_attention.cuh"
#include "tile_attention.cuh"

namespace {

int fail(int code, const char* fmt, ...) {
  char text[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  return arcq_host::fail(code, text);
}
bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// As a programmatic dependent of the kernel before it (see arcq_b200.cu), `cluster` blocks of the x dimension to a cluster.
template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = grid;
  lc.blockDim = dim3(threads);
  lc.dynamicSmemBytes = smem;
  lc.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (arcq_host::dependent_launches()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  lc.attrs = attr;
  lc.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&lc, kernel, static_cast<KArgs>(args)...);
  const cudaError_t left = cudaGetLastError();
  return e != cudaSuccess ? e : left;
}

int log2_of(int64_t v) {
  int s = 0;
  while ((1ll << s) < v) ++s;
  return s;
}

int check_cache(const arcq_kv_cache* c) {
  if (c == nullptr) return fail(ARCQ_E_BAD_ARG, "null pointer argument");
  if (c->bits != 2 && c->bits != 3 && c->bits != 4 && c->bits != 16) return fail(ARCQ_E_BAD_ARG, "bits must be 2, 3, 4 or 16, got %d", c->bits);
  if (c->heads <= 0 || c->heads > 65535 || c->pages < 0 || c->pages > 0x7fffffffLL) return fail(ARCQ_E_BAD_SHAPE, "bad cache: pages=%lld heads=%lld", (long long)c->pages, (long long)c->heads);
  if (c->page_size < 16 || c->page_size > (1 << 20) || (c->page_size & (c->page_size - 1)) != 0)
    return fail(ARCQ_E_UNSUPPORTED, "page size %lld: a power of two of at least 16 tokens", (long long)c->page_size);
  if (c->bits != 16 && (c->codebooks == nullptr || !aligned(c->codebooks, 4))) return fail(ARCQ_E_BAD_ARG, "packed pages need codebooks");
  if (c->pages == 0) return ARCQ_OK;
  if (c->k_pages == nullptr || c->v_pages == nullptr) return fail(ARCQ_E_BAD_ARG, "null pointer argument");
  if (!aligned(c->k_pages, 16) || !aligned(c->v_pages, 16)) return fail(ARCQ_E_ALIGN, "pages must be 16-byte aligned");
  if (c->bits == 16) {
    if (c->dtype != ARCQ_DT_F16 && c->dtype != ARCQ_DT_BF16) return fail(ARCQ_E_BAD_ARG, "pages in 16 bits are fp16 or bf16");
    return ARCQ_OK;
  }
  if (c->k_stats == nullptr || c->v_stats == nullptr) return fail(ARCQ_E_BAD_ARG, "null pointer argument");
  if (!aligned(c->k_stats, 16) || !aligned(c->v_stats, 16)) return fail(ARCQ_E_ALIGN, "statistics must be 16-byte aligned");
  return ARCQ_OK;
}

arcq::KvCacheParams cache_params(const arcq_kv_cache* c, const int64_t* slots, int64_t tokens) {
  arcq::KvCacheParams p = {};
  p.slots = reinterpret_cast<const long long*>(slots);
  p.tokens = tokens;
  p.slot_count = c->pages * c->page_size;
  p.heads = static_cast<int>(c->heads);
  p.page_shift = log2_of(c->page_size);
  const int levels = c->bits == 16 ? 0 : 1 << c->bits;
  for (int i = 0; i < 2; ++i) {
    p.kv[i].pages = static_cast<uint8_t*>(i ? c->v_pages : c->k_pages);
    p.kv[i].stats = static_cast<__half2*>(i ? c->v_stats : c->k_stats);
    p.kv[i].levels = c->codebooks + i * levels;
  }
  return p;
}

int blocks_for(long long items, int per_block, int per_sm) {
  const long long need = (items + per_block - 1) / per_block, cap = static_cast<long long>(arcq_host::sm_count()) * per_sm;
  return static_cast<int>(need < 1 ? 1 : need < cap ? need : cap);
}

// From so many groups of keys on a lane a group is the faster way; below, eight lanes a group finish sooner: 1200 groups in 4 bits 3.2 against
// 2.7 us, 3600 groups 3.3 against 3.7, 12 000 3.8 against 6.1, 196 608 24 against 61.
constexpr long long kWriteTileGroups = 2500;

template <typename T, int BITS> cudaError_t write_packed(const arcq::KvCacheParams& p, cudaStream_t st) {
  const long long groups = p.tokens * p.heads;
  if constexpr (sizeof(T) == 2) {
    if (groups >= kWriteTileGroups) {
      auto k = arcq::kv_write_tile_kernel<T, BITS>;
      static thread_local int done_dev = -1;
      int dev = 0;
      cudaGetDevice(&dev);
      if (done_dev != dev) {
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(arcq::kWriteSmem));
        if (e != cudaSuccess) return e;
        done_dev = dev;
      }
      return launch(k, dim3(blocks_for(groups, arcq::kWriteWarps * 32, 2), 2), arcq::kWriteThreads, arcq::kWriteSmem, 1, st, p);
    }
  }
  return launch(arcq::kv_write_kernel<T, BITS>, dim3(blocks_for(groups, 32, 4), 2), 256, 0, 1, st, p);
}
template <typename T> cudaError_t write_packed(const arcq::KvCacheParams& p, int bits, cudaStream_t st) {
  switch (bits) {
    case 4: return write_packed<T, 4>(p, st);
    case 3: return write_packed<T, 3>(p, st);
    default: return write_packed<T, 2>(p, st);
  }
}

constexpr int kReadBlocks = 4;                 // an SM, of keys and as many of values
template <typename O> cudaError_t read_cache(const arcq::KvCacheParams& p, int bits, int dtype, cudaStream_t st) {
  const dim3 grid(blocks_for(p.tokens * p.heads * 4, 256, kReadBlocks), 2);
  switch (bits) {
    case 16:
      if (dtype == ARCQ_DT_F16) return launch(arcq::kv_read_kernel<__half, 16, O>, grid, 256, 0, 1, st, p);
      return launch(arcq::kv_read_kernel<__nv_bfloat16, 16, O>, grid, 256, 0, 1, st, p);
    case 4: return launch(arcq::kv_read_kernel<__half, 4, O>, grid, 256, 0, 1, st, p);
    case 3: return launch(arcq::kv_read_kernel<__half, 3, O>, grid, 256, 0, 1, st, p);
    default: return launch(arcq::kv_read_kernel<__half, 2, O>, grid, 256, 0, 1, st, p);
  }
}

// ---- few rows: the steps of all units cut evenly, parts joined behind
void split_shape(arcq::AttendParams& p) {
  const long long rows = static_cast<long long>(p.max_new) * p.group;
  p.tiles = static_cast<int>((rows + arcq::kSplitRows - 1) / arcq::kSplitRows);
  p.part_rows = static_cast<int>(rows < arcq::kSplitRows ? rows : arcq::kSplitRows);
}
// rows of a key head that the split kernel may have; a workspace is asked for up to them
bool few_rows(const arcq::AttendParams& p) { return static_cast<long long>(p.max_new) * p.group <= 4 * arcq::kSplitRows; }

// Over up to so many keys units are not cut between blocks, which spares the second kernel: 12 heads, 1 token, 4 bits, 512 keys 9.4 us against 11.2,
// 1024 keys 11.5 against 13.0, 1536 keys 13.4 against 12.5; 50 sequences of up to 1024 keys 16.6 against 16.2.
constexpr int kWholeUnitKeys = 1152;

// About how long calls over up to kWholeUnitKeys keys take (us; fitted over 60 to 1500 key heads, 1 to 64 rows, 10 to 500 keys; off by a fifth).
// Split kernel, units cut between a block's warps: every warp has as much to do, and the block joins parts.  Units whole in a warp: nothing is
// joined, but a warp has whole units to do, at up to twice the pace where few warps have any.  The latter is ahead where units are many or
// short: 600 key heads, 16 rows, 16 bits, 64 keys 8.3 against 14.2, 500 keys 24.9 against 30.9; 204 key heads, 1 row, 500 keys 17.7 against 10.6.
struct SplitTimes {
  double cut, whole;
};
template <int BITS> SplitTimes split_times(const arcq::AttendParams& p) {
  const double rows = static_cast<double>(p.max_new) * p.group, warps = static_cast<double>(arcq_host::sm_count()) * arcq::kSplitWarps;
  const double units = static_cast<double>(p.batch) * p.kv_heads * ceil(rows / arcq::kSplitRows), steps = p.max_keys / arcq::SplitStep<BITS>::kKeys + 1;
  const double set_up = BITS == 16 ? 4.7 : 8.0, a_block = units / arcq_host::sm_count();
  const double join = BITS == 16 ? (rows <= 8 ? 1.2 + 0.05 * rows * a_block : 4.0 + 1.75 * a_block) : (rows <= 8 ? 2.4 : 4.0 + 0.5 * a_block);
  const double share = fmax(units * steps / warps, 0.4), busy = fmin(units / warps, 1.0);
  const double cut_step = BITS != 16 && rows > 8 ? 2.2 : 1.25, whole_step = BITS == 16 ? 0.45 * (1.0 + busy) : 1.0 + 1.3 * busy;
  return {set_up + join + share * cut_step, set_up + ceil(units / warps) * steps * whole_step};
}
// Up to 128 rows: blocks of one stream, two on an SM, where there is a second for it and the keys are few, so that one block's set-up, loads and
// join run beside the other's products; or where there is one tile of keys.  384 key heads, 40 rows: 128 keys 13.4 us against two streams'
// 21.5, 384 keys 23.8 against 29.7, 577 keys 33.7 against 37.0, 900 keys 47.1 against 47.3, 1500 keys 65.1 against 62.2; 140 key heads, 48 rows:
// 128 keys 7.0 against 7.9, 250 keys 9.0 against 9.2, 500 keys 12.9 against 11.1, 900 keys 20.8 against 15.7.
bool one_stream_is_ahead(const arcq::AttendParams& p) {
  const int key_tiles = (p.max_keys + arcq::kTileKeys - 1) / arcq::kTileKeys;
  return key_tiles <= 1 || (key_tiles <= 6 && static_cast<long long>(p.batch) * p.kv_heads > arcq_host::sm_count());
}

// The tile kernel likewise, for up to 128 rows
template <int BITS> double tile_time(const arcq::AttendParams& p) {
  const double units = static_cast<double>(p.batch) * p.kv_heads, sms = arcq_host::sm_count(), tiles = fmax(ceil(p.max_keys / static_cast<double>(arcq::kTileKeys)), 1.0);
  const double splits = fmax(fmin(fmin(floor(sms / units), 8.0), tiles), 1.0);    // blocks of a cluster
  const double one = 5.8 + 2.2 * (tiles - 1.0), two = 7.4 + 0.85 * (ceil(tiles / splits) - 1.0) + (splits > 1.0 ? 1.0 : 0.0);
  return 0.5 + (BITS == 16 && one_stream_is_ahead(p) ? ceil(units / (2.0 * sms)) * one : ceil(units / sms) * two);
}
// Up to 8 rows a key head the split kernel is always ahead (12 heads, 8 rows, 4 bits: over 300 tokens 8.3 us against the tile kernel's 9.3, over 16 000
// 20.6 against 33.7); above, over short contexts, by the times (1500 key heads, 16 rows, 30 keys: 16 bits 7.4
// against 35.5, 4 bits 9.0 against 79; 204 key heads, 250 keys: 16 bits 13.1 against 9.9).  Over long ones, 9 to 32 rows, it is where keys times key heads
// are many.  In 4 bits, 16 rows: 192 000 of them 28.8 against 33.9; below, 48 000 21.2 against 18.0; 32 rows: 384 000 32.7 against 33.0, 768 000
// 55 against 64.  In 16 bits, where the tile kernel has no codes to look up: 192 000 34.0 against 30.1, 360 000 41.1 against 44.8.
template <int BITS> bool split_is_ahead(const arcq::AttendParams& p) {
  constexpr long long kMany = BITS == 16 ? 5 << 16 : 2 << 16;
  const long long rows = static_cast<long long>(p.max_new) * p.group;
  if (rows <= 8 || !few_rows(p)) return few_rows(p);
  if (p.max_keys <= kWholeUnitKeys) {
    const SplitTimes t = split_times<BITS>(p);
    return fmin(t.cut, t.whole) < tile_time<BITS>(p);
  }
  return rows <= 2 * arcq::kSplitRows && static_cast<long long>(p.batch) * p.kv_heads * p.max_keys > kMany;
}

template <int BITS, typename E> int launch_split(arcq::AttendParams& p, int64_t workspace_bytes, cudaStream_t st) {
  auto k = arcq::split_attention_kernel<BITS, E>;
  constexpr size_t smem = arcq::split_parts<BITS>() + arcq::kSplitSharedParts + 128;
  static_assert(smem + arcq::kSplitBase <= 227 * 1024, "");
  static thread_local int done_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (done_dev != dev) {
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    cudaFuncAttributes a = {};
    int reserved = 0;
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, k);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&reserved, cudaDevAttrReservedSharedMemoryPerBlock, dev);
    if (e != cudaSuccess) return arcq_host::cuda_fail(e, "attention set-up");
    if (BITS != 16 && a.sharedSizeBytes + reserved + 128 > arcq::kSplitBase)       // the rings are laid out around the table
      return fail(ARCQ_E_CUDA, "attention: %lld bytes of shared memory before the rings, %lld are provided for", (long long)(a.sharedSizeBytes + reserved), (long long)arcq::kSplitBase);
    done_dev = dev;
  }
  split_shape(p);
  const int sms = arcq_host::sm_count();
  if (p.workspace == nullptr || workspace_bytes < arcq::split_workspace(p, sms))
    return fail(ARCQ_E_BAD_ARG, "workspace of %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)arcq::split_workspace(p, sms));
  const long long units = arcq::split_units(p), unit_steps = p.max_keys / arcq::SplitStep<BITS>::kKeys + 1, steps = units * unit_steps;
  if (static_cast<double>(units) * unit_steps > 1073741823.0) return fail(ARCQ_E_TOO_LARGE, "too many queries and keys for one call");
  const SplitTimes times = split_times<BITS>(p);
  p.whole_units = p.max_keys > kWholeUnitKeys ? 0 : times.whole < times.cut ? 2 : 1;
  cudaError_t e = launch(k, dim3(static_cast<unsigned>(steps < sms ? steps : sms)), arcq::kSplitThreads, smem, 1, st, p);
  if (e == cudaSuccess && !p.whole_units) e = launch(arcq::join_attention_kernel, dim3(static_cast<unsigned>(units)), arcq::kJoinThreads, 0, 1, st, p);
  return e == cudaSuccess ? ARCQ_OK : arcq_host::cuda_fail(e, "attention launch");
}

// How many clusters of a size run at a time; 0: none, or it cannot be said
template <typename Kernel> int clusters_at_a_time(Kernel k, int size, int threads, size_t smem) {
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = size;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  lc.gridDim = dim3(size * arcq_host::sm_count() * 2);
  lc.blockDim = dim3(threads);
  lc.dynamicSmemBytes = smem;
  lc.attrs = &attr;
  lc.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, k, &lc) == cudaSuccess) return n;
  cudaGetLastError();
  return 0;
}
// What a round of blocks counts besides its tiles of keys, in tiles (1.7 us for both streams): more than a block's set-up, which is some 4 by tile_time,
// since blocks of a further round start unevenly.  Over 27 calls of 1 to 24 sequences and 64 to 2048 queries it hardly matters (2, 4, 7 and 10 within
// 0.1 % of one another in all); 13 sequences of 256 over 2000, 12 heads, 4 bits: 75.4 us with 2 and 4, 73.7 with 7 and 10; 13 x 256 over 2309 in 16 bits
// 75.6 and 76.7.
constexpr double kTileSetUp = 7.0;

// Blocks of a row tile, 1 to 8: the cluster size for which the rounds of blocks over the SMs take the fewest tiles of keys, a block's set-up and
// the joining of results counted as tiles.
template <int BITS, typename E, int STREAMS> int launch_tile(arcq::AttendParams& p, cudaStream_t st) {
  auto k = arcq::tile_attention_kernel<BITS, E, STREAMS, false>, ranked = arcq::tile_attention_kernel<BITS, E, STREAMS, true>;
  constexpr size_t smem = arcq::tile_smem_layout(BITS != 16, STREAMS).total;
  constexpr int threads = arcq::tile_threads(STREAMS), block_rows = STREAMS * arcq::kTileRows;
  static thread_local int done_dev = -1, room[9];                               // clusters of a size that run at a time
  int dev = 0;
  cudaGetDevice(&dev);
  if (done_dev != dev) {
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(ranked, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    cudaFuncAttributes a = {}, b = {};
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, k);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&b, ranked);
    if (e != cudaSuccess) return arcq_host::cuda_fail(e, "attention set-up");
    const int got = arcq_host::launch_regs() > 0 ? arcq_host::launch_regs() : a.numRegs < b.numRegs ? a.numRegs : b.numRegs;
    if (STREAMS > 1 && got < arcq::kTileLaunchRegs)             // the warp groups' hand-over would wait for good
      return fail(ARCQ_E_CUDA, "attention: compiled for %d registers a thread, its warp groups share out %d", got, arcq::kTileLaunchRegs);
    room[1] = arcq_host::sm_count() * (3 - STREAMS);
    for (int s = 2; s <= 8; ++s) room[s] = clusters_at_a_time(k, s, threads, smem);
    done_dev = dev;
  }
  const long long all_rows = static_cast<long long>(p.max_new) * p.group;
  const long long tiles = (all_rows + block_rows - 1) / block_rows;
  if (static_cast<double>(p.batch) * p.kv_heads * tiles > 2147483647.0) return fail(ARCQ_E_TOO_LARGE, "too many queries for one call");
  p.tiles = static_cast<int>(tiles);
  const long long units = static_cast<long long>(p.batch) * p.kv_heads * p.tiles;
  const double key_tiles = (p.max_keys + arcq::kTileKeys - 1) / arcq::kTileKeys, each = STREAMS == 1 || all_rows > arcq::kTileRows ? 1.0 : 0.5;
  int splits = 1;
  double best = 1e30;
  for (int s = 1; s <= 8 && (s == 1 || s <= key_tiles); ++s) {
    if (room[s] <= 0) continue;
    const double cost = ceil(static_cast<double>(units) / room[s]) * (ceil(key_tiles / s) * each + kTileSetUp + (s > 1 ? 1.0 : 0.0));
    if (cost < best) {
      best = cost;
      splits = s;
    }
  }
  p.splits = splits;
  // Sequences in the order of their work where there are a few rounds of blocks; more rounds even out by themselves, and each block pays some 0.3 us.
  // 24 sequences, 1 to 197 tokens over 625 to 2500, 2 rounds: 51.2 us against 64.7; 64 sequences, 3.5 rounds: 76 against 84; 96 over 300 states, 3.9
  // rounds: 50.4 against 47.6; 16 over up to 2309 states, 5.2 rounds: 161 against 159.5.
  const bool in_order = p.batch > 1 && p.batch <= arcq::kTileRanked && (p.lengths != nullptr || p.starts != nullptr) && units > room[splits] && units <= 4ll * room[splits];
  p.poll_limit = arcq_host::poll_limit();
  p.status = arcq_host::status_ptr();
  if (units * splits > 0x7fffffffLL) return fail(ARCQ_E_TOO_LARGE, "too many queries for one call");
  const cudaError_t e = launch(in_order ? ranked : k, dim3(static_cast<unsigned>(units * splits)), threads, smem, splits, st, p);
  return e == cudaSuccess ? ARCQ_OK : arcq_host::cuda_fail(e, "attention launch");
}

template <int BITS, typename E> int launch_attention(arcq::AttendParams& p, int64_t workspace_bytes, cudaStream_t st) {
  if (split_is_ahead<BITS>(p)) return launch_split<BITS, E>(p, workspace_bytes, st);
  // no blocks for rows that q has not got (the split kernel's grid goes by the steps, its workspace by what the caller said)
  if (p.starts != nullptr && p.max_new > p.q_rows) p.max_new = static_cast<int>(p.q_rows);
  if constexpr (BITS == 16)
    if (static_cast<long long>(p.max_new) * p.group <= arcq::kTileRows && one_stream_is_ahead(p)) return launch_tile<BITS, E, 1>(p, st);
  return launch_tile<BITS, E, 2>(p, st);
}

int run_attention(arcq::AttendParams& p, int bits, int dtype, void* workspace, int64_t workspace_bytes, cudaStream_t st) {
  p.workspace = workspace;
  if (!aligned(workspace, 16)) return fail(ARCQ_E_ALIGN, "the workspace must be 16-byte aligned");
  switch (bits) {
    case 4: return launch_attention<4, __half>(p, workspace_bytes, st);
    case 3: return launch_attention<3, __half>(p, workspace_bytes, st);
    case 2: return launch_attention<2, __half>(p, workspace_bytes, st);
    default: return dtype == ARCQ_DT_BF16 ? launch_attention<16, __nv_bfloat16>(p, workspace_bytes, st) : launch_attention<16, __half>(p, workspace_bytes, st);
  }
}

int check_query(const void* q, int dtype, const void* out, int64_t heads, int64_t kv_heads, float scale) {
  if (q == nullptr || out == nullptr) return fail(ARCQ_E_BAD_ARG, "null pointer argument");
  if (dtype != ARCQ_DT_F16 && dtype != ARCQ_DT_BF16) return fail(ARCQ_E_BAD_ARG, "queries are fp16 or bf16");
  if (heads <= 0 || kv_heads <= 0 || heads > 65535 || heads % kv_heads != 0)
    return fail(ARCQ_E_BAD_SHAPE, "%lld heads over %lld key heads", (long long)heads, (long long)kv_heads);
  if (!(scale > 0.0f) || !isfinite(scale * 1.44269504088896340736f)) return fail(ARCQ_E_BAD_ARG, "scale must be positive and finite");
  if (!aligned(q, 16) || !aligned(out, 16)) return fail(ARCQ_E_ALIGN, "queries and out must be 16-byte aligned");
  return ARCQ_OK;
}
// Keys are counted in 32 bits, rounded up to whole tiles.
constexpr long long kMostKeys = 0x7fffffffLL - (arcq::kTileKeys - 1);
// Rows of a key head, and those of its last block, are counted in 32 bits.
bool too_many_rows(int64_t max_new, int64_t group) { return max_new * group > 0x7fffffffLL - 256; }
bool strides_ok(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] % 8 != 0) return false;
  return true;
}

// Whether `out`, `bytes` long, lies over any of a tensor of 64 values a head with these sizes and strides (in values).
bool overlaps(const void* out, int64_t bytes, const void* t, int n, const int64_t* sizes, const int64_t* strides) {
  int64_t lo = 0, hi = 63;
  for (int i = 0; i < n; ++i) {
    if (sizes[i] == 0) return false;
    (strides[i] < 0 ? lo : hi) += (sizes[i] - 1) * strides[i];
  }
  const char *const a = static_cast<const char*>(out), *const b = static_cast<const char*>(t);
  return a < b + 2 * (hi + 1) && b + 2 * lo < a + bytes;
}

// Whether `out`, `bytes` long, lies over any of the `size` bytes at t.
bool lies_over(const void* out, int64_t bytes, const void* t, __int128 size) {
  const __int128 a = reinterpret_cast<uintptr_t>(out), b = reinterpret_cast<uintptr_t>(t);
  return t != nullptr && a < b + size && b < a + bytes;
}
bool over_cache(const void* out, int64_t bytes, const arcq_kv_cache* c) {
  const __int128 rows = static_cast<__int128>(c->pages) * c->heads * c->page_size, row = c->bits == 16 ? 128 : 8 * c->bits;
  if (lies_over(out, bytes, c->k_pages, rows * row) || lies_over(out, bytes, c->v_pages, rows * row)) return true;
  return c->bits != 16 && (lies_over(out, bytes, c->k_stats, rows * 4) || lies_over(out, bytes, c->v_stats, rows * 4) ||
                           lies_over(out, bytes, c->codebooks, 8ll << c->bits));
}

}  // namespace

extern "C" {

int arcq_kv_cache_write(const arcq_kv_cache* cache, const float* thresholds, const void* k, const void* v, int x_dtype, int64_t tokens,
                        const int64_t* k_strides, const int64_t* v_strides, const int64_t* slots, void* stream) {
  if (const int rc = check_cache(cache)) return rc;
  if (tokens < 0 || tokens > 0x7fffffffLL || tokens * cache->heads > 0x7fffffffLL) return fail(ARCQ_E_BAD_SHAPE, "bad number of tokens %lld", (long long)tokens);
  if (tokens == 0 || cache->pages == 0) return ARCQ_OK;
  if (k == nullptr || v == nullptr || slots == nullptr || k_strides == nullptr || v_strides == nullptr || (cache->bits != 16 && thresholds == nullptr))
    return fail(ARCQ_E_BAD_ARG, "null pointer argument");
  if (x_dtype != ARCQ_DT_F32 && x_dtype != ARCQ_DT_F16 && x_dtype != ARCQ_DT_BF16) return fail(ARCQ_E_BAD_ARG, "bad element type %d", x_dtype);
  if (cache->bits == 16 && x_dtype != cache->dtype) return fail(ARCQ_E_BAD_ARG, "keys and values must have the type of the pages");
  if (!aligned(k, 16) || !aligned(v, 16) || !strides_ok(k_strides, 2) || !strides_ok(v_strides, 2))
    return fail(ARCQ_E_ALIGN, "keys and values must be 16-byte aligned, their strides multiples of 8 values");
  arcq::KvCacheParams p = cache_params(cache, slots, tokens);
  const int levels = cache->bits == 16 ? 0 : (1 << cache->bits) - 1;
  for (int i = 0; i < 2; ++i) {
    p.kv[i].x = i ? v : k;
    p.kv[i].token_stride = (i ? v_strides : k_strides)[0];
    p.kv[i].head_stride = (i ? v_strides : k_strides)[1];
    p.kv[i].thresholds = thresholds != nullptr ? thresholds + i * levels : nullptr;
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (cache->bits == 16) e = launch(arcq::kv_write_copy_kernel, dim3(blocks_for(tokens * cache->heads * 8, 256, 4), 2), 256, 0, 1, st, p);
  else if (x_dtype == ARCQ_DT_F32) e = write_packed<float>(p, cache->bits, st);
  else if (x_dtype == ARCQ_DT_F16) e = write_packed<__half>(p, cache->bits, st);
  else e = write_packed<__nv_bfloat16>(p, cache->bits, st);
  return e == cudaSuccess ? ARCQ_OK : arcq_host::cuda_fail(e, "cache write launch");
}

int arcq_kv_cache_read(const arcq_kv_cache* cache, const int64_t* slots, int64_t tokens, void* k_out, void* v_out, int out_dtype, void* stream) {
  if (const int rc = check_cache(cache)) return rc;
  if (tokens < 0 || tokens > 0x7fffffffLL || tokens * cache->heads > 0x7fffffffLL) return fail(ARCQ_E_BAD_SHAPE, "bad number of tokens %lld", (long long)tokens);
  if (tokens == 0) return ARCQ_OK;
  if (k_out == nullptr || v_out == nullptr || slots == nullptr) return fail(ARCQ_E_BAD_ARG, "null pointer argument");
  if (!aligned(k_out, 32) || !aligned(v_out, 32)) return fail(ARCQ_E_ALIGN, "outputs must be 32-byte aligned");
  arcq::KvCacheParams p = cache_params(cache, slots, tokens);
  p.kv[0].out = k_out;
  p.kv[1].out = v_out;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (out_dtype == ARCQ_DT_F32) e = read_cache<float>(p, cache->bits, cache->dtype, st);
  else if (out_dtype == ARCQ_DT_F16) e = read_cache<__half>(p, cache->bits, cache->dtype, st);
  else if (out_dtype == ARCQ_DT_BF16) e = read_cache<__nv_bfloat16>(p, cache->bits, cache->dtype, st);
  else return fail(ARCQ_E_BAD_ARG, "bad element type %d", out_dtype);
  return e == cudaSuccess ? ARCQ_OK : arcq_host::cuda_fail(e, "cache read launch");
}

int64_t arcq_attention_workspace(int64_t batch, int64_t max_new, int64_t heads, int64_t kv_heads) {
  if (batch <= 0 || max_new <= 0 || heads <= 0 || kv_heads <= 0 || batch > 0x7fffffffLL || max_new > 0x7fffffffLL || heads > 65535 || heads % kv_heads != 0) return 0;
  arcq::AttendParams p = {};
  p.batch = static_cast<int>(batch);
  p.max_new = static_cast<int>(max_new);
  p.kv_heads = static_cast<int>(kv_heads);
  p.group = static_cast<int>(heads / kv_heads);
  if (!few_rows(p)) return 0;
  split_shape(p);
  return arcq::split_workspace(p, arcq_host::sm_count());
}

int arcq_paged_attention(const arcq_kv_cache* cache, const void* q, int q_dtype, int64_t q_rows, const int64_t* q_strides, int64_t heads,
                         int64_t batch, const int32_t* page_table, int64_t table_width, const int32_t* lengths, const int32_t* starts,
                         int64_t max_new, int causal, float scale, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = check_cache(cache)) return rc;
  if (batch < 0 || table_width < 0 || max_new < 0 || q_rows < 0 || q_rows > 0x7fffffffLL || batch > 0x7fffffffLL || max_new > 0x7fffffffLL)
    return fail(ARCQ_E_BAD_SHAPE, "bad shape: batch=%lld table=%lld new=%lld rows=%lld", (long long)batch, (long long)table_width, (long long)max_new, (long long)q_rows);
  if (starts == nullptr && batch * max_new != q_rows) return fail(ARCQ_E_BAD_SHAPE, "%lld queries for %lld sequences of %lld", (long long)q_rows, (long long)batch, (long long)max_new);
  if (table_width > 0x7fffffffLL || table_width * cache->page_size > kMostKeys) return fail(ARCQ_E_TOO_LARGE, "contexts of more than 2^31 tokens");
  if (batch == 0 || q_rows == 0 || max_new == 0) return ARCQ_OK;
  if (lengths == nullptr || (page_table == nullptr && table_width > 0) || q_strides == nullptr) return fail(ARCQ_E_BAD_ARG, "null pointer argument");
  if (const int rc = check_query(q, q_dtype, out, heads, cache->heads, scale)) return rc;
  if (too_many_rows(max_new, heads / cache->heads)) return fail(ARCQ_E_TOO_LARGE, "%lld new tokens a sequence are too many", (long long)max_new);
  const int64_t q_sizes[] = {q_rows, heads};
  if (overlaps(out, q_rows * heads * 128, q, 2, q_sizes, q_strides)) return fail(ARCQ_E_BAD_ARG, "out lies over the queries");
  if (over_cache(out, q_rows * heads * 128, cache)) return fail(ARCQ_E_BAD_ARG, "out lies over the cache");
  if (lies_over(out, q_rows * heads * 128, page_table, 4 * batch * table_width) || lies_over(out, q_rows * heads * 128, lengths, 4 * batch) ||
      lies_over(out, q_rows * heads * 128, starts, 4 * (batch + 1)))
    return fail(ARCQ_E_BAD_ARG, "out lies over the page table, the lengths or the starts");
  if (cache->bits == 16 && q_dtype != cache->dtype) return fail(ARCQ_E_BAD_ARG, "queries must have the type of the pages");
  if (!strides_ok(q_strides, 2)) return fail(ARCQ_E_ALIGN, "strides of the queries must be multiples of 8 values");
  arcq::AttendParams p = {};
  const int row = cache->bits == 16 ? 128 : 8 * cache->bits;
  for (int i = 0; i < 2; ++i) {
    arcq::AttendView& a = i ? p.v : p.k;
    a.rows = static_cast<const uint8_t*>(i ? cache->v_pages : cache->k_pages);
    a.stats = static_cast<const __half2*>(i ? cache->v_stats : cache->k_stats);
    a.token_stride = row;
    a.head_stride = cache->page_size * row;
    a.block_stride = cache->heads * a.head_stride;
  }
  p.codebooks = cache->codebooks;
  p.table = page_table;
  p.table_width = static_cast<int>(table_width);
  p.page_shift = log2_of(cache->page_size);
  p.pages = static_cast<int>(cache->pages);
  p.lengths = lengths;
  p.max_keys = static_cast<int>(table_width * cache->page_size);
  p.q = q;
  p.q_token = q_strides[0];
  p.q_head = q_strides[1];
  p.q_batch = max_new * q_strides[0];
  p.q_rows = q_rows;
  p.starts = starts;
  p.max_new = static_cast<int>(max_new);
  p.causal = causal != 0;
  p.q_bf16 = q_dtype == ARCQ_DT_BF16;
  p.scale_log2 = scale * 1.44269504088896340736f;
  p.out = out;
  p.heads = static_cast<int>(heads);
  p.kv_heads = static_cast<int>(cache->heads);
  p.group = p.heads / p.kv_heads;
  p.batch = static_cast<int>(batch);
  return run_attention(p, cache->bits, cache->dtype, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int arcq_cross_attention(const void* q, const void* k, const void* v, int dtype, int64_t batch, int64_t queries, int64_t states, int64_t heads,
                         int64_t kv_heads, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, const int32_t* lengths,
                         const uint8_t* mask, int64_t mask_stride, float scale, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (batch < 0 || queries < 0 || states < 0 || batch > 0x7fffffffLL || queries > 0x7fffffffLL || batch * queries > 0x7fffffffLL || states > kMostKeys)
    return fail(ARCQ_E_BAD_SHAPE, "bad shape: batch=%lld queries=%lld states=%lld", (long long)batch, (long long)queries, (long long)states);
  if (batch == 0 || queries == 0) return ARCQ_OK;
  if (q_strides == nullptr || k_strides == nullptr || v_strides == nullptr || (states > 0 && (k == nullptr || v == nullptr)))
    return fail(ARCQ_E_BAD_ARG, "null pointer argument");
  if (const int rc = check_query(q, dtype, out, heads, kv_heads, scale)) return rc;
  if (too_many_rows(queries, heads / kv_heads)) return fail(ARCQ_E_TOO_LARGE, "%lld queries a sequence are too many", (long long)queries);
  const int64_t q_sizes[] = {batch, queries, heads}, kv_sizes[] = {batch, states, kv_heads}, bytes = batch * queries * heads * 128;
  if (overlaps(out, bytes, q, 3, q_sizes, q_strides) || overlaps(out, bytes, k, 3, kv_sizes, k_strides) || overlaps(out, bytes, v, 3, kv_sizes, v_strides))
    return fail(ARCQ_E_BAD_ARG, "out lies over the queries, keys or values");
  if (lies_over(out, bytes, lengths, 4 * batch) || (mask_stride >= 0 && lies_over(out, bytes, mask, static_cast<__int128>(batch - 1) * mask_stride + states)))
    return fail(ARCQ_E_BAD_ARG, "out lies over the lengths or the mask");
  if (lengths != nullptr && mask != nullptr) return fail(ARCQ_E_BAD_ARG, "lengths or a mask, not both");
  if (!aligned(k, 16) || !aligned(v, 16)) return fail(ARCQ_E_ALIGN, "keys and values must be 16-byte aligned");
  if (!strides_ok(q_strides, 3) || !strides_ok(k_strides, 3) || !strides_ok(v_strides, 3)) return fail(ARCQ_E_ALIGN, "strides must be multiples of 8 values");
  arcq::AttendParams p = {};
  for (int i = 0; i < 2; ++i) {
    arcq::AttendView& a = i ? p.v : p.k;
    const int64_t* const s = i ? v_strides : k_strides;
    a.rows = static_cast<const uint8_t*>(i ? v : k);
    a.block_stride = 2 * s[0];
    a.token_stride = 2 * s[1];
    a.head_stride = 2 * s[2];
  }
  p.lengths = lengths;
  p.mask = mask;
  p.mask_stride = mask_stride;
  p.max_keys = static_cast<int>(states);
  p.q = q;
  p.q_batch = q_strides[0];
  p.q_token = q_strides[1];
  p.q_head = q_strides[2];
  p.q_rows = batch * queries;
  p.max_new = static_cast<int>(queries);
  p.q_bf16 = dtype == ARCQ_DT_BF16;
  p.scale_log2 = scale * 1.44269504088896340736f;
  p.out = out;
  p.heads = static_cast<int>(heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.group = p.heads / p.kv_heads;
  p.batch = static_cast<int>(batch);
  return run_attention(p, 16, dtype, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
