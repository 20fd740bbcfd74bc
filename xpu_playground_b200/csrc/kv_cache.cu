// Page operators of the serving cache (xpu_kv_* in include/xpu_cuda.h).
//
// Each call is a planning kernel of one CTA, which checks the whole request,
// takes pages and rewrites lens (or refuses and changes nothing), and where
// rows or pages move a second kernel over the whole GPU that copies what the
// plan lists. Between them the workspace holds
//   [0] 1 if the plan was accepted, [1] entries, [2] first page id that
//   compaction renames, [4 ..] per entry {source page, new page, rows}, and
//   behind those compaction's new id of every page.
// All page choices are by ascending id, so the result does not depend on
// the order in which threads run.
#include <algorithm>

#include "common.cuh"
#include "xpu_internal.h"

namespace xpu {
namespace {

constexpr uint32_t kPlanThreads = 1024;
constexpr uint32_t kHeader = 4, kEntry = 3;

__device__ __forceinline__ uint32_t pages_of(uint32_t positions, uint32_t size) { return (positions + size - 1) / size; }

// Exclusive prefix sum over the CTA in thread order; *total gets the sum.
__device__ uint32_t block_scan(uint32_t v, uint32_t *total) {
  __shared__ uint32_t warp_sums[32];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t inc = v;
#pragma unroll
  for (uint32_t o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(kFullMask, inc, o);
    if (lane >= o) inc += up;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  const uint32_t mine = warp_sums[lane];
  uint32_t sums = mine;
#pragma unroll
  for (uint32_t o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(kFullMask, sums, o);
    if (lane >= o) sums += up;
  }
  *total = __shfl_sync(kFullMask, sums, 31);
  return __shfl_sync(kFullMask, sums - mine, warp) + inc - v;
}

// The `want` lowest free pages in ascending order into list; false if there
// are fewer.
__device__ bool lowest_free(const xpu_kv_cache_t &c, uint32_t want, uint32_t *list) {
  uint32_t found = 0;
  for (uint32_t base = 0; base < c.pages && found < want; base += kPlanThreads) {
    const uint32_t p = base + threadIdx.x;
    const bool is_free = p < c.pages && c.refs[p] == 0;
    uint32_t total;
    const uint32_t rank = found + block_scan(is_free, &total);
    if (is_free && rank < want) list[rank] = p;
    found += total;
  }
  return found >= want;
}

// Marks this thread's sequence id (valid threads only) in a bitmap; true if
// every valid id of the CTA is in range and named once.
__device__ bool named_once(const xpu_kv_cache_t &c, bool valid, int32_t s, uint32_t *bitmap) {
  for (uint32_t i = threadIdx.x; i < XPU_KV_MAX_SEQUENCES / 32; i += kPlanThreads) bitmap[i] = 0;
  __syncthreads();
  bool ok = true;
  if (valid) {
    ok = s >= 0 && static_cast<uint32_t>(s) < c.sequences;
    if (ok) ok = !(atomicOr(&bitmap[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u);
  }
  return __syncthreads_and(ok);
}

__device__ __forceinline__ uint32_t len_of(const xpu_kv_cache_t &c, int32_t s) {
  const int32_t n = c.lens[s];
  return static_cast<uint32_t>(min(max(n, 0), static_cast<int32_t>(c.table_width * c.page_size)));
}

__device__ __forceinline__ bool page_ok(const xpu_kv_cache_t &c, int32_t p) {
  return p >= 0 && static_cast<uint32_t>(p) < c.pages;
}

__device__ __forceinline__ void refuse(const xpu_kv_cache_t &c, uint32_t bit) {
  if (threadIdx.x == 0) {
    atomicOr(c.status, bit);
    c.workspace[0] = 0;
    c.workspace[1] = 0;
  }
}

__global__ void __launch_bounds__(kPlanThreads) k_kv_extend(const __grid_constant__ xpu_kv_cache_t c,
                                                            const int32_t *sequences, const int32_t *starts,
                                                            uint32_t count) {
  __shared__ uint32_t bitmap[XPU_KV_MAX_SEQUENCES / 32];
  const uint32_t i = threadIdx.x;
  const bool mine = i < count;
  const int32_t s = mine ? sequences[i] : -1, more = mine ? starts[i + 1] - starts[i] : 0;
  if (!named_once(c, mine, s, bitmap) || __syncthreads_or(more < 0)) return refuse(c, XPU_KV_BAD_SEQUENCE);
  const uint32_t old = mine ? len_of(c, s) : 0;
  const uint32_t first = pages_of(old, c.page_size);
  const uint64_t after = static_cast<uint64_t>(old) + more;
  if (__syncthreads_or(after > static_cast<uint64_t>(c.table_width) * c.page_size)) return refuse(c, XPU_KV_EXHAUSTED);
  const uint32_t need = pages_of(static_cast<uint32_t>(after), c.page_size) - first;
  uint32_t total;
  const uint32_t rank = block_scan(need, &total);
  uint32_t *list = reinterpret_cast<uint32_t *>(c.workspace) + kHeader;
  if (total > c.pages || !lowest_free(c, total, list)) return refuse(c, XPU_KV_EXHAUSTED);
  __syncthreads();
  for (uint32_t j = 0; j < need; ++j) {
    const uint32_t p = list[rank + j];
    c.tables[static_cast<size_t>(s) * c.table_width + first + j] = static_cast<int32_t>(p);
    c.refs[p] = 1;
  }
  if (mine) c.lens[s] = static_cast<int32_t>(after);
  if (i == 0) c.workspace[0] = 1;
}

// One warp per (token, K or V, layer): the token's row of every head.
__global__ void __launch_bounds__(256) k_kv_write(const __grid_constant__ xpu_kv_cache_t c, const int32_t *sequences,
                                                  const int32_t *starts, uint32_t count, uint32_t tokens,
                                                  const int32_t *rows, const uint16_t *k, const uint16_t *v,
                                                  uint32_t held, uint64_t layer_stride, uint64_t row_stride,
                                                  uint32_t layer, uint32_t layers) {
  if (c.workspace[0] == 0) return;
  const uint32_t lane = threadIdx.x & 31, per_head = c.head_dim / 8, chunks = c.kv_heads * per_head;
  const uint64_t warps = static_cast<uint64_t>(gridDim.x) * (blockDim.x / 32);
  const uint32_t listed = static_cast<uint32_t>(max(starts[count], 0));
  if (listed > tokens && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(c.status, XPU_KV_BAD_INDEX);
  tokens = min(tokens, listed);
  const uint64_t work = static_cast<uint64_t>(tokens) * layers * 2;
  for (uint64_t w = static_cast<uint64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32; w < work; w += warps) {
    const uint32_t t = static_cast<uint32_t>(w % tokens), which = static_cast<uint32_t>(w / tokens);
    uint32_t lo = 0, hi = count;  // the last i with starts[i] <= t
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (starts[mid] <= static_cast<int32_t>(t)) lo = mid;
      else hi = mid;
    }
    const int32_t s = sequences[lo], row = rows ? rows[t] : static_cast<int32_t>(t);
    bool ok = s >= 0 && static_cast<uint32_t>(s) < c.sequences && row >= 0 && static_cast<uint32_t>(row) < held &&
              static_cast<int32_t>(t) >= starts[lo] && static_cast<int32_t>(t) < starts[lo + 1];
    int64_t position = 0;
    int32_t page = -1;
    if (ok) {
      position = static_cast<int64_t>(c.lens[s]) - (starts[lo + 1] - static_cast<int32_t>(t));
      ok = position >= 0 && position < static_cast<int64_t>(c.table_width) * c.page_size;
    }
    if (ok) page = c.tables[static_cast<size_t>(s) * c.table_width + position / c.page_size];
    if (!ok || !page_ok(c, page)) {
      if (lane == 0) atomicOr(c.status, XPU_KV_BAD_INDEX);
      continue;
    }
    const uint32_t l = which >> 1, slot = static_cast<uint32_t>(position) % c.page_size;
    const uint4 *src = reinterpret_cast<const uint4 *>((which & 1 ? v : k) + l * layer_stride + row * row_stride);
    uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(which & 1 ? c.v : c.k)) +
                 (static_cast<size_t>(layer + l) * c.pages + page) * chunks * c.page_size;
    for (uint32_t e = lane; e < chunks; e += 32)
      dst[(static_cast<size_t>(e / per_head) * c.page_size + slot) * per_head + e % per_head] = src[e];
  }
}

__global__ void __launch_bounds__(kPlanThreads) k_kv_trim(const __grid_constant__ xpu_kv_cache_t c,
                                                          const int32_t *sequences, const int32_t *new_lens,
                                                          uint32_t count) {
  __shared__ uint32_t bitmap[XPU_KV_MAX_SEQUENCES / 32];
  const uint32_t i = threadIdx.x;
  const bool mine = i < count;
  const int32_t s = mine ? sequences[i] : -1, want = mine ? new_lens[i] : 0;
  if (!named_once(c, mine, s, bitmap) || __syncthreads_or(want < 0)) return refuse(c, XPU_KV_BAD_SEQUENCE);
  const uint32_t old = mine ? len_of(c, s) : 0, len = min(old, static_cast<uint32_t>(want));
  int32_t *table = c.tables + static_cast<size_t>(mine ? s : 0) * c.table_width;
  bool cut = false;
  if (len < old && len % c.page_size) {
    const int32_t p = table[len / c.page_size];
    cut = page_ok(c, p) && c.refs[p] > 1;
  }
  if (__syncthreads_or(cut)) return refuse(c, XPU_KV_SHARED_CUT);
  for (uint32_t j = pages_of(len, c.page_size); j < pages_of(old, c.page_size); ++j) {
    const int32_t p = table[j];
    if (page_ok(c, p)) atomicSub(&c.refs[p], 1);
    table[j] = -1;
  }
  if (mine) c.lens[s] = static_cast<int32_t>(len);
}

__global__ void __launch_bounds__(kPlanThreads) k_kv_fork(const __grid_constant__ xpu_kv_cache_t c,
                                                          const int32_t *parents, const int32_t *children,
                                                          uint32_t count) {
  __shared__ uint32_t bitmap[XPU_KV_MAX_SEQUENCES / 32];
  const uint32_t i = threadIdx.x;
  const bool mine = i < count;
  const int32_t from = mine ? parents[i] : -1, to = mine ? children[i] : -1;
  bool bad = mine && (from < 0 || static_cast<uint32_t>(from) >= c.sequences);
  bad = !named_once(c, mine, to, bitmap) || __syncthreads_or(bad);
  if (!bad) bad = mine && (len_of(c, to) != 0 || (bitmap[from >> 5] >> (from & 31) & 1u));
  if (__syncthreads_or(bad)) return refuse(c, XPU_KV_BAD_SEQUENCE);
  const uint32_t len = mine ? len_of(c, from) : 0, part = len % c.page_size;
  const int32_t *table = c.tables + static_cast<size_t>(mine ? from : 0) * c.table_width;
  const int32_t last = part ? table[len / c.page_size] : -1;
  uint32_t total;
  const uint32_t rank = block_scan(part != 0, &total);
  // the list of free pages lies behind the entries that will name them
  uint32_t *list = reinterpret_cast<uint32_t *>(c.workspace) + kHeader + kEntry * XPU_KV_MAX_REQUESTS;
  if (total > c.pages || !lowest_free(c, total, list)) return refuse(c, XPU_KV_EXHAUSTED);
  __syncthreads();
  if (part) {
    const int32_t p = static_cast<int32_t>(list[rank]);
    int32_t *entry = c.workspace + kHeader + kEntry * rank;
    entry[0] = last;
    entry[1] = p;
    entry[2] = static_cast<int32_t>(part);
    c.refs[p] = 1;
    c.tables[static_cast<size_t>(to) * c.table_width + len / c.page_size] = p;
  }
  if (mine) c.lens[to] = static_cast<int32_t>(len);
  if (i == 0) {
    c.workspace[0] = 1;
    c.workspace[1] = static_cast<int32_t>(total);
  }
}

__global__ void __launch_bounds__(256) k_kv_share(const __grid_constant__ xpu_kv_cache_t c, const int32_t *parents,
                                                  const int32_t *children, uint32_t count) {
  if (c.workspace[0] == 0) return;
  const uint32_t i = blockIdx.x;
  const uint32_t full = len_of(c, parents[i]) / c.page_size;
  const int32_t *from = c.tables + static_cast<size_t>(parents[i]) * c.table_width;
  int32_t *to = c.tables + static_cast<size_t>(children[i]) * c.table_width;
  for (uint32_t j = threadIdx.x; j < full; j += blockDim.x) {
    const int32_t p = from[j];
    if (page_ok(c, p)) atomicAdd(&c.refs[p], 1);
    to[j] = p;
  }
}

__global__ void __launch_bounds__(kPlanThreads) k_kv_compact(const __grid_constant__ xpu_kv_cache_t c) {
  __shared__ uint32_t live_total;
  uint32_t live = 0;
  for (uint32_t p = threadIdx.x; p < c.pages; p += kPlanThreads) live += c.refs[p] > 0;
  uint32_t total;
  block_scan(live, &total);
  if (threadIdx.x == 0) live_total = total;
  __syncthreads();
  const uint32_t keep = live_total;
  uint32_t holes = 0, moves = 0;
  for (uint32_t base = 0; base < c.pages; base += kPlanThreads) {
    const uint32_t p = base + threadIdx.x;
    const bool hole = p < keep && c.refs[p] <= 0, move = p >= keep && p < c.pages && c.refs[p] > 0;
    uint32_t n;
    const uint32_t h = holes + block_scan(hole, &n);
    holes += n;
    if (hole) c.workspace[kHeader + kEntry * h + 1] = static_cast<int32_t>(p);
    const uint32_t m = moves + block_scan(move, &n);
    moves += n;
    if (move) c.workspace[kHeader + kEntry * m] = static_cast<int32_t>(p);
  }
  __syncthreads();
  int32_t *renamed = c.workspace + kHeader + kEntry * c.pages;
  for (uint32_t m = threadIdx.x; m < moves; m += kPlanThreads) {
    int32_t *entry = c.workspace + kHeader + kEntry * m;
    entry[2] = static_cast<int32_t>(c.page_size);
    renamed[entry[0]] = entry[1];
    c.refs[entry[1]] = c.refs[entry[0]];
    c.refs[entry[0]] = 0;
  }
  if (threadIdx.x == 0) {
    c.workspace[0] = 1;
    c.workspace[1] = static_cast<int32_t>(moves);
    c.workspace[2] = static_cast<int32_t>(keep);
  }
}

__global__ void __launch_bounds__(256) k_kv_rename(const __grid_constant__ xpu_kv_cache_t c) {
  const int32_t keep = c.workspace[2];
  const int32_t *renamed = c.workspace + kHeader + kEntry * c.pages;
  const uint64_t entries = static_cast<uint64_t>(c.sequences) * c.table_width;
  for (uint64_t e = blockIdx.x * 256ull + threadIdx.x; e < entries; e += gridDim.x * 256ull) {
    const int32_t p = c.tables[e];
    if (p >= keep && page_ok(c, p)) c.tables[e] = renamed[p];
  }
}

// Copies the planned entries: one warp per (entry, layer, K or V, head), whose
// rows are contiguous on both sides.
__global__ void __launch_bounds__(256) k_kv_copy(const __grid_constant__ xpu_kv_cache_t c) {
  const uint32_t entries = static_cast<uint32_t>(c.workspace[1]), lane = threadIdx.x & 31, per_row = c.head_dim / 8;
  const uint64_t per_page = static_cast<uint64_t>(c.kv_heads) * c.page_size * per_row;
  const uint64_t work = static_cast<uint64_t>(entries) * c.layers * 2 * c.kv_heads;
  const uint64_t warps = static_cast<uint64_t>(gridDim.x) * 8;
  for (uint64_t w = blockIdx.x * 8ull + threadIdx.x / 32; w < work; w += warps) {
    const uint32_t head = static_cast<uint32_t>(w % c.kv_heads), which = static_cast<uint32_t>(w / c.kv_heads % 2);
    const uint64_t layer = w / (2 * c.kv_heads) % c.layers;
    const int32_t *entry = c.workspace + kHeader + kEntry * (w / (2ull * c.kv_heads * c.layers));
    if (!page_ok(c, entry[0])) {
      if (lane == 0) atomicOr(c.status, XPU_KV_BAD_INDEX);
      continue;
    }
    uint4 *pool = reinterpret_cast<uint4 *>(which ? c.v : c.k) + layer * c.pages * per_page +
                  static_cast<uint64_t>(head) * c.page_size * per_row;
    const uint4 *src = pool + static_cast<uint64_t>(entry[0]) * per_page;
    uint4 *dst = pool + static_cast<uint64_t>(entry[1]) * per_page;
    for (uint32_t e = lane; e < static_cast<uint32_t>(entry[2]) * per_row; e += 32) dst[e] = src[e];
  }
}

uint32_t blocks_for(uint64_t warps) { return static_cast<uint32_t>(std::min<uint64_t>((warps + 7) / 8, 148 * 8)); }

}  // namespace

size_t kv_workspace_bytes(uint32_t pages) {
  // header, an entry per page (or request), and a page list or the new ids
  return 4 * (kHeader + kEntry * static_cast<size_t>(std::max(pages, XPU_KV_MAX_REQUESTS)) +
              std::max(pages, XPU_KV_MAX_REQUESTS));
}

cudaError_t kv_extend_launch(const xpu_kv_cache_t &c, const int32_t *sequences, const int32_t *starts, uint32_t count,
                             cudaStream_t s) {
  k_kv_extend<<<1, kPlanThreads, 0, s>>>(c, sequences, starts, count);
  return cudaGetLastError();
}

cudaError_t kv_write_launch(const xpu_kv_cache_t &c, const int32_t *sequences, const int32_t *starts, uint32_t count,
                            uint32_t tokens, const int32_t *rows, const void *k, const void *v, uint32_t held,
                            uint64_t layer_stride, uint64_t row_stride, uint32_t layer, uint32_t layers,
                            cudaStream_t s) {
  k_kv_write<<<blocks_for(static_cast<uint64_t>(tokens) * layers * 2), 256, 0, s>>>(
      c, sequences, starts, count, tokens, rows, static_cast<const uint16_t *>(k), static_cast<const uint16_t *>(v), held,
      layer_stride, row_stride, layer, layers);
  return cudaGetLastError();
}

cudaError_t kv_trim_launch(const xpu_kv_cache_t &c, const int32_t *sequences, const int32_t *new_lens, uint32_t count,
                           cudaStream_t s) {
  k_kv_trim<<<1, kPlanThreads, 0, s>>>(c, sequences, new_lens, count);
  return cudaGetLastError();
}

cudaError_t kv_fork_launch(const xpu_kv_cache_t &c, const int32_t *parents, const int32_t *children, uint32_t count,
                           cudaStream_t s) {
  k_kv_fork<<<1, kPlanThreads, 0, s>>>(c, parents, children, count);
  k_kv_share<<<count, 256, 0, s>>>(c, parents, children, count);
  k_kv_copy<<<blocks_for(static_cast<uint64_t>(count) * c.layers * 2 * c.kv_heads), 256, 0, s>>>(c);
  return cudaGetLastError();
}

cudaError_t kv_compact_launch(const xpu_kv_cache_t &c, cudaStream_t s) {
  k_kv_compact<<<1, kPlanThreads, 0, s>>>(c);
  k_kv_rename<<<blocks_for(static_cast<uint64_t>(c.sequences) * c.table_width / 32 + 1), 256, 0, s>>>(c);
  k_kv_copy<<<148 * 8, 256, 0, s>>>(c);
  return cudaGetLastError();
}

}  // namespace xpu
