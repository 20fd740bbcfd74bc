// Page operators of the serving cache (xpu_kv_* in include/xpu_cuda.h).
//
// Each call is one kernel of two parts. One block plans: it checks the whole
// request, takes pages and rewrites lens (or refuses and changes nothing). Then
// all blocks copy what the plan lists. All page choices are by ascending id, so
// the result does not depend on the order in which threads run. The planning
// block is the one that draws ticket 0, hence one that runs, and the others
// wait (bounded) for its flag: nothing depends on which blocks are resident.
//
// Small calls are a chain of memory latencies of 0.6 to 0.8 us each (ticket,
// lists, lens, release, flag, lens, table, rows), so what does not depend on
// the plan is loaded before it: the lists and the first 4096 reference counts
// under the ticket, the rows to be written under the wait.
//
// What the copies move is bound by memory: 32 warps an SM with four to eight
// 16-byte loads in flight each. A row of one head (128 or 256 bytes) is contiguous
// on both sides, a page's rows of one head too. Measured (a trim or free before
// each, as a serving loop has it): 4 prompts of 301 to 2048 tokens, 36 layers, 5.5 TB/s
// read and written (0.85 of a plain copy); 64 forks with pages of 128 5.7 TB/s;
// compaction of a half-empty 9.7 GB pool 5.9 to 6.2 TB/s; 16 sequences' accepted tokens
// 13 us, 4 forks 11 us, where two launches from Python take 9 to 13.
//
// The workspace, zeroed once by the caller: {accepted, entries, first id that
// compaction renames, ticket, ready, blocks that have seen it, sequences of the last extension, -}, per
// entry {source page, new page, rows}, behind those compaction's new ids or a list of free pages, and
// last the extension's sequences {id, length before it}, which no other operator touches:
// its writes may come layer by layer with other calls between them.
#include <algorithm>

#include "common.cuh"
#include "serving.h"
#include "stream.cuh"

namespace xpu {
namespace {

constexpr uint32_t kThreads = 1024, kWarps = kThreads / 32;
constexpr uint32_t kHeader = 8, kEntry = 3;
constexpr uint32_t kFew = 1024;  // pages whose ids a plan keeps in shared memory
enum { kAccepted, kEntries, kRenamedFrom, kTicket, kReady, kSeen, kExtended };
constexpr long long kPlanWaitCycles = 4000000000ll;  // ~2 s at 1.9 GHz

// The next kernel may be set up from here on; this one reads nothing before the
// one before it has ended.
__device__ __forceinline__ void after_previous() {
  grid_dep_launch();
  grid_dep_wait();
}

// 16 bytes of a row that is read once. The rows may come from the kernel before, which can still run
// when this one has begun: coherent loads, kept behind the wait for its end.
__device__ __forceinline__ uint4 ld_row16(const uint4 *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

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

// Reference counts of pages 4 i .. 4 i + 3; behind the pool as if in use.
__device__ __forceinline__ int4 refs4(const xpu_kv_cache_t &c, uint32_t i) {
  int4 r = make_int4(1, 1, 1, 1);
  const uint32_t p = 4 * i;
  if (p + 3 < c.pages && (reinterpret_cast<uintptr_t>(c.refs) & 15u) == 0) return reinterpret_cast<const int4 *>(c.refs)[i];
  if (p < c.pages) r.x = c.refs[p];
  if (p + 1 < c.pages) r.y = c.refs[p + 1];
  if (p + 2 < c.pages) r.z = c.refs[p + 2];
  if (p + 3 < c.pages) r.w = c.refs[p + 3];
  return r;
}

// The `want` lowest free pages in ascending order into list; false if there
// are fewer. first: refs4 of this thread's first pages.
__device__ bool lowest_free(const xpu_kv_cache_t &c, int4 first, uint32_t want, uint32_t *list) {
  uint32_t found = 0;
  for (uint32_t base = 0; base < c.pages && found < want; base += 4 * kThreads) {
    const int4 r = base ? refs4(c, base / 4 + threadIdx.x) : first;
    const int32_t v[4] = {r.x, r.y, r.z, r.w};
    uint32_t total, mine = 0;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) mine += v[e] == 0;
    uint32_t rank = found + block_scan(mine, &total);
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      if (v[e] != 0) continue;
      if (rank < want) list[rank] = base + 4 * threadIdx.x + e;
      ++rank;
    }
    found += total;
  }
  return found >= want;
}

// Marks this thread's sequence id (valid threads only) in a bitmap; true if
// every valid id of the CTA is in range and named once.
__device__ bool named_once(const xpu_kv_cache_t &c, bool valid, int32_t s, uint32_t *bitmap) {
  for (uint32_t i = threadIdx.x; i < XPU_KV_MAX_SEQUENCES / 32; i += kThreads) bitmap[i] = 0;
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
    c.workspace[kAccepted] = 0;
    c.workspace[kEntries] = 0;
  }
}

__device__ __forceinline__ void accept(const xpu_kv_cache_t &c, uint32_t entries) {
  if (threadIdx.x == 0) {
    c.workspace[kAccepted] = 1;
    c.workspace[kEntries] = static_cast<int32_t>(entries);
  }
}

// Runs plan() in the block that comes first and lets the others wait for it;
// false if the plan was refused or the wait gave up. The ticket counts round by
// itself; the flag is taken back by the last block that has seen it.
template <typename Plan>
__device__ bool after_plan(const xpu_kv_cache_t &c, Plan plan) {
  __shared__ int32_t told;
  uint32_t *ws = reinterpret_cast<uint32_t *>(c.workspace);
  if (threadIdx.x == 0) told = atomicInc(ws + kTicket, gridDim.x - 1) == 0 ? 0 : -1;
  __syncthreads();
  const bool planner = told == 0;
  __syncthreads();
  if (planner) {
    plan();
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    int32_t v = 0;
    if (planner) {
      v = c.workspace[kAccepted] ? 1 : 2;
      asm volatile("st.release.gpu.global.s32 [%0], %1;" ::"l"(c.workspace + kReady), "r"(v) : "memory");
    } else {
      const long long start = clock64();
      for (;;) {
        asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(c.workspace + kReady) : "memory");
        if (v || clock64() - start > kPlanWaitCycles) break;
        __nanosleep(20);
      }
      if (!v) atomicOr(c.status, XPU_KV_TIMEOUT);
    }
    told = v;
  }
  __syncthreads();
  if (threadIdx.x == 0 && atomicInc(ws + kSeen, gridDim.x - 1) == gridDim.x - 1) c.workspace[kReady] = 0;
  return told == 1;
}

// Places of the workspace behind the header and the entries.
__host__ __device__ constexpr uint32_t listed_pages(uint32_t pages) { return pages > XPU_KV_MAX_REQUESTS ? pages : XPU_KV_MAX_REQUESTS; }
__host__ __device__ constexpr uint32_t extension_at(uint32_t pages) { return kHeader + (kEntry + 1) * listed_pages(pages); }

// What the plan wrote, read past the L1.
__device__ __forceinline__ int32_t planned(const xpu_kv_cache_t &c, uint32_t at) { return __ldcg(c.workspace + at); }

// ------------------------------------------------------------------ append ----

struct Extension {  // one thread's request
  int32_t sequence, more;
  int4 refs;
  __device__ Extension(const xpu_kv_cache_t &c, const int32_t *sequences, const int32_t *starts, uint32_t count) {
    const uint32_t i = threadIdx.x;
    sequence = i < count ? sequences[i] : -1;
    more = i < count ? starts[i + 1] - starts[i] : 0;
    refs = refs4(c, i);
  }
};

// *before: this thread's sequence's length so far.
__device__ void plan_extend(const xpu_kv_cache_t &c, const Extension &x, uint32_t count, uint32_t *bitmap, uint32_t *few,
                            uint32_t *before) {
  const uint32_t i = threadIdx.x;
  const bool mine = i < count;
  const int32_t s = x.sequence;
  const bool in_range = mine && s >= 0 && static_cast<uint32_t>(s) < c.sequences;
  const uint32_t old = *before = in_range ? len_of(c, s) : 0;
  if (!named_once(c, mine, s, bitmap) || __syncthreads_or(x.more < 0)) return refuse(c, XPU_KV_BAD_SEQUENCE);
  const uint32_t first = pages_of(old, c.page_size);
  const uint64_t after = static_cast<uint64_t>(old) + x.more;
  if (__syncthreads_or(after > static_cast<uint64_t>(c.table_width) * c.page_size)) return refuse(c, XPU_KV_EXHAUSTED);
  const uint32_t need = pages_of(static_cast<uint32_t>(after), c.page_size) - first;
  uint32_t total;
  const uint32_t rank = block_scan(need, &total);
  uint32_t *list = total <= kFew ? few : reinterpret_cast<uint32_t *>(c.workspace) + kHeader;
  if (total > c.pages || !lowest_free(c, x.refs, total, list)) return refuse(c, XPU_KV_EXHAUSTED);
  __syncthreads();
  for (uint32_t j = 0; j < need; ++j) {
    const uint32_t p = list[rank + j];
    c.tables[static_cast<size_t>(s) * c.table_width + first + j] = static_cast<int32_t>(p);
    c.refs[p] = 1;
  }
  if (mine) c.lens[s] = static_cast<int32_t>(after);
  accept(c, 0);
}

struct Rows {
  bool extended;  // the positions of the last extension, else those that this call has added
  const int32_t *rows;
  const uint16_t *k, *v;
  uint32_t tokens, held;
  uint64_t layer_stride, row_stride;
  uint32_t layer, layers;
};

// One warp per (layer, K or V, token): the token's row of every head. What is
// known before the plan, and the row's first 128 pieces.
struct Piece {
  const uint4 *src;
  uint4 v[4];
  uint32_t which, after, t;  // layer * 2 + K or V; tokens of the sequence from this one on, and before it
  uint32_t request;
  int32_t sequence;
};

struct Writer {
  const xpu_kv_cache_t &c;
  const int32_t *sequences, *starts;
  const Rows &r;
  uint32_t count, tokens, shift, chunks, page_shift;
  uint64_t work, warps, w;

  __device__ Writer(const xpu_kv_cache_t &c_, const int32_t *sequences_, const int32_t *starts_, uint32_t count_,
                    const Rows &r_)
      : c(c_), sequences(sequences_), starts(starts_), r(r_), count(count_) {
    const uint32_t listed = static_cast<uint32_t>(max(starts[count], 0));
    if (listed > r.tokens && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(c.status, XPU_KV_BAD_INDEX);
    tokens = min(r.tokens, listed);
    shift = c.head_dim == 128 ? 4 : 3;  // 16-byte pieces of a head's row
    chunks = c.kv_heads << shift;
    page_shift = 31 - __clz(c.page_size);
    work = static_cast<uint64_t>(tokens) * r.layers * 2;
    warps = static_cast<uint64_t>(gridDim.x) * kWarps;
    w = static_cast<uint64_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
  }
  __device__ bool more() const { return w < work; }

  __device__ void fetch(Piece &p) {
    const uint32_t lane = threadIdx.x & 31, t = static_cast<uint32_t>(w % tokens);
    p.which = static_cast<uint32_t>(w / tokens);
    w += warps;
    uint32_t lo = 0, hi = count;  // the last i with starts[i] <= t
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (starts[mid] <= static_cast<int32_t>(t)) lo = mid;
      else hi = mid;
    }
    const int32_t s = sequences[lo], row = r.rows ? r.rows[t] : static_cast<int32_t>(t);
    const int32_t begin = starts[lo], end = starts[lo + 1];
    const bool ok = s >= 0 && static_cast<uint32_t>(s) < c.sequences && row >= 0 && static_cast<uint32_t>(row) < r.held &&
                    static_cast<int32_t>(t) >= begin && static_cast<int32_t>(t) < end;
    p.sequence = ok ? s : -1;
    p.after = static_cast<uint32_t>(end) - t;
    p.t = t - static_cast<uint32_t>(begin);
    p.request = lo;
    p.src = nullptr;
    if (!ok) return;
    p.src = reinterpret_cast<const uint4 *>((p.which & 1 ? r.v : r.k) + (p.which >> 1) * r.layer_stride + row * r.row_stride);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      if (lane + 32 * i < chunks) p.v[i] = ld_row16(p.src + lane + 32 * i);
  }

  __device__ void put(const Piece &p) const {
    const uint32_t lane = threadIdx.x & 31;
    int64_t position = -1;
    if (p.sequence >= 0) {
      const int32_t len = __ldcg(c.lens + p.sequence);
      position = static_cast<int64_t>(len) - p.after;
      if (r.extended) {
        const int32_t *record = c.workspace + extension_at(c.pages) + 2 * p.request;
        position = p.request < static_cast<uint32_t>(planned(c, kExtended)) && __ldcg(record) == p.sequence
                       ? static_cast<int64_t>(__ldcg(record + 1)) + p.t
                       : -1;
        if (position >= len) position = -1;  // trimmed off since
      }
    }
    int32_t page = -1;
    if (position >= 0 && position < static_cast<int64_t>(c.table_width) * c.page_size)
      page = __ldcg(c.tables + static_cast<size_t>(p.sequence) * c.table_width + (position >> page_shift));
    if (!page_ok(c, page)) {
      if (lane == 0) atomicOr(c.status, XPU_KV_BAD_INDEX);
      return;
    }
    const uint32_t slot = static_cast<uint32_t>(position) & (c.page_size - 1), rest = (1u << shift) - 1;
    uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.which & 1 ? c.v : c.k)) +
                 (static_cast<size_t>(r.layer + (p.which >> 1)) * c.pages + page) * chunks * c.page_size;
    auto at = [&](uint32_t e) { return ((static_cast<size_t>(e >> shift) * c.page_size + slot) << shift) + (e & rest); };
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      if (lane + 32 * i < chunks) __stcs(dst + at(lane + 32 * i), p.v[i]);
    for (uint32_t e = lane + 128; e < chunks; e += 32) dst[at(e)] = ld_row16(p.src + e);
  }

  // `have`: the first piece is fetched already
  __device__ void run(Piece &first, bool have) {
    Piece p = first;
    while (have) {
      Piece following;
      const bool another = more();
      if (another) fetch(following);
      put(p);
      p = following;
      have = another;
    }
  }
};

__global__ void __launch_bounds__(kThreads) k_kv_extend(const __grid_constant__ xpu_kv_cache_t c, const int32_t *sequences,
                                                        const int32_t *starts, uint32_t count) {
  __shared__ uint32_t bitmap[XPU_KV_MAX_SEQUENCES / 32], few[kFew];
  after_previous();
  const Extension x(c, sequences, starts, count);
  uint32_t before;
  plan_extend(c, x, count, bitmap, few, &before);
  __syncthreads();
  const bool accepted = c.workspace[kAccepted];
  if (accepted && threadIdx.x < count) {
    int32_t *record = c.workspace + extension_at(c.pages) + 2 * threadIdx.x;
    record[0] = x.sequence;
    record[1] = static_cast<int32_t>(before);
  }
  if (threadIdx.x == 0) c.workspace[kExtended] = accepted ? static_cast<int32_t>(count) : 0;
}

__global__ void __launch_bounds__(kThreads) k_kv_write(const __grid_constant__ xpu_kv_cache_t c, const int32_t *sequences,
                                                       const int32_t *starts, uint32_t count,
                                                       const __grid_constant__ Rows r) {
  after_previous();
  if (!planned(c, kExtended)) return;  // refused
  Writer writer(c, sequences, starts, count, r);
  Piece first;
  const bool have = writer.more();
  if (have) writer.fetch(first);
  writer.run(first, have);
}

__global__ void __launch_bounds__(kThreads) k_kv_append(const __grid_constant__ xpu_kv_cache_t c, const int32_t *sequences,
                                                        const int32_t *starts, uint32_t count,
                                                        const __grid_constant__ Rows r) {
  __shared__ uint32_t bitmap[XPU_KV_MAX_SEQUENCES / 32], few[kFew];
  after_previous();
  const Extension x(c, sequences, starts, count);
  Writer writer(c, sequences, starts, count, r);
  Piece first;
  const bool have = writer.more();
  if (have) writer.fetch(first);
  uint32_t before;
  if (after_plan(c, [&] { plan_extend(c, x, count, bitmap, few, &before); })) writer.run(first, have);
}

// -------------------------------------------------------------------- trim ----

__global__ void __launch_bounds__(kThreads) k_kv_trim(const __grid_constant__ xpu_kv_cache_t c, const int32_t *sequences,
                                                      const int32_t *new_lens, uint32_t count) {
  __shared__ uint32_t bitmap[XPU_KV_MAX_SEQUENCES / 32];
  __shared__ uint32_t range[XPU_KV_MAX_REQUESTS][2];
  after_previous();
  const uint32_t i = threadIdx.x;
  const bool mine = i < count;
  const int32_t s = mine ? sequences[i] : -1, want = mine ? new_lens[i] : 0;
  if (!named_once(c, mine, s, bitmap) || __syncthreads_or(want < 0)) return refuse(c, XPU_KV_BAD_SEQUENCE);
  const uint32_t old = mine ? len_of(c, s) : 0, len = min(old, static_cast<uint32_t>(want));
  bool cut = false;
  if (len < old && len % c.page_size) {
    const int32_t p = c.tables[static_cast<size_t>(s) * c.table_width + len / c.page_size];
    cut = page_ok(c, p) && c.refs[p] > 1;
  }
  if (__syncthreads_or(cut)) return refuse(c, XPU_KV_SHARED_CUT);
  range[i][0] = pages_of(len, c.page_size);
  range[i][1] = pages_of(old, c.page_size);
  if (mine) c.lens[s] = static_cast<int32_t>(len);
  __syncthreads();
  // a warp per sequence, so that a long table is let go of by many threads
  for (uint32_t q = threadIdx.x / 32; q < count; q += kWarps) {
    int32_t *table = c.tables + static_cast<size_t>(sequences[q]) * c.table_width;
    for (uint32_t j = range[q][0] + (threadIdx.x & 31); j < range[q][1]; j += 32) {
      const int32_t p = table[j];
      if (page_ok(c, p)) atomicSub(&c.refs[p], 1);
      table[j] = -1;
    }
  }
}

// ---------------------------------------------------------- fork and compact ----

// Copies the planned entries: one warp per (entry, layer, K or V, head).
__device__ void copy_entries(const xpu_kv_cache_t &c) {
  const uint32_t entries = static_cast<uint32_t>(planned(c, kEntries)), lane = threadIdx.x & 31, per_row = c.head_dim / 8;
  const uint64_t per_page = static_cast<uint64_t>(c.kv_heads) * c.page_size * per_row;
  const uint32_t per_entry = c.layers * 2 * c.kv_heads;
  const uint64_t work = static_cast<uint64_t>(entries) * per_entry, warps = static_cast<uint64_t>(gridDim.x) * kWarps;
  for (uint64_t w = static_cast<uint64_t>(blockIdx.x) * kWarps + threadIdx.x / 32; w < work; w += warps) {
    const uint32_t at = static_cast<uint32_t>(w / per_entry), part = static_cast<uint32_t>(w % per_entry);
    const uint32_t head = part % c.kv_heads, which = part / c.kv_heads;  // layer * 2 + K or V
    const int32_t from = planned(c, kHeader + kEntry * at), to = planned(c, kHeader + kEntry * at + 1);
    const uint32_t pieces = static_cast<uint32_t>(planned(c, kHeader + kEntry * at + 2)) * per_row;
    if (!page_ok(c, from)) {
      if (lane == 0) atomicOr(c.status, XPU_KV_BAD_INDEX);
      continue;
    }
    uint4 *pool = reinterpret_cast<uint4 *>(which & 1 ? c.v : c.k) + static_cast<uint64_t>(which >> 1) * c.pages * per_page +
                  static_cast<uint64_t>(head) * c.page_size * per_row;
    const uint4 *src = pool + static_cast<uint64_t>(from) * per_page;
    uint4 *dst = pool + static_cast<uint64_t>(to) * per_page;
    for (uint32_t e0 = lane; e0 < pieces; e0 += 256) {
      uint4 v[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        if (e0 + 32 * i < pieces) v[i] = src[e0 + 32 * i];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        if (e0 + 32 * i < pieces) dst[e0 + 32 * i] = v[i];
    }
  }
}

__device__ void plan_fork(const xpu_kv_cache_t &c, int32_t from, int32_t to, int4 refs, uint32_t count, uint32_t *bitmap,
                          uint32_t *few) {
  const uint32_t i = threadIdx.x;
  const bool mine = i < count;
  bool bad = mine && (from < 0 || static_cast<uint32_t>(from) >= c.sequences);
  const uint32_t len = mine && !bad ? len_of(c, from) : 0, part = len % c.page_size;
  bad = !named_once(c, mine, to, bitmap) || __syncthreads_or(bad);
  if (!bad) bad = mine && (len_of(c, to) != 0 || (bitmap[from >> 5] >> (from & 31) & 1u));
  if (__syncthreads_or(bad)) return refuse(c, XPU_KV_BAD_SEQUENCE);
  const int32_t last = part ? c.tables[static_cast<size_t>(from) * c.table_width + len / c.page_size] : -1;
  uint32_t total;
  const uint32_t rank = block_scan(part != 0, &total);
  if (total > c.pages || !lowest_free(c, refs, total, few)) return refuse(c, XPU_KV_EXHAUSTED);
  __syncthreads();
  if (part) {
    const int32_t p = static_cast<int32_t>(few[rank]);
    int32_t *entry = c.workspace + kHeader + kEntry * rank;
    entry[0] = last;
    entry[1] = p;
    entry[2] = static_cast<int32_t>(part);
    c.refs[p] = 1;
    c.tables[static_cast<size_t>(to) * c.table_width + len / c.page_size] = p;
  }
  if (mine) c.lens[to] = static_cast<int32_t>(len);
  accept(c, total);
}

__global__ void __launch_bounds__(kThreads) k_kv_fork(const __grid_constant__ xpu_kv_cache_t c, const int32_t *parents,
                                                      const int32_t *children, uint32_t count) {
  static_assert(kFew >= XPU_KV_MAX_REQUESTS, "a page per child");
  __shared__ uint32_t bitmap[XPU_KV_MAX_SEQUENCES / 32], few[kFew];
  after_previous();
  const int32_t from = threadIdx.x < count ? parents[threadIdx.x] : -1, to = threadIdx.x < count ? children[threadIdx.x] : -1;
  const int4 refs = refs4(c, threadIdx.x);
  if (!after_plan(c, [&] { plan_fork(c, from, to, refs, count, bitmap, few); })) return;
  // full pages are shared: a warp per child
  for (uint32_t i = blockIdx.x * kWarps + threadIdx.x / 32; i < count; i += gridDim.x * kWarps) {
    const uint32_t full = len_of(c, parents[i]) / c.page_size;
    const int32_t *row = c.tables + static_cast<size_t>(parents[i]) * c.table_width;
    int32_t *copy = c.tables + static_cast<size_t>(children[i]) * c.table_width;
    for (uint32_t j = threadIdx.x & 31; j < full; j += 32) {
      const int32_t p = row[j];
      if (page_ok(c, p)) atomicAdd(&c.refs[p], 1);
      copy[j] = p;
    }
  }
  copy_entries(c);
}

__device__ void plan_compact(const xpu_kv_cache_t &c, int4 first) {
  uint32_t live = 0;
  for (uint32_t i = threadIdx.x; 4 * i < c.pages; i += kThreads) {
    const int4 r = i == threadIdx.x ? first : refs4(c, i);
    const uint32_t p = 4 * i;
    live += (r.x > 0) + (p + 1 < c.pages && r.y > 0) + (p + 2 < c.pages && r.z > 0) + (p + 3 < c.pages && r.w > 0);
  }
  uint32_t keep;
  block_scan(live, &keep);
  uint32_t holes = 0, moves = 0;
  for (uint32_t base = 0; base < c.pages; base += 4 * kThreads) {
    const uint32_t p = base + 4 * threadIdx.x;
    const int4 r = base ? refs4(c, base / 4 + threadIdx.x) : first;
    const int32_t v[4] = {r.x, r.y, r.z, r.w};
    uint32_t n = 0, total;  // holes in the low half, moves in the high half
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e)
      n += (p + e < keep && v[e] <= 0) + ((p + e >= keep && p + e < c.pages && v[e] > 0) << 16);
    const uint32_t before = block_scan(n, &total);
    uint32_t h = holes + (before & 0xffffu), m = moves + (before >> 16);
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      if (p + e < keep && v[e] <= 0) c.workspace[kHeader + kEntry * h++ + 1] = static_cast<int32_t>(p + e);
      if (p + e >= keep && p + e < c.pages && v[e] > 0) c.workspace[kHeader + kEntry * m++] = static_cast<int32_t>(p + e);
    }
    holes += total & 0xffffu;
    moves += total >> 16;
  }
  __syncthreads();
  int32_t *renamed = c.workspace + kHeader + kEntry * c.pages;
  for (uint32_t m = threadIdx.x; m < moves; m += kThreads) {
    int32_t *entry = c.workspace + kHeader + kEntry * m;
    entry[2] = static_cast<int32_t>(c.page_size);
    renamed[entry[0]] = entry[1];
    c.refs[entry[1]] = c.refs[entry[0]];
    c.refs[entry[0]] = 0;
  }
  if (threadIdx.x == 0) c.workspace[kRenamedFrom] = static_cast<int32_t>(keep);
  accept(c, moves);
}

__global__ void __launch_bounds__(kThreads) k_kv_compact(const __grid_constant__ xpu_kv_cache_t c) {
  after_previous();
  const int4 refs = refs4(c, threadIdx.x);
  if (!after_plan(c, [&] { plan_compact(c, refs); })) return;
  const int32_t keep = planned(c, kRenamedFrom), renamed = static_cast<int32_t>(kHeader + kEntry * c.pages);
  const uint64_t entries = static_cast<uint64_t>(c.sequences) * c.table_width;
  for (uint64_t e = static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x; e < entries;
       e += static_cast<uint64_t>(gridDim.x) * kThreads) {
    const int32_t p = c.tables[e];
    if (p >= keep && page_ok(c, p)) c.tables[e] = planned(c, static_cast<uint32_t>(renamed + p));
  }
  copy_entries(c);
}

uint32_t blocks_for(uint64_t warps) {
  return static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>((warps + kWarps - 1) / kWarps, sm_count())));
}

}  // namespace

size_t kv_workspace_bytes(uint32_t pages) {
  // header, an entry per page (or request), a page list or the new ids, and the last extension
  return 4 * (kHeader + (kEntry + 1) * static_cast<size_t>(listed_pages(pages)) + 2 * XPU_KV_MAX_REQUESTS);
}

cudaError_t kv_extend_launch(const xpu_kv_cache_t &c, const int32_t *sequences, const int32_t *starts, uint32_t count,
                             cudaStream_t s) {
  return launch_after(k_kv_extend, 1, kThreads, 0, s, c, sequences, starts, count);
}

cudaError_t kv_write_launch(const xpu_kv_cache_t &c, const int32_t *sequences, const int32_t *starts, uint32_t count,
                            uint32_t tokens, const int32_t *rows, const void *k, const void *v, uint32_t held,
                            uint64_t layer_stride, uint64_t row_stride, uint32_t layer, uint32_t layers, bool extend,
                            cudaStream_t s) {
  const Rows r{!extend, rows, static_cast<const uint16_t *>(k), static_cast<const uint16_t *>(v), tokens, held, layer_stride, row_stride,
               layer, layers};
  const uint32_t blocks = blocks_for(static_cast<uint64_t>(tokens) * layers * 2);
  return launch_after(extend ? k_kv_append : k_kv_write, blocks, kThreads, 0, s, c, sequences, starts, count, r);
}

cudaError_t kv_trim_launch(const xpu_kv_cache_t &c, const int32_t *sequences, const int32_t *new_lens, uint32_t count,
                           cudaStream_t s) {
  return launch_after(k_kv_trim, 1, kThreads, 0, s, c, sequences, new_lens, count);
}

cudaError_t kv_fork_launch(const xpu_kv_cache_t &c, const int32_t *parents, const int32_t *children, uint32_t count,
                           cudaStream_t s) {
  return launch_after(k_kv_fork, blocks_for(static_cast<uint64_t>(count) * c.layers * 2 * c.kv_heads), kThreads, 0, s, c,
                      parents, children, count);
}

cudaError_t kv_compact_launch(const xpu_kv_cache_t &c, cudaStream_t s) {
  return launch_after(k_kv_compact, blocks_for(static_cast<uint64_t>(c.pages) / 2 * c.layers * 2 * c.kv_heads), kThreads, 0,
                      s, c);
}

}  // namespace xpu
