// Attention of the serving path: causal over packed prompts, and of drafted
// token trees over the paged cache (xpu_prompt_attention and
// xpu_tree_attention in include/xpu_cuda.h).
//
// Both are  out_r = sum_j p_rj v_j / sum_j p_rj,  p_rj = exp(scale q_r . k_j - m_r)
// over the keys j that row r may attend, taken 128 keys at a time with the
// running maximum and sum of a softmax, both products on the tensor cores
// (tcgen05). A row is one query head of one position (node); a row tile is the
// 128 rows of 128 / group positions, all query heads of one kv head, so one
// read of a key serves the whole group. A thread block works on a segment: up
// to two row tiles against a run of key tiles. Twelve warps:
//   0-3, 4-7  softmax of row tile 0 / 1, one thread a row: scores from TMEM,
//             mask, maximum, p = 2^(c s - c m) with c = scale log2 e, p rounded
//             to the input type and written back to TMEM over the scores as the
//             A operand of the second product; FP32 sum of the unrounded p.
//             The reference maximum m moves only when the true one has passed
//             it by 2^8 (fp16: 2^4), so the accumulator in TMEM is rarely
//             rescaled; in fp16 p is 2^11 times as large, for its range (Weights).
//             At the end out = O / l, rounded once;
//   8         issues S_t = Q_t K^T (both operands in shared memory) and O_t +=
//             P_t V (P from TMEM, V as it stands in memory, MN-major); S_t overwrites
//             the P_t that the product before it read. While one tile is in its
//             softmax the tensor cores work for the other;
//   9         TMA loads: Q tiles, and a ring of K and V tiles (trees: V by warp 10);
//   10, 11    cleaning (trees: 11): in key tiles with masked keys, V rows that no row may
//             attend are zeroed (0 x NaN would reach the sums), and rows with
//             non-finite values are zeroed and listed; the rows that do attend
//             them get p v added at the end (add_listed).
// A segment of at most 128 rows (drafted trees, mostly) would leave one softmax
// group idle: there both groups work for the same rows, on even and odd key
// tiles, and join their sums at the end.
//
// What bounds it. Long prompts: per pair of row tiles and key tile the tensor
// cores need 2048 cycles (32 instructions of 64) and the loop takes about 3200,
// the chain scores -> softmax (about 2000 cycles, half of them the special
// function unit's) -> P V -> next scores of one tile; 8192 tokens, 32/8 heads: 412
// us (1335 TFLOP/s) for a few passes, 493 us (1110) kept up under the power limit
// (B200's cuBLAS: 1707 and 1405). Emulating a part of the exponentials on the FMA
// pipe, half tiles of 64 keys (64-column score products run at 55 cycles, not 32)
// and starting the exponentials with the old maximum were all slower. Trees of up
// to 32 nodes: reading the cache, 5.4 TB/s (16 x 12288 positions, pages of 16).
//
// Waits are bounded; a timeout sets a sticky device word that
// xpu_device_status reads, and every role leaves.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <functional>
#include <queue>
#include <vector>

#include "common.cuh"
#include "serving.h"
#include "stream.cuh"
#include "tcgen05.cuh"

namespace xpu {

__device__ unsigned int g_attention_error = 0;

namespace {

constexpr uint32_t kKeys = 128;        // keys per tile
constexpr uint32_t kBox = 128 * 128;   // bytes of 128 rows x 64 elements, 128-byte swizzled
constexpr uint32_t kThreads = 384;
constexpr uint32_t kMmaWarp = 8, kLoadWarp = 9, kCleanWarp = 10;
constexpr unsigned kErrAttentionTimeout = 4u;
constexpr uint32_t kBadRing = 8;
constexpr uint32_t kEarlyKeys = 96;    // of a tile's probabilities, handed to the tensor cores before the rest
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Powers of two: how far a maximum may pass the reference before the accumulator is rescaled, and
// the weight of the reference itself, so that no weight passes 2^15. bf16 holds FP32's exponents.
// fp16's smallest step is 2^-24: lifted by 2^kLift, weights keep their relative rounding down to
// 2^-(14 + kLift) of the reference's and are lost below 2^-(25 + kLift), not below 2^-25, where many
// of them can still make up the result (16384 keys 17.5 nats below one). The sum of weights is lifted
// with them; its logarithm takes the lift out. Rescaling from 2^4 on costs 16 packed prompts of 1 to 2047
// tokens, 16/8 heads, 149 -> 154 us (2^6 with a lift of 9: 149, with a quarter of the range lost).
template <typename T>
struct Weights {
  static constexpr float kRescale = 8.f, kLift = 0.f;
};
template <>
struct Weights<__half> {
  static constexpr float kRescale = 4.f, kLift = 15.f - kRescale;
};

template <int D, bool TREE>
struct Shape {
  static constexpr uint32_t kBoxes = D / 64, kTile = kBoxes * kBox;
  // as many K/V tiles in flight as the shared memory holds beside Q
  static constexpr uint32_t kStages = D == 64 ? 8 : (TREE ? 4 : 5);
  static constexpr uint32_t kSmem = 1024 + (2 + kStages) * kTile;
};

struct BadRows {  // listed keys of one half (64 keys) of up to two tiles of a segment
  uint32_t tiles;
  uint32_t tile[2], mask[2][2];
};

struct TreeEntry {
  uint32_t first, units;  // key tiles and units (row block, kv head) of the sequences before this one
  uint32_t len, begin, named;  // cached positions, first node, sequence * 128 + nodes
};

struct Barriers {
  uint64_t q_full, q_empty, drain;
  uint64_t kv_full[8], kv_empty[8], clean[8];
  uint64_t s_full[2], p_early[2], p_ready[2], o_full[2], joined;
  uint32_t tmem;
  int failed;
  uint32_t ended[8];  // segments that each softmax warp is done with
  BadRows bad[kBadRing][2];
};

struct TreeArgs {
  xpu_kv_cache_t cache;
  const int32_t *sequences, *starts;
  const uint64_t *ancestors;
  uint32_t layer, count, page_shift;  // page_size = 2^page_shift
  uint32_t *arrived;  // per block: parts of the unit that begins there, 0 between calls
  float *partial;     // two slots a block, as partial_rows() places them, then the rows' {m, l}
};

struct Args {
  CUtensorMap q, k, v;              // packed
  CUtensorMap cached_k, cached_v;   // one layer of the pool, 64 elements x page
  AttnTensors t;
  const int32_t *plan;
  TreeArgs tree;
};

// A run of key tiles for one or two row tiles.
struct Segment {
  uint32_t q0, npos, head;   // first position's row of q, positions, kv head
  uint32_t base, len, pos0;  // prompt: key 0's row, prompt length, first position. tree: first node, cached
                             // positions, first node of the segment
  uint32_t nodes;            // tree
  int32_t sequence;
  uint32_t first, n, n0, n1; // key tiles: first, all, row tile 0's, row tile 1's
  uint32_t masked_from;      // the first key tile that some row may not attend as a whole
  bool both;                 // both softmax groups on row tile 0, even and odd key tiles
  int32_t slot;              // partial result, -1 = whole
  uint32_t unit, unit_size;  // the whole unit in the cut of all work
};

// ------------------------------------------------------------ small parts ----

__device__ __forceinline__ bool failed(const Barriers &b) { return *const_cast<const volatile int *>(&b.failed) != 0; }
// The same answers for the whole warp, so that its lanes leave together.
__device__ __forceinline__ bool warp_failed(const Barriers &b) { return __any_sync(kFullMask, failed(b)); }
__device__ __forceinline__ bool warp_wait(Barriers &b, uint64_t *bar, uint32_t parity) {
  if (__all_sync(kFullMask, mbar_wait(bar, parity))) return true;
  b.failed = 1;
  return false;
}

// The cleaning warps, before they list segment `segment`: every softmax warp is done with the
// segment that had its ring entry. A count and not an mbarrier, whose two phases the softmax
// warps could pass both while a cleaning warp is late.
__device__ __forceinline__ bool wait_listed(Barriers &b, uint32_t segment) {
  if (segment < kBadRing) return true;
  const volatile uint32_t *ended = b.ended + (threadIdx.x & 7);
  const long long start = clock64();
  while (!__all_sync(kFullMask, *ended > segment - kBadRing)) {
    if (warp_failed(b)) return false;
    if (__any_sync(kFullMask, clock64() - start > kWaitCycles)) {
      b.failed = 1;
      return false;
    }
  }
  __threadfence_block();
  return true;
}

// A value that all lanes hold, in a form the compiler knows to be uniform.
__device__ __forceinline__ uint32_t same(uint32_t v) { return __shfl_sync(kFullMask, v, 0); }

__host__ __device__ constexpr uint32_t attn_idesc(bool fp16, uint32_t n, bool b_kmajor) {
  return (1u << 4) | ((fp16 ? 0u : 1u) << 7) | ((fp16 ? 0u : 1u) << 10) | ((b_kmajor ? 0u : 1u) << 16) | ((n >> 3) << 17) |
         ((128u >> 4) << 24);  // FP32 accumulator, A and B types, B's order, N, M = 128
}

// D (TMEM) += A (TMEM) . B (shared memory)
__device__ __forceinline__ void mma1_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

#define XPU_R32(r)                                                                                                  \
  "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),        \
      "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),         \
      "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),        \
      "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])

// This warp's 32 TMEM lanes x 32 columns; several may be in flight before tmem_wait_ld().
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : XPU_R32(r)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// tmem_wait_ld() that the 64 values loaded before it cannot be used ahead of.
__device__ __forceinline__ void tmem_wait_ld64(uint32_t *x) {
#define XPU_RW(i) "+r"(x[i]), "+r"(x[i + 1]), "+r"(x[i + 2]), "+r"(x[i + 3]), "+r"(x[i + 4]), "+r"(x[i + 5]), "+r"(x[i + 6]), "+r"(x[i + 7])
  asm volatile("tcgen05.wait::ld.sync.aligned;" : XPU_RW(0), XPU_RW(8), XPU_RW(16)::"memory");
  asm volatile("" : XPU_RW(24), XPU_RW(32), XPU_RW(40)::"memory");
  asm volatile("" : XPU_RW(48), XPU_RW(56)::"memory");
#undef XPU_RW
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, uint32_t x, uint32_t y, uint32_t z,
                                            uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two FP32 numbers in one 64-bit register, and the packed operations on them.
struct Pair {
  uint64_t v;
  __device__ __forceinline__ Pair(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ explicit Pair(uint64_t w) : v(w) {}
  __device__ __forceinline__ void get(float &lo, float &hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
};
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a.v), "l"(b.v), "l"(c.v));
  return Pair(d);
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a.v), "l"(b.v));
  return Pair(d);
}
// Natural logarithm of 2^(c m - lift) l; -inf where the sum is empty.
template <typename T>
__device__ __forceinline__ float log_sum(float m, float l, float c) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(l));
  return l == 0.f ? -INFINITY : fmaf(m, c, y - Weights<T>::kLift) * kLn2;
}
// Largest of three, NaN if one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// 0 w + sum of both 16-bit halves: the sum stays 0 until a half is infinite or
// NaN, and is NaN from then on.
template <typename T>
__device__ __forceinline__ uint32_t add_zero_times(uint32_t w, uint32_t sum) {
  uint32_t d;
  if (std::is_same<T, __half>::value) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(w), "r"(0u), "r"(sum));
  else asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(w), "r"(0u), "r"(sum));
  return d;
}

// Rows of 64 bytes, one in each lane's registers, stored so that the four lanes
// of a quad write one row at a time: 64 bytes in a row where a lane's own row
// would make 32 lines of every store (the epilogue took 4000 cycles that way).
struct QuadRows {
  unsigned long long row[4];  // the quad's rows
  uint32_t stores;            // a bit per lane whose row is stored
  __device__ QuadRows(void *own, bool store) {
    const uint32_t lane = threadIdx.x & 31;
    stores = __ballot_sync(kFullMask, store);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      row[k] = __shfl_sync(kFullMask, reinterpret_cast<unsigned long long>(own), (lane & 28) + k) + (lane & 3) * 16;
  }
  __device__ bool any() const { return stores != 0; }
  // 16 words of this lane's row, for its bytes `at` ...
  __device__ void put(const uint32_t *w, uint32_t at) const {
    const uint32_t lane = threadIdx.x & 31;
    uint4 v[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) v[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    // a 4 x 4 transposition: lane i of the quad ends with piece i of row k in v[k]
    auto swap = [&](uint4 &low, uint4 &high, uint32_t bit) {
      const bool up = lane & bit;
      const uint4 away = up ? low : high;
      uint4 come;
      come.x = __shfl_xor_sync(kFullMask, away.x, bit);
      come.y = __shfl_xor_sync(kFullMask, away.y, bit);
      come.z = __shfl_xor_sync(kFullMask, away.z, bit);
      come.w = __shfl_xor_sync(kFullMask, away.w, bit);
      if (up) low = come;
      else high = come;
    };
    swap(v[0], v[1], 1);
    swap(v[2], v[3], 1);
    swap(v[0], v[2], 2);
    swap(v[1], v[3], 2);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      if (stores >> ((lane & 28) + k) & 1u) *reinterpret_cast<uint4 *>(row[k] + at) = v[k];
  }
};

// --------------------------------------------------------------- segments ----

// The prompt plan's items of this block, in order.
struct PromptWalk {
  const int4 *items;
  int32_t i, end;
  uint32_t positions, tokens;
  __device__ PromptWalk(const Args &a, uint32_t group) {
    items = reinterpret_cast<const int4 *>(a.plan + plan_items_at(static_cast<uint32_t>(a.plan[0])));
    i = a.plan[kPlanHeader + blockIdx.x];
    end = a.plan[kPlanHeader + blockIdx.x + 1];
    positions = tile_positions(group);
    tokens = a.t.tokens;
  }
  __device__ bool next(Segment &s) {
    if (i >= end) return false;
    const int4 it = items[i++];
    s.base = it.x;
    s.len = it.y;
    s.pos0 = it.z;
    s.head = it.w;
    s.q0 = s.base + s.pos0;
    s.npos = min(2 * positions, s.len - s.pos0);
    s.first = 0;
    s.n0 = (s.pos0 + min(positions, s.npos) - 1) / kKeys + 1;
    s.n1 = s.npos > positions ? (s.pos0 + s.npos - 1) / kKeys + 1 : 0;
    s.n = max(s.n0, s.n1);
    s.masked_from = (s.pos0 + 1) / kKeys;
    s.both = false;
    s.slot = -1;
    s.nodes = 0;
    s.sequence = 0;
    return true;
  }
};

__device__ __forceinline__ uint32_t entry_tiles(const TreeEntry &e) { return (e.len + kKeys - 1) / kKeys + 1; }
__device__ __forceinline__ uint32_t entry_nodes(const TreeEntry &e) { return e.named & 127u; }

// One thread's sequence of the tree call, from the device's lists, every value
// brought into range.
struct TreeRequest {
  int32_t begin, end, sequence, len;
  bool mine;
  __device__ TreeRequest(const TreeArgs &a, uint32_t i) : begin(0), end(0), sequence(-1), len(0), mine(i < a.count) {
    if (!mine) return;
    begin = a.starts[i];
    end = a.starts[i + 1];
    sequence = a.sequences[i];
    if (sequence >= 0 && static_cast<uint32_t>(sequence) < a.cache.sequences) len = a.cache.lens[sequence];
  }
};

// Fills table[0 .. count] (count + 1 entries: the last holds the totals); all
// threads of the block. `first`: this thread's first request.
__device__ void tree_table(const TreeArgs &a, uint32_t tokens, uint32_t kv_heads, uint32_t group, TreeEntry *table,
                           uint2 *scratch, const TreeRequest &first) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const xpu_kv_cache_t &c = a.cache;
  const int32_t longest = static_cast<int32_t>(c.table_width * c.page_size);
  uint2 before = make_uint2(0, 0);
  bool bad = false;
  for (uint32_t at = 0; at < a.count; at += blockDim.x) {
    const TreeRequest r = at ? TreeRequest(a, at + threadIdx.x) : first;
    TreeEntry e{0, 0, 0, 0, 0};
    uint32_t tiles = 0, units = 0;
    if (r.mine) {
      const bool listed = r.begin >= 0 && r.end >= r.begin && static_cast<uint32_t>(r.end) <= tokens;
      const bool named = r.sequence >= 0 && static_cast<uint32_t>(r.sequence) < c.sequences;
      bad |= !listed || !named || r.len < 0 || r.len > longest ||
             (listed && r.end - r.begin > static_cast<int32_t>(XPU_TREE_MAX_NODES));
      const uint32_t nodes = listed ? min(static_cast<uint32_t>(r.end - r.begin), XPU_TREE_MAX_NODES) : 0;
      e.len = static_cast<uint32_t>(min(max(r.len, 0), longest));
      e.begin = listed ? static_cast<uint32_t>(r.begin) : 0;
      e.named = (named ? static_cast<uint32_t>(r.sequence) : 0) * 128u + nodes;
      const uint32_t span = 2 * tile_positions(group);
      units = (nodes + span - 1) / span * kv_heads;
      tiles = units * entry_tiles(e);
    }
    uint32_t inc = tiles, inc_units = units;
#pragma unroll
    for (uint32_t o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(kFullMask, inc, o), up_units = __shfl_up_sync(kFullMask, inc_units, o);
      if (lane >= o) inc += up, inc_units += up_units;
    }
    if (at) __syncthreads();
    if (lane == 31) scratch[warp] = make_uint2(inc, inc_units);
    __syncthreads();
    e.first = before.x + inc - tiles;
    e.units = before.y + inc_units - units;
    for (uint32_t w = 0; w < warps; ++w) {
      const uint2 sum = scratch[w];
      if (w < warp) e.first += sum.x, e.units += sum.y;
      before.x += sum.x, before.y += sum.y;
    }
    if (r.mine) table[at + threadIdx.x] = e;
  }
  if (threadIdx.x == 0) table[a.count] = TreeEntry{before.x, before.y, 0, 0, 0};
  if (bad && blockIdx.x == 0) atomicOr(c.status, XPU_KV_BAD_INDEX);
}

// How the work is cut: every unit counts as its key tiles and `lead` more, for
// what beginning and ending one costs (about 10,000 cycles, three to four tiles), and
// each block gets the same number (geometric mean over 16 random batches with 3, 4, 5, 6 and
// 8 more: 31.7, 31.4, 31.6, 31.5 and 31.8 us). With no more tiles than blocks it is one tile each
// (2048 positions, 8 kv heads: 12.4 us in a graph; two each, with blocks that end one unit
// and begin the next, 15.9 us).
struct TreeCut {
  uint32_t lead, share, total;
  __device__ TreeCut(const TreeEntry &sums, uint32_t blocks) {
    lead = sums.first > blocks ? 4 : 0;
    total = sums.first + lead * sums.units;
    share = max((total + blocks - 1) / blocks, 1u);
  }
  __device__ uint32_t at(const TreeEntry &e) const { return e.first + lead * e.units; }
};

// This block's share of all (sequence, row block, kv head, key tile), in that order.
struct TreeWalk {
  const TreeEntry *table;
  TreeCut cut;
  uint32_t group, kv_heads, i, at, begin, end;
  __device__ TreeWalk(const Args &a, const TreeEntry *t, uint32_t g)
      : table(t), cut(t[a.tree.count], gridDim.x), group(g), kv_heads(a.t.kv_heads) {
    begin = at = min(cut.total, blockIdx.x * cut.share);
    end = min(cut.total, begin + cut.share);
    uint32_t lo = 0, hi = a.tree.count;  // the last entry that starts at or before `at`
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (cut.at(table[mid]) <= at) lo = mid;
      else hi = mid;
    }
    i = lo;
  }
  __device__ bool next(Segment &s) {
    for (;;) {
      if (at >= end) return false;
      while (cut.at(table[i + 1]) <= at) ++i;
      const TreeEntry e = table[i];
      const uint32_t tiles = entry_tiles(e), size = cut.lead + tiles, off = at - cut.at(e), unit = off / size;
      const uint32_t in = off - unit * size, stop = min(size, in + end - at), positions = tile_positions(group);
      at += stop - in;
      if (stop <= cut.lead) continue;  // nothing of the unit but its lead
      s.first = max(in, cut.lead) - cut.lead;
      s.n = stop - cut.lead - s.first;
      const uint32_t block = unit / kv_heads;
      s.head = unit - block * kv_heads;
      s.pos0 = block * 2 * positions;
      s.nodes = entry_nodes(e);
      s.npos = min(2 * positions, s.nodes - s.pos0);
      s.base = e.begin;
      s.q0 = e.begin + s.pos0;
      s.len = e.len;
      s.masked_from = e.len / kKeys;
      s.sequence = static_cast<int32_t>(e.named >> 7);
      s.both = s.npos <= positions;
      s.n0 = s.both ? (s.n + 1) / 2 : s.n;
      s.n1 = s.both ? s.n / 2 : s.n;
      s.unit = cut.at(e) + unit * size;
      s.unit_size = size;
      s.slot = s.n == tiles ? -1 : static_cast<int32_t>(2 * blockIdx.x + (begin >= s.unit ? 0 : 1));
      return true;
    }
  }
};

// Key tile `tile` of a segment holds this many keys that some row may attend.
template <bool TREE>
__device__ __forceinline__ uint32_t valid_keys(const Segment &s, uint32_t tile) {
  if (TREE && tile * kKeys >= s.len) return s.nodes;  // the drafts
  return min(kKeys, s.len - tile * kKeys);
}
// ------------------------------------------------------------- add_listed ----

// Adds p v of the segment's listed keys (non-finite values, zeroed in the
// product) to columns [col, col + 32) of one row, times inv, in FP32: the row is
// rounded once, with everything in it. Rare: plain loops over global memory.
template <typename T, int D, bool TREE>
__device__ __noinline__ void add_listed(const Args &a, const Segment &s, const BadRows *bad, uint32_t position,
                                        uint32_t q_head, uint64_t set, float m, float inv, uint32_t col, float *o) {
  const T *q = static_cast<const T *>(a.t.q) + (s.q0 - s.pos0 + static_cast<size_t>(position)) * a.t.q_stride + q_head * D;
  const float c = a.t.scale * kLog2e;
  for (uint32_t at = 0; at < 4 * 64; ++at) {  // half, listed tile, key of the half
    const uint32_t half = at >> 7, i = at >> 6 & 1, j = at & 63;
    const uint32_t listed = *const_cast<const volatile uint32_t *>(&bad[half].tiles);
    __threadfence_block();
    if (i >= listed || !(bad[half].mask[i][j >> 5] >> (j & 31) & 1u)) continue;
    const uint32_t in_tile = half * 64 + j, tile = bad[half].tile[i], key = tile * kKeys + in_tile;
    const T *k, *v;
    if (!TREE || tile * kKeys >= s.len) {  // packed: a prompt's key, or a draft
      if (TREE ? !(set >> in_tile & 1u) : key > position) continue;
      const size_t at = (static_cast<size_t>(s.base) + (TREE ? in_tile : key)) * a.t.kv_stride + s.head * D;
      k = static_cast<const T *>(a.t.k) + at;
      v = static_cast<const T *>(a.t.v) + at;
    } else {
      const xpu_kv_cache_t &kc = a.tree.cache;
      const int32_t page = kc.tables[static_cast<size_t>(s.sequence) * kc.table_width + key / kc.page_size];
      if (page < 0 || static_cast<uint32_t>(page) >= kc.pages) continue;
      const size_t at = (((static_cast<size_t>(a.tree.layer) * kc.pages + page) * kc.kv_heads + s.head) * kc.page_size +
                         key % kc.page_size) * D;
      k = static_cast<const T *>(kc.k) + at;
      v = static_cast<const T *>(kc.v) + at;
    }
    float dot = 0.f;
    for (uint32_t d = 0; d < D; ++d) dot = fmaf(Elem<T>::to_float(q[d]), Elem<T>::to_float(k[d]), dot);
    const float p = exp2f(fmaf(dot, c, m == -INFINITY ? 0.f : fmaf(-m, c, Weights<T>::kLift))) * inv;
    for (uint32_t d = 0; d < 32; ++d) o[d] = fmaf(p, Elem<T>::to_float(v[col + d]), o[d]);
  }
}

// ------------------------------------------------------------------- join ----

// Partial results lie so that a warp's 32 rows (lanes) are next to each other:
// [slot][block of 32 rows][D / 4][32 rows][4 columns], so that both sides move
// whole lines; and their maxima and sums [slot][256 rows]{m, l}.
__device__ __forceinline__ float *partial_rows(const TreeArgs &a, uint32_t slot, uint32_t block, uint32_t d) {
  return a.partial + (static_cast<size_t>(slot) * 8 + block) * 32 * d;
}

// Rows of a unit from the partial results of blocks c0 .. c1, added in that
// order, by the 8 softmax warps. The loops are short on purpose: a block joins once or
// twice, and code that runs once costs about six cycles an instruction to fetch.
// Loads take 900 cycles, so each thread has sixteen of them in flight.
template <typename T, int D>
struct Join {
  const Args &a;
  const Segment &s;
  uint32_t group, positions, share, c0, c1;
  const float2 *sums;
  static constexpr uint32_t kTogether = 8;  // parts in flight

  __device__ uint32_t slot(uint32_t x) const { return 2 * x + (x * share >= s.unit ? 0 : 1); }
  __device__ float2 part_sums(uint32_t x, uint32_t row) const { return __ldcg(sums + slot(x) * 256 + row); }

  // Up to eight rows, all in the first block: lane = row + 8 piece, each thread four columns
  // of a row, so that the rows' pieces, which lie next to each other, are loaded together; the
  // maximum moves along.
  __device__ void few(uint32_t warp) const {
    const uint32_t lane = threadIdx.x & 31, r = lane & 7, piece = warp * 4 + (lane >> 3);
    if (piece >= D / 4) return;
    const float c = a.t.scale * kLog2e;
    float m = -INFINITY, l = 0.f, o[4] = {};
#pragma unroll 1
    for (uint32_t x0 = c0; x0 <= c1; x0 += kTogether) {
      float2 ml[kTogether];
      float4 v[kTogether];
#pragma unroll
      for (uint32_t e = 0; e < kTogether; ++e) {
        const uint32_t from = slot(min(x0 + e, c1));
        ml[e] = __ldcg(sums + from * 256 + r);
        v[e] = __ldcg(reinterpret_cast<const float4 *>(partial_rows(a.tree, from, 0, D)) + piece * 32 + r);
      }
      float top = m;
#pragma unroll
      for (uint32_t e = 0; e < kTogether; ++e) {
        if (x0 + e > c1) {  // behind the last part: nothing, also where its copy holds an infinity
          ml[e].x = -INFINITY;
          v[e] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        top = fmaxf(top, ml[e].x);
      }
      const float keep = m == -INFINITY ? 0.f : exp2_approx((m - top) * c);
      m = top;
      l *= keep;
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) o[k] *= keep;
#pragma unroll
      for (uint32_t e = 0; e < kTogether; ++e) {
        const float w = ml[e].x == -INFINITY ? 0.f : exp2_approx((ml[e].x - top) * c);
        l = fmaf(w, ml[e].y, l);
        o[0] = fmaf(w, v[e].x, o[0]), o[1] = fmaf(w, v[e].y, o[1]), o[2] = fmaf(w, v[e].z, o[2]), o[3] = fmaf(w, v[e].w, o[3]);
      }
    }
    if (r >= s.npos * group) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const uint32_t index = r / group, head = s.head * group + r - index * group;
    const size_t token = static_cast<size_t>(s.q0) + index;
    reinterpret_cast<uint2 *>(static_cast<T *>(a.t.out) + token * a.t.out_stride + head * D)[piece] =
        make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
    if (a.t.lse && piece == 0) a.t.lse[token * a.t.q_heads + head] = log_sum<T>(m, l, c);
  }

  // Any number: a block of 32 rows a warp, a row a lane, 64 columns at a time. With one row
  // tile, two warps a block, half of the columns each.
  __device__ void many(uint32_t warp) const {
    const bool halves = D == 128 && s.both;
    const uint32_t block = halves ? warp & 3 : warp, first = halves ? (warp >> 2) * 64 : 0, end = halves ? first + 64 : D;
    const uint32_t lane = threadIdx.x & 31, in_tile = (warp & 3) * 32 + lane, row = block * 32 + lane;
    const uint32_t in = in_tile / group, index = (block >> 2) * positions + in, head = s.head * group + in_tile - in * group;
    const bool mine = in < positions && index < s.npos;
    const size_t token = static_cast<size_t>(s.q0) + index;
    const QuadRows out(static_cast<T *>(a.t.out) + token * a.t.out_stride + head * D, mine);
    if (!out.any()) return;
    const float c = a.t.scale * kLog2e;
    float m = -INFINITY, l = 0.f;
#pragma unroll 1
    for (uint32_t x0 = c0; x0 <= c1; x0 += 4) {
      float2 ml[4];
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) ml[e] = part_sums(min(x0 + e, c1), row);
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        if (x0 + e > c1 || ml[e].x == -INFINITY) continue;
        const float top = fmaxf(m, ml[e].x);
        l = l * exp2_approx((m - top) * c) + ml[e].y * exp2_approx((ml[e].x - top) * c);
        m = top;
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
    for (uint32_t q = first; q < end; q += 64) {
      float o[64] = {};
#pragma unroll 1
      for (uint32_t x = c0; x <= c1; ++x) {
        const float4 *src = reinterpret_cast<const float4 *>(partial_rows(a.tree, slot(x), block, D)) + q / 4 * 32 + lane;
        float4 v[16];
#pragma unroll
        for (uint32_t k = 0; k < 16; ++k) v[k] = __ldcg(src + 32 * k);
        const float mx = part_sums(x, row).x, w = mx == -INFINITY ? 0.f : exp2_approx((mx - m) * c) * inv;
#pragma unroll
        for (uint32_t k = 0; k < 16; ++k) {
          o[4 * k] = fmaf(w, v[k].x, o[4 * k]), o[4 * k + 1] = fmaf(w, v[k].y, o[4 * k + 1]);
          o[4 * k + 2] = fmaf(w, v[k].z, o[4 * k + 2]), o[4 * k + 3] = fmaf(w, v[k].w, o[4 * k + 3]);
        }
      }
      uint32_t p[32];
#pragma unroll
      for (uint32_t k = 0; k < 32; ++k) p[k] = pack2<T>(o[2 * k], o[2 * k + 1]);
      out.put(p, q * 2);
      out.put(p + 16, q * 2 + 64);
    }
    if (a.t.lse && mine && first == 0) a.t.lse[token * a.t.q_heads + head] = log_sum<T>(m, l, c);
  }
};

// ----------------------------------------------------------------- kernel ----

template <typename T, int D, bool TREE>
__global__ void __launch_bounds__(kThreads, 1) k_attention(const __grid_constant__ Args a) {
  using S = Shape<D, TREE>;
  using Walk = typename std::conditional<TREE, TreeWalk, PromptWalk>::type;
  constexpr bool kFp16 = std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ Barriers b;
  __shared__ TreeEntry table[TREE ? XPU_KV_MAX_REQUESTS + 1 : 1];
  __shared__ float joined[TREE ? 2 : 1][TREE ? 128 : 1][2];
  __shared__ uint2 scratch[kThreads / 32];
  __shared__ bool last;
  const uint32_t a0 = smem_addr(smem_raw);
  uint8_t *q_smem = smem_raw + ((a0 + 1023u) / 1024u * 1024u - a0), *ring = q_smem + 2 * S::kTile;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t group = a.t.q_heads / a.t.kv_heads, positions = tile_positions(group);

  if (threadIdx.x >= 32 && threadIdx.x < (TREE ? 37 : 35)) {
    const CUtensorMap *map = threadIdx.x == 32 ? &a.q : threadIdx.x == 33 ? &a.k : threadIdx.x == 34 ? &a.v
                             : threadIdx.x == 35 ? &a.cached_k : &a.cached_v;
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  }
  if (threadIdx.x == 0) {
    mbar_init(&b.q_full, 1);
    mbar_init(&b.q_empty, 1);
    mbar_init(&b.drain, 1);
    for (uint32_t i = 0; i < S::kStages; ++i) {
      mbar_init(&b.kv_full[i], 1);
      mbar_init(&b.kv_empty[i], TREE ? 2 : 3);  // the products and the cleaning warps
      mbar_init(&b.clean[i], TREE ? 1 : 2);
    }
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(&b.s_full[i], 1);
      mbar_init(&b.p_early[i], 4);
      mbar_init(&b.p_ready[i], 4);
      mbar_init(&b.o_full[i], 1);
    }
    mbar_init(&b.joined, 8);
    fence_mbar_init();
    for (uint32_t i = 0; i < 8; ++i) b.ended[i] = 0;
    b.failed = 0;
  }
  if (warp == kMmaWarp) {
    tmem_alloc1(&b.tmem, 512);
    // The next kernel's blocks may come from here on, not earlier: one that takes TMEM before
    // this block has its own would wait for this grid's end, and this block for that TMEM.
    grid_dep_launch();
  }
  grid_dep_wait();  // up to here nothing was read but the arguments
  if constexpr (TREE)
    tree_table(a.tree, a.t.tokens, a.t.kv_heads, group, table, scratch, TreeRequest(a.tree, threadIdx.x));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = b.tmem;
  auto walk = [&] {
    if constexpr (TREE) return Walk(a, table, group);
    else return Walk(a, group);
  }();
  Segment s;

  // the launch's 384 x 168 registers: 256 x 208 + 128 x 88
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------------------ softmax ----
    const uint32_t t = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (warp & 3) * 32u << 16;
    const uint32_t s_addr = tmem + lanes + t * 128, o_addr = tmem + lanes + 256;  // O_t at + 128 t
    const float c = a.t.scale * kLog2e;
    const uint32_t in_tile = r / group, q_head_in_group = r % group;
    uint32_t uses = 0, done = 0, segment = 0, joins = 0;
    // every softmax warp, bounded like every wait
    auto meet = [&] {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b.joined);
      const bool ok = warp_wait(b, &b.joined, joins++ & 1);
      tc_fence_after();
      return ok;
    };
    for (; walk.next(s) && !warp_failed(b); ++segment) {
      const uint32_t index = (s.both ? 0 : t * positions) + in_tile;  // position inside the segment
      const bool mine = r < positions * group && index < s.npos;
      const uint32_t position = s.pos0 + min(index, s.npos - 1);
      const uint64_t set = TREE ? a.tree.ancestors[s.base + position] : 0;
      const uint32_t tiles = t ? s.n1 : s.n0;
      float m = -INFINITY, l = 0.f;
      for (uint32_t i = 0; i < tiles; ++i, ++uses) {
        const uint32_t tile = s.first + (s.both ? 2 * i + t : i);
        if (!warp_wait(b, &b.s_full[t], uses & 1)) break;
        tc_fence_after();
        const bool masked = tile >= s.masked_from;
        uint32_t x[kKeys];
        tmem_ld32(s_addr, x);
        tmem_ld32(s_addr + 32, x + 32);
        tmem_wait_ld64(x);
        tmem_ld32(s_addr + 64, x + 64);
        tmem_ld32(s_addr + 96, x + 96);
        uint32_t attended[4];  // this row's keys of the tile, a bit each
        if (masked) {
          if (TREE && tile * kKeys >= s.len) {  // the drafts
            const uint64_t own = set & (s.nodes >= 64 ? ~0ull : (1ull << s.nodes) - 1);
            attended[0] = static_cast<uint32_t>(own), attended[1] = static_cast<uint32_t>(own >> 32);
            attended[2] = attended[3] = 0;
          } else {
            const uint32_t end = TREE ? s.len : position + 1, many = end - min(tile * kKeys, end);
#pragma unroll
            for (uint32_t w = 0; w < 4; ++w)
              attended[w] = many >= 32 * (w + 1) ? 0xffffffffu : many > 32 * w ? (1u << (many - 32 * w)) - 1u : 0u;
          }
        }
        auto mask = [&](uint32_t from) {
#pragma unroll
          for (uint32_t j = from; j < from + 64; ++j)
            if (!(attended[j >> 5] & 1u << (j & 31))) x[j] = 0xff800000u;
        };
        if (masked) mask(0);
        // p of 32 keys from x[32 q] on, in pairs, and their sum
        const Pair c2(c, c);
        Pair sum0(0.f, 0.f), sum1(0.f, 0.f);
        auto quarter = [&](uint32_t q, Pair mc2, uint32_t *p) {
#pragma unroll
          for (uint32_t j = 0; j < 16; ++j) {
            const Pair y = fma2(Pair(__uint_as_float(x[32 * q + 2 * j]), __uint_as_float(x[32 * q + 2 * j + 1])), c2, mc2);
            float lo, hi;
            y.get(lo, hi);
            lo = exp2_approx(lo);
            hi = exp2_approx(hi);
            if (j & 1) sum1 = add2(sum1, Pair(lo, hi));
            else sum0 = add2(sum0, Pair(lo, hi));
            p[j] = pack2<T>(lo, hi);
          }
        };
        auto publish = [&](uint64_t *bar) {
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar);
        };
        // a row with an infinite or undefined score is undefined as a whole
        auto shift = [&] {
          const float mc = m == -INFINITY ? 0.f : (m == INFINITY ? NAN : fmaf(-m, c, Weights<T>::kLift));
          return Pair(mc, mc);
        };
        float top4[4] = {m, m, m, m};  // four chains; NaN if one score is
        auto search = [&](uint32_t from) {
#pragma unroll
          for (uint32_t j = from; j < from + 64; j += 8)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
              top4[e] = max3_nan(top4[e], __uint_as_float(x[j + 2 * e]), __uint_as_float(x[j + 2 * e + 1]));
        };
        search(0);
        tmem_wait_ld64(x + 64);
        if (masked) mask(64);
        search(64);
        const float top = max3_nan(max3_nan(top4[0], top4[1], top4[2]), top4[3], top4[3]);
        // m = -inf included, and NaN; not the rows behind the last whole position (126 and 127 of a group of 7),
        // whose queries no load writes: stale NaN would rescale for every key tile
        const bool grown = mine && top != m && !((top - m) * c <= Weights<T>::kRescale);
        if (__any_sync(kFullMask, grown)) {
          // the others of the warp go along, so that they need none of their own soon
          const float keep = top != m ? exp2_approx((m - top) * c) : 1.f;
          m = top;
          l *= keep;
          if (i > 0) {
#pragma unroll 1
            for (uint32_t q = 0; q < D / 32; ++q) {
              uint32_t o[32];
              tmem_ld32(o_addr + t * 128 + 32 * q, o);
              tmem_wait_ld();
#pragma unroll
              for (uint32_t j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
              tmem_st32(o_addr + t * 128 + 32 * q, o);
            }
          }
        }
        const Pair mc2 = shift();
#pragma unroll
        for (uint32_t q = 0; q < kKeys / 32; ++q) {
          uint32_t p[16];
          quarter(q, mc2, p);
          tmem_st16(s_addr + 16 * q, p);
          if (32 * (q + 1) == kEarlyKeys) publish(&b.p_early[t]);
        }
        float sum[4];
        sum0.get(sum[0], sum[1]);
        sum1.get(sum[2], sum[3]);
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        publish(&b.p_ready[t]);
      }
      if (warp_failed(b)) break;
      if (tiles) {
        if (!warp_wait(b, &b.o_full[t], done & 1)) break;
        ++done;
        tc_fence_after();
      }
      // ---------------------------------------------------- join and write ----
      [[maybe_unused]] float weight[2] = {1.f, 1.f};
      uint32_t col = 0, cols = D;
      if (TREE && s.both) {
        joined[t][r][0] = m;
        joined[t][r][1] = l;
        if (!meet()) break;
        const float m0 = joined[0][r][0], m1 = joined[1][r][0];
        m = fmaxf(m0, m1);
        weight[0] = m0 == -INFINITY ? 0.f : exp2_approx((m0 - m) * c);
        weight[1] = m1 == -INFINITY ? 0.f : exp2_approx((m1 - m) * c);
        l = weight[0] * joined[0][r][1] + weight[1] * joined[1][r][1];
        col = t * (D / 2);
        cols = D / 2;
      }
      if (tiles || s.both) {
        const bool whole = s.slot < 0;
        const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        const size_t token = s.q0 - s.pos0 + static_cast<size_t>(position);
        const uint32_t q_head = s.head * group + q_head_in_group;
        T *dst16 = static_cast<T *>(a.t.out) + token * a.t.out_stride + q_head * D;
        float *dst32 = nullptr;
        if (TREE && !whole) {
          const uint32_t row = (s.both ? 0 : t * 128) + r;
          dst32 = partial_rows(a.tree, s.slot, row >> 5, D) + (row & 31) * 4;
          if (mine && col == 0)
            reinterpret_cast<float2 *>(a.tree.partial + 2ull * gridDim.x * 256 * D)[s.slot * 256 + row] = make_float2(m, l);
        } else if (mine && a.t.lse && col == 0 && token < a.t.tokens) {
          a.t.lse[token * a.t.q_heads + q_head] = log_sum<T>(m, l, c);
        }
        const bool store = mine && token < a.t.tokens;
        const BadRows *bad = b.bad[segment % kBadRing];
        const bool listed = store && s.first + s.n > s.masked_from &&
                            (*const_cast<const volatile uint32_t *>(&bad[0].tiles) |
                             *const_cast<const volatile uint32_t *>(&bad[1].tiles)) != 0;
        const QuadRows out(dst16, store);
        if (out.any()) {
#pragma unroll 1
          for (uint32_t q = col; q < col + cols; q += 32) {
            uint32_t o[32];
            tmem_ld32(o_addr + (TREE && s.both ? 0 : t * 128) + q, o);
            tmem_wait_ld();
            const float w0 = TREE && s.both ? weight[0] * inv : inv;
#pragma unroll
            for (uint32_t j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * w0);
            if (TREE && s.both && s.n1) {
              uint32_t o1[32];
              tmem_ld32(o_addr + 128 + q, o1);
              tmem_wait_ld();
              const float w1 = weight[1] * inv;
#pragma unroll
              for (uint32_t j = 0; j < 32; ++j)
                o[j] = __float_as_uint(fmaf(__uint_as_float(o1[j]), w1, __uint_as_float(o[j])));
            }
            if (listed) {
              float f[32];
#pragma unroll
              for (uint32_t j = 0; j < 32; ++j) f[j] = __uint_as_float(o[j]);
              add_listed<T, D, TREE>(a, s, bad, position, q_head, set, m, inv, q, f);
#pragma unroll
              for (uint32_t j = 0; j < 32; ++j) o[j] = __float_as_uint(f[j]);
            }
            __syncwarp();
            if (TREE && dst32) {
              if (store) {
#pragma unroll
                for (uint32_t j = 0; j < 32; j += 4)
                  *reinterpret_cast<uint4 *>(dst32 + (q + j) * 32) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
              }
            } else {
#pragma unroll
              for (uint32_t j = 0; j < 16; ++j) o[j] = pack2<T>(__uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1]));
              out.put(o, q * 2);
            }
          }
        }
      }
      if constexpr (TREE) {
        if (s.slot >= 0) {
          // The block that completes a unit adds up its parts, in the order of the
          // key tiles whoever comes last.
          if (!meet()) break;
          const uint32_t share = walk.cut.share, c0 = (s.unit + walk.cut.lead) / share, c1 = (s.unit + s.unit_size - 1) / share;
          if (threadIdx.x == 0) {
            uint32_t before;  // releases this block's part, acquires the others'
            asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                         : "=r"(before)
                         : "l"(a.tree.arrived + c0)
                         : "memory");
            last = before == c1 - c0;
            if (last) a.tree.arrived[c0] = 0;
          }
          if (!meet()) break;
          if (last) {
            const float2 *sums = reinterpret_cast<const float2 *>(a.tree.partial + 2ull * gridDim.x * 256 * D);
            const Join<T, D> join{a, s, group, positions, share, c0, c1, sums};
            if (s.npos * group <= 8) join.few(warp);
            else join.many(warp);
          }
          if (!meet()) break;
        } else if (s.both && !meet()) {  // the other group may still read this one's accumulator and sums
          break;
        }
      }
      // A group without a row tile in the segments that follow runs far behind the other one if it has
      // listed values to add.
      __syncwarp();
      if (lane == 0) {
        __threadfence_block();
        *const_cast<volatile uint32_t *>(&b.ended[warp]) = segment + 1;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  }
  if (warp < 8) {
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------------- MMA ----
    // The whole warp walks along, with every value the same in all lanes, and
    // one lane issues: operands then stay in uniform registers. With a single
    // lane in the loop each instruction took 72 to 90 cycles to issue where the
    // tensor cores need 64. Their queue covers about four instructions.
    constexpr uint32_t qk_desc = attn_idesc(kFp16, kKeys, true), pv_desc = attn_idesc(kFp16, D, false);
    const uint32_t tm = same(tmem), smem0 = same(smem_addr(q_smem));
    const uint64_t q_desc = smem_desc(smem0, 16, 1024);
    const uint64_t k_desc = smem_desc(smem0 + 2 * S::kTile, 16, 1024), v_desc = smem_desc(smem0 + 2 * S::kTile, kBox, 1024);
    uint32_t slot = 0, phase = 0;  // the ring's next entry: K 0, V 0, K 1, V 1, ...
    uint32_t cleaned = 0, p_uses = 0, segment = 0;  // phases: a bit per ring entry, per row tile
    const bool leader = elect_one();
    bool ok = true;
    auto advance = [&](uint32_t &at, uint32_t &ph) {
      if (++at == S::kStages) at = 0, ph ^= 1;
    };
    auto commit = [&](uint64_t *bar) {
      if (leader) mma1_commit(bar);
    };
    auto clean = [&](uint32_t tile, uint32_t at) {
      if (tile < s.masked_from) return true;
      const bool done = warp_wait(b, &b.clean[at], cleaned >> at & 1);
      cleaned ^= 1u << at;
      return done;
    };
    for (; ok && walk.next(s); ++segment) {
      s.n = same(s.n), s.n0 = same(s.n0), s.n1 = same(s.n1), s.first = same(s.first);
      s.masked_from = same(s.masked_from);
      if (TREE) s.both = same(s.both);
      if (!(ok = warp_wait(b, &b.q_full, segment & 1))) break;
      // Turn j: O_t += P_t V_j, then S_t of the key tile that t comes to next, for t =
      // 0 and 1; with both groups on row tile 0, t = j & 1 alone. One place for each
      // product keeps the code short.
      const bool both = TREE && s.both;
      const uint32_t ahead = both ? 2 : 1;
      uint32_t v = slot, v_phase = phase, k = slot, k_phase = phase;  // next V and next K
      advance(v, v_phase);
      uint32_t seen = 0;  // K tiles known to be there
      for (int32_t j = -static_cast<int32_t>(ahead); ok && j < static_cast<int32_t>(s.n); ++j) {
        const uint32_t next = static_cast<uint32_t>(j) + ahead;  // key tile of this turn's S
        if (j >= 0 && !(ok = warp_wait(b, &b.kv_full[v], v_phase) && clean(s.first + j, v))) break;
        const uint64_t dv = v_desc + (v * S::kTile >> 4), dk = k_desc + (k * S::kTile >> 4);
#pragma unroll(TREE ? 1 : 2)
        for (uint32_t t = both ? j & 1 : 0; t < (both ? (j & 1) + 1u : 2u); ++t) {
          const uint32_t tiles = both ? s.n : t ? s.n1 : s.n0, s_tmem = tm + t * 128, o_tmem = s_tmem + 256;
          if (j >= 0 && static_cast<uint32_t>(j) < tiles) {
            const uint32_t accumulate = j >= static_cast<int32_t>(ahead), uses = p_uses >> t & 1;
            if (!(ok = warp_wait(b, &b.p_early[t], uses))) break;
            tc_fence_after();
            if (leader) {
#pragma unroll
              for (uint32_t kk = 0; kk < kEarlyKeys / 16; ++kk)
                mma1_ts(o_tmem, s_tmem + kk * 8, dv + (kk * 2048u >> 4), pv_desc, kk ? 1 : accumulate);
            }
            if (!(ok = warp_wait(b, &b.p_ready[t], uses))) break;
            tc_fence_after();
            if (leader) {
#pragma unroll
              for (uint32_t kk = kEarlyKeys / 16; kk < kKeys / 16; ++kk)
                mma1_ts(o_tmem, s_tmem + kk * 8, dv + (kk * 2048u >> 4), pv_desc, 1);
            }
            p_uses ^= 1u << t;
            if (next >= tiles) commit(&b.o_full[t]);
            // the ring entry is free before the wait for the next one
            if (both || t == (static_cast<uint32_t>(j) < s.n1 ? 1 : 0)) commit(&b.kv_empty[v]);
          }
          if (next < tiles) {
            if (seen <= next) {
              if (!(ok = warp_wait(b, &b.kv_full[k], k_phase))) break;
              tc_fence_after();
              seen = next + 1;
            }
            const uint64_t dq = q_desc + (both ? 0 : t * (S::kTile >> 4));
            if (leader) {
#pragma unroll
              for (uint32_t kk = 0; kk < D / 16; ++kk) {
                const uint32_t off = (kk / 4 * kBox + kk % 4 * 32) >> 4;
                mma1_f16(s_tmem, dq + off, dk + off, qk_desc, kk != 0);
              }
              mma1_commit(&b.s_full[t]);
            }
          }
        }
        if (!ok) break;
        if (j >= 0) {
          slot = v, phase = v_phase;
          advance(v, v_phase);
          advance(v, v_phase);
        }
        if (next < s.n) {
          commit(&b.kv_empty[k]);
          if (next + 1 == s.n) commit(&b.q_empty);
          advance(k, k_phase);
          advance(k, k_phase);
        }
      }
      advance(slot, phase);
      ok = ok && !warp_failed(b);
    }
    if (!ok) {  // nothing issued may still run when TMEM is freed
      b.failed = 1;
      commit(&b.drain);
      warp_wait(b, &b.drain, 0);
    }
  } else if (warp == kLoadWarp || (TREE && warp == kLoadWarp + 1)) {
    // --------------------------------------------------------------- loads ----
    // A tree's key tile is up to 16 copies of a page, too many for one warp to issue
    // in the time that they take: one warp loads K, another V. The ring then has an even
    // number of entries, so that each warp sees every turn of its own.
    static_assert(!TREE || S::kStages % 2 == 0, "K and V keep to their entries");
    static_assert(S::kStages >= 4, "the products hold up to three entries");
    const uint32_t first_which = TREE ? warp - kLoadWarp : 0, last_which = TREE ? first_which : 1;
    const bool leader = elect_one();
    uint32_t loaded = first_which, segment = 0, q_loads = 0;
    // lane p: the id of page p of a cached key tile (behind the pool, where reads
    // give zeros, if it is out of range)
    auto page_of = [&](const Segment &g, uint32_t tile) {
      int32_t page = 0;
      if constexpr (TREE) {
        const xpu_kv_cache_t &kc = a.tree.cache;
        const uint32_t at = tile * kKeys + (lane << a.tree.page_shift);
        if (lane << a.tree.page_shift < kKeys && at < g.len) {
          page = kc.tables[static_cast<size_t>(g.sequence) * kc.table_width + (at >> a.tree.page_shift)];
          if (page < 0 || static_cast<uint32_t>(page) >= kc.pages) {
            atomicOr(kc.status, XPU_KV_BAD_INDEX);
            page = static_cast<int32_t>(kc.pages);
          }
        }
      }
      return page;
    };
    auto load_q = [&](const Segment &g) {
      if (leader) {
        const uint32_t tiles = !g.both && g.npos > positions ? 2 : 1;
        mbar_expect_tx(&b.q_full, tiles * positions * group * 128 * S::kBoxes);
        for (uint32_t t = 0; t < tiles; ++t)
          for (uint32_t h = 0; h < S::kBoxes; ++h)
            tma_load_3d(q_smem + t * S::kTile + h * kBox, &a.q, 64 * h, g.head * group, g.q0 + t * positions, &b.q_full);
      }
      ++q_loads;
    };
    Segment following;
    bool more = walk.next(following);
    if (more && first_which == 0) load_q(following);
    int32_t next_page = more ? page_of(following, following.first) : 0;
    bool ok = true;
    for (; ok && more && !warp_failed(b); ++segment) {
      s = following;
      for (uint32_t j = 0; j < s.n && ok; ++j) {
        const uint32_t tile = s.first + j, at = tile * kKeys;
        const bool packed = !TREE || at >= s.len;
        // the next tile's pages are looked up under this tile's wait
        const int32_t page = next_page;
        if (j + 1 < s.n) {
          next_page = page_of(s, tile + 1);
        } else {
          more = walk.next(following);
          if (more) next_page = page_of(following, following.first);
        }
#pragma unroll 1
        for (uint32_t which = first_which; which <= last_which; ++which) {
          const uint32_t slot = loaded % S::kStages, use = loaded / S::kStages;
          if (use > 0 && !(ok = warp_wait(b, &b.kv_empty[slot], (use - 1) & 1))) break;
          uint64_t *bar = &b.kv_full[slot];
          uint8_t *dst = ring + slot * S::kTile;
          loaded += TREE ? 2 : 1;
          if (packed) {
            if (leader) {
              // a tree's drafts: half a tile, XPU_TREE_MAX_NODES rows
              mbar_expect_tx(bar, TREE ? S::kTile / 2 : S::kTile);
              for (uint32_t h = 0; h < S::kBoxes; ++h)
                tma_load_3d(dst + h * kBox, which ? &a.v : &a.k, 64 * h, s.head, s.base + (TREE ? 0 : at), bar);
            }
          } else {
            const xpu_kv_cache_t &kc = a.tree.cache;
            const uint32_t bytes = kc.page_size * 128, pages = (min(kKeys, s.len - at) + kc.page_size - 1) >> a.tree.page_shift;
            const uint32_t row = (static_cast<uint32_t>(page) * kc.kv_heads + s.head) * kc.page_size;
            if (leader) mbar_expect_tx(bar, pages * bytes * S::kBoxes);
#pragma unroll 1
            for (uint32_t p = 0; p < pages; ++p) {
              const int32_t y = static_cast<int32_t>(__shfl_sync(kFullMask, row, p));
              if (leader) {
#pragma unroll
                for (uint32_t h = 0; h < S::kBoxes; ++h)
                  tma_load_2d_plain(dst + h * kBox + p * bytes, which ? &a.cached_v : &a.cached_k, 64 * h, y, bar);
              }
            }
          }
          // a later segment's rows after its first keys, which need not wait for the rows before them
          if (j == 0 && which == 0 && segment > 0) {
            if (!(ok = warp_wait(b, &b.q_empty, (segment - 1) & 1))) break;
            load_q(s);
          }
        }
      }
    }
    if (warp_failed(b)) {  // what was asked for lands before the block's memory is given up
      for (uint32_t i = loaded > S::kStages ? loaded - S::kStages : first_which; i < loaded; i += TREE ? 2 : 1)
        mbar_wait(&b.kv_full[i % S::kStages], i / S::kStages & 1);
      if (q_loads) mbar_wait(&b.q_full, (q_loads - 1) & 1);
    }
  } else {
    // ------------------------------------------------------------ cleaning ----
    // keys 64 half .. of a tile: a warp each half, or (trees) one warp both
    const uint32_t half0 = TREE ? 0 : warp - kCleanWarp;
    uint32_t loaded = 0, segment = 0;
    for (; walk.next(s) && !warp_failed(b); ++segment) {
      BadRows *bad = &b.bad[segment % kBadRing][half0];
      uint32_t listed[2] = {0, 0};
      if (s.first + s.n > s.masked_from && !wait_listed(b, segment)) break;
      if (lane < (TREE ? 2 : 1) && s.first + s.n > s.masked_from) bad[lane].tiles = 0;
      __syncwarp();
      for (uint32_t e = 0; e < 2 * s.n; ++e) {  // every ring entry, so as never to be a turn ahead or behind
        const uint32_t i = loaded + e, slot = i % S::kStages, tile = s.first + e / 2;
        if (!warp_wait(b, &b.kv_full[slot], i / S::kStages & 1)) break;
        if (e % 2 == 0 || tile < s.masked_from) {
          if (lane == 0) mbar_arrive(&b.kv_empty[slot]);
          continue;
        }
        const uint32_t valid = valid_keys<TREE>(s, tile);
#pragma unroll
        for (uint32_t h = 0; h < (TREE ? 2 : 1); ++h) {
          uint32_t any = 0;
#pragma unroll 1
          for (uint32_t g = 0; g < 2; ++g) {
            const uint32_t key = (half0 + h) * 64 + g * 32 + lane;
            uint8_t *row = ring + slot * S::kTile + key * 128;
            const bool inside = key < valid;
            uint32_t sums[4] = {0, 0, 0, 0};
            if (inside) {
#pragma unroll
              for (uint32_t x = 0; x < 8 * S::kBoxes; ++x) {  // 16-byte pieces, each lane from another bank
                const uint4 w = *reinterpret_cast<const uint4 *>(row + x / 8 * kBox + ((x + lane) & 7) * 16);
                sums[0] = add_zero_times<T>(w.x, sums[0]);
                sums[1] = add_zero_times<T>(w.y, sums[1]);
                sums[2] = add_zero_times<T>(w.z, sums[2]);
                sums[3] = add_zero_times<T>(w.w, sums[3]);
              }
            }
            const bool spoilt = ((sums[0] | sums[1] | sums[2] | sums[3]) & 0x7fff7fffu) != 0;
            if (!inside || spoilt) {
#pragma unroll
              for (uint32_t x = 0; x < 8 * S::kBoxes; ++x)
                *reinterpret_cast<uint4 *>(row + x / 8 * kBox + ((x + lane) & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            const uint32_t found = __ballot_sync(kFullMask, spoilt);
            any |= found;
            if (lane == 0 && listed[h] < 2) bad[h].mask[listed[h]][g] = found;
          }
          if (any && listed[h] < 2) {
            if (lane == 0) {
              bad[h].tile[listed[h]] = tile;
              __threadfence_block();
              *const_cast<volatile uint32_t *>(&bad[h].tiles) = listed[h] + 1;
            }
            ++listed[h];
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&b.clean[slot]);
          mbar_arrive(&b.kv_empty[slot]);
        }
      }
      loaded += 2 * s.n;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && b.failed) atomicOr(&g_attention_error, kErrAttentionTimeout);
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc1(tmem, 512);
  }
}

// ------------------------------------------------------------------- host ----

cudaError_t packed_map(CUtensorMap *map, const void *base, const AttnTensors &t, uint32_t heads, uint64_t stride,
                       uint32_t box_heads, uint32_t box_rows) {
  return make_tmap_3d_u16_box(map, base, t.head_dim, heads, t.tokens, t.head_dim, stride, 64, box_heads, box_rows);
}

cudaError_t packed_maps(Args &a, uint32_t kv_rows) {
  const AttnTensors &t = a.t;
  const uint32_t group = t.q_heads / t.kv_heads;
  cudaError_t e = packed_map(&a.q, t.q, t, t.q_heads, t.q_stride, group, tile_positions(group));
  if (e == cudaSuccess) e = packed_map(&a.k, t.k, t, t.kv_heads, t.kv_stride, 1, kv_rows);
  if (e == cudaSuccess) e = packed_map(&a.v, t.v, t, t.kv_heads, t.kv_stride, 1, kv_rows);
  return e;
}

template <typename T, int D, bool TREE>
cudaError_t launch(const Args &a, uint32_t blocks, cudaStream_t s) {
  constexpr uint32_t smem = Shape<D, TREE>::kSmem;
  static std::atomic<bool> allowed[64];  // the shared memory, once per device
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device > 63 || !allowed[device].load(std::memory_order_relaxed)) {
    e = cudaFuncSetAttribute(k_attention<T, D, TREE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (device < 64) allowed[device].store(true, std::memory_order_relaxed);
  }
  return launch_after(k_attention<T, D, TREE>, blocks, kThreads, smem, s, a);
}

template <bool TREE>
cudaError_t launch_any(bool fp16, const Args &a, uint32_t blocks, cudaStream_t s) {
  if (a.t.head_dim == 128)
    return fp16 ? launch<__half, 128, TREE>(a, blocks, s) : launch<__nv_bfloat16, 128, TREE>(a, blocks, s);
  return fp16 ? launch<__half, 64, TREE>(a, blocks, s) : launch<__nv_bfloat16, 64, TREE>(a, blocks, s);
}

}  // namespace

uint32_t sm_count() {
  static std::atomic<int> known[64];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) {
    cudaGetLastError();
    return 148;
  }
  int sms = known[device & 63].load(std::memory_order_relaxed);
  if (sms == 0) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
      cudaGetLastError();
      return 148;
    }
    known[device & 63].store(sms, std::memory_order_relaxed);
  }
  return static_cast<uint32_t>(sms);
}

unsigned take_attention_error() {
  unsigned v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_attention_error, sizeof(v)) != cudaSuccess) return 0;
  if (v) cudaMemcpyToSymbol(g_attention_error, &zero, sizeof(zero));
  return v;
}

size_t prompt_plan(const uint32_t *lens, uint32_t count, uint32_t q_heads, uint32_t kv_heads, uint32_t sms, int32_t *plan,
                   size_t capacity) {
  const uint32_t group = q_heads / kv_heads, span = 2 * tile_positions(group);
  struct Item {
    int32_t token, len, pos, head;
    uint32_t cost;
  };
  std::vector<Item> items;
  uint64_t tokens = 0;
  for (uint32_t i = 0; i < count; ++i) {
    for (uint32_t pos = 0; pos < lens[i]; pos += span)
      for (uint32_t h = 0; h < kv_heads; ++h)
        items.push_back({static_cast<int32_t>(tokens), static_cast<int32_t>(lens[i]), static_cast<int32_t>(pos),
                         static_cast<int32_t>(h), (std::min(pos + span, lens[i]) + 127) / 128 + 2});
    tokens += lens[i];
  }
  const uint32_t blocks = static_cast<uint32_t>(std::min<size_t>(items.size(), sms));
  const size_t used = plan_items_at(blocks) + 4 * items.size();
  if (used > capacity) return used;
  // longest first, each to the block with the least work
  std::stable_sort(items.begin(), items.end(), [](const Item &a, const Item &b) { return a.cost > b.cost; });
  std::vector<std::vector<const Item *>> per(blocks);
  using Load = std::pair<uint64_t, uint32_t>;
  std::priority_queue<Load, std::vector<Load>, std::greater<Load>> loads;
  for (uint32_t b = 0; b < blocks; ++b) loads.push({0, b});
  for (const Item &it : items) {
    const Load least = loads.top();
    loads.pop();
    per[least.second].push_back(&it);
    loads.push({least.first + it.cost, least.second});
  }
  plan[0] = static_cast<int32_t>(blocks);
  plan[1] = static_cast<int32_t>(tokens);
  plan[2] = static_cast<int32_t>(items.size());
  plan[3] = static_cast<int32_t>(group);
  std::fill(plan + kPlanHeader, plan + plan_items_at(blocks), 0);
  int32_t at = 0, *out = plan + plan_items_at(blocks);
  for (uint32_t b = 0; b < blocks; ++b) {
    plan[kPlanHeader + b] = at;
    for (const Item *it : per[b]) {
      const int32_t v[4] = {it->token, it->len, it->pos, it->head};
      std::copy(v, v + 4, out + 4 * at++);
    }
  }
  plan[kPlanHeader + blocks] = at;
  return used;
}

cudaError_t prompt_attention_launch(bool fp16, const int32_t *plan, uint32_t blocks, const AttnTensors &t,
                                    cudaStream_t s) {
  Args a = {};
  a.t = t;
  a.plan = plan;
  const cudaError_t e = packed_maps(a, kKeys);
  return e != cudaSuccess ? e : launch_any<false>(fp16, a, blocks, s);
}

namespace {
constexpr uint32_t kArrivedBytes = 4096;  // up to 1024 blocks
}

size_t tree_workspace_bytes(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t head_dim) {
  // arrivals, and two partial results a block: 256 rows of outputs, and their maxima and sums
  return kArrivedBytes + 2ull * sm_count() * 256 * (head_dim + 2) * 4;
}

cudaError_t tree_attention_launch(const xpu_kv_cache_t &c, uint32_t layer, const int32_t *sequences,
                                  const int32_t *starts, const uint64_t *ancestors, uint32_t count,
                                  const AttnTensors &t, void *workspace, cudaStream_t s) {
  Args a = {};
  a.t = t;
  a.tree = {c, sequences, starts, ancestors, layer, count, static_cast<uint32_t>(__builtin_ctz(c.page_size)),
            static_cast<uint32_t *>(workspace),
            reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + kArrivedBytes)};
  cudaError_t e = packed_maps(a, XPU_TREE_MAX_NODES);
  if (e != cudaSuccess) return e;
  const uint64_t rows = static_cast<uint64_t>(c.pages) * c.kv_heads * c.page_size;
  const size_t offset = static_cast<size_t>(layer) * rows * c.head_dim;
  e = make_tmap_2d_u16_swizzled(&a.cached_k, static_cast<const uint16_t *>(c.k) + offset, c.head_dim, rows, c.head_dim, 64,
                                c.page_size);
  if (e != cudaSuccess) return e;
  e = make_tmap_2d_u16_swizzled(&a.cached_v, static_cast<const uint16_t *>(c.v) + offset, c.head_dim, rows, c.head_dim, 64,
                                c.page_size);
  if (e != cudaSuccess) return e;
  return launch_any<true>(c.dtype == XPU_FP16, a, sm_count(), s);
}

}  // namespace xpu
