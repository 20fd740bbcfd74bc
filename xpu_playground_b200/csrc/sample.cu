// Choosing a token from a row of 16-bit logits (xpu_sample in include/xpu_cuda.h).
//
// The order is that of falling logits, of equal ones the lowest id first; what top-k,
// top-p and min-p keep is a beginning of it, and the token is the first whose sum of
// weights exceeds u times that of the beginning. Nothing is sorted: a row has at most
// 65536 different values, so a histogram of them, in shared memory with 16-bit counters,
// says all about it. A weight exp((l - l_max) / T) is computed once a value, in 64 bits, as
// are the sums: where u falls between 151936 sums must not hang on rounding. Prefix
// sums over groups of 32 values, then over the values of one group, answer each
// question ("the last value whose prefix is below x"); the answer is a value
// and which of its occurrences it is, and a second look at the row finds its place.
// Sums are in a fixed order: results repeat bit for bit.
//
// Rows with a small top-k (a temperature of 0 is top-k 1) need no histogram: each thread's largest
// logit is found first, and no logit below the k-th of those can be among the k. What is left, a few times
// k, is listed and put in order by one block, a token a thread.
//
// SIZE blocks of a cluster share a row, a run of it each: as many as are resident at once for all rows. Four and eight
// blocks hold their runs in registers, one and two read theirs again from the L2.
//
// Rows of 151936 bf16 logits, us without top-k / top-k 50 / temperature 0: 1 row 15.7 / 9.3 / 6.2; 148 rows 35 / 17.6 / 12.4; 1024
// rows 194 / 99 / 69, where memory would take 48. One row is a chain of latencies. Of many rows an SM has one at a time (its
// histogram), which takes 43000 cycles: counting 24000 (a warp's 32 additions meet random banks, 3.5 to one of them; the
// memory needs 13000), finding the groups 4000, their sums 6000 (11000 in fp16, which has ten times the values), prefix sums, the
// search and the token's place 7000. With a top-k 27000: reading 17000, bounds and the list 7000, the choice 3000.
//
// Short rows need none of this: they are sorted whole.
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "serving.h"
#include "stream.cuh"
#include "tcgen05.cuh"

namespace xpu {
namespace {

constexpr uint32_t kThreads = 1024, kWarps = kThreads / 32;
constexpr uint32_t kKeys = 65536, kGroups = kKeys / 32;
constexpr uint32_t kSmem = kKeys * 2;
constexpr uint32_t kMostListed = 256;  // top-k up to which the largest logits are looked for first
constexpr uint32_t kListed = kThreads;
constexpr uint32_t kJoined = 1u << 31;                  // a group's counters in block 0 are the row's: beside its count,
constexpr uint16_t kJoinedGroup = 0x8000;               // and beside its number
// Listed tokens up to which a token's place is counted, above which they are sorted: one row, top-k 200 (256 tokens) 12.3 and 14.3 us,
// top-k 250 (512) 15.7 and 15.1; top-k 50 (64 or 128) 9.3 and 12.2.
constexpr uint32_t kRanked = 256;
// Groups up to which a warp takes one at a time: 6200 cycles for 100 (bf16), 28000 for 1000 (fp16), where a thread each takes
// 10500 for up to 1024.
constexpr uint32_t kMostGroups = 192;
constexpr int kHeld = 5, kBatch = 4;  // pieces of 8 logits a thread holds of its block's run, or has in flight
static_assert(kHeld * kThreads * 8 < 65536, "counters of a held run do not overflow");
constexpr uint32_t kHeavy = 2 * XPU_SAMPLE_MAX_VOCABULARY / 32768 + 1;
constexpr uint32_t kRound = 32768;  // logits after which counters near overflow are emptied (slow way)

// 16-bit floats as whole numbers of the same order; -0 is 0.
__device__ __forceinline__ uint32_t key_of(uint32_t bits) {
  const uint32_t key = bits & 0x8000u ? bits ^ 0xffffu : bits | 0x8000u;
  return key == 0x7fffu ? 0x8000u : key;
}

template <typename T>
struct Keys;
template <>
struct Keys<__nv_bfloat16> {
  using Two = __nv_bfloat162;
  static constexpr uint32_t kMinusInf = 0x007f, kPlusInf = 0xff80;
  static constexpr uint32_t kMask = 0xff80ff80u, kLowest2 = 0xff7fff7fu;  // two of -inf, and of the lowest finite value
};
template <>
struct Keys<__half> {
  using Two = __half2;
  static constexpr uint32_t kMinusInf = 0x03ff, kPlusInf = 0xfc00;
  static constexpr uint32_t kMask = 0xfc00fc00u, kLowest2 = 0xfbfffbffu;
};

template <typename T>
__device__ __forceinline__ typename Keys<T>::Two as_two(uint32_t word) {
  return *reinterpret_cast<const typename Keys<T>::Two *>(&word);
}
// The larger of each half; NaN if one is.
template <typename T>
__device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t b) {
  const typename Keys<T>::Two v = __hmax2_nan(as_two<T>(a), as_two<T>(b));
  return *reinterpret_cast<const uint32_t *>(&v);
}
// Whether all of a piece's logits are above the lowest finite value.
template <typename T>
__device__ __forceinline__ bool all_above_lowest(const uint4 &v) {
  const auto least = __hmin2(__hmin2(as_two<T>(v.x), as_two<T>(v.y)), __hmin2(as_two<T>(v.z), as_two<T>(v.w)));
  return __hbgt2(least, as_two<T>(Keys<T>::kLowest2));
}

template <typename T>
__device__ __forceinline__ double value_of(uint32_t key) {
  const uint32_t bits = key & 0x8000u ? key & 0x7fffu : key ^ 0xffffu;
  return static_cast<double>(Elem<T>::lo(bits));
}

// Piece p of a row whose logits are [skipped, skipped + count) from base on; places outside are -inf.
template <typename T>
__device__ __noinline__ uint4 edge_piece(const uint16_t *base, uint32_t skipped, uint32_t count, uint32_t p) {
  uint32_t u[4];
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    u[i] = Keys<T>::kMask;
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t at = 8 * p + 2 * i + h;
      if (at >= skipped && at < skipped + count)
        u[i] = (u[i] & (h ? 0xffffu : 0xffff0000u)) | static_cast<uint32_t>(*reinterpret_cast<const volatile uint16_t *>(base + at)) << (16 * h);
    }
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// A row of logits at any 2-byte aligned address, in pieces of 8 from a 16-byte boundary on; places outside are -inf.
template <typename T>
struct Row {
  const uint16_t *base;  // 16-byte aligned, at or before the first logit
  uint32_t skipped, count, pieces;
  __device__ Row(const uint16_t *row, uint32_t vocabulary) : count(vocabulary) {
    skipped = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) & 15u) / 2;
    base = row - skipped;
    pieces = (skipped + count + 7) / 8;
  }
  __device__ __forceinline__ uint4 piece(uint32_t p) const {
    if (p == 0 || p + 1 == pieces) return edge_piece<T>(base, skipped, count, p);
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(base + 8ull * p) : "memory");
    return v;
  }
};

// The pieces begin .. end of a row that a block has, one a thread a turn.
template <typename T, bool HELD>
struct Run {
  Row<T> row;
  uint32_t begin, end;
  uint4 held[HELD ? kHeld : 1];
  __device__ Run(const uint16_t *logits, uint32_t vocabulary, uint32_t rank, uint32_t size) : row(logits, vocabulary) {
    const uint32_t share = (row.pieces + size - 1) / size;
    begin = min(rank * share, row.pieces);
    end = min(begin + share, row.pieces);
    if (HELD) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const uint32_t p = begin + threadIdx.x + i * kThreads;
        held[i] = make_uint4(Keys<T>::kMask, Keys<T>::kMask, Keys<T>::kMask, Keys<T>::kMask);
        if (p < end) held[i] = row.piece(p);
      }
    }
  }
  // use(piece, its number) for this thread's pieces from `from` on and below `to`; both at whole turns.
  template <typename Use>
  __device__ __forceinline__ void each(uint32_t from, uint32_t to, Use use) const {
    if (HELD) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (begin + threadIdx.x + i * kThreads < end) use(held[i], begin + threadIdx.x + i * kThreads);
      return;
    }
    for (uint32_t p = from + threadIdx.x; p < to; p += kBatch * kThreads) {
      uint4 v[kBatch];
#pragma unroll
      for (uint32_t i = 0; i < kBatch; ++i)
        if (p + i * kThreads < to) v[i] = row.piece(p + i * kThreads);
#pragma unroll
      for (uint32_t i = 0; i < kBatch; ++i)
        if (p + i * kThreads < to) use(v[i], p + i * kThreads);
    }
  }
};

__device__ __forceinline__ uint32_t element(const uint4 &v, int i) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  return u[i / 2] >> (16 * (i % 2)) & 0xffffu;
}

struct Shared {
  uint32_t counts[kGroups];  // logits of each group that is not empty, falling; then of the groups before it
  double masses[kGroups];    // likewise their weights
  union {
    uint16_t groups[kGroups];  // those that are not empty
    uint64_t list[kListed];    // key << 32 | ~id of what can be among the first k
  };
  uint32_t occupied[2][kWarps];  // 32 magnitudes each that this block's run has: of positive values, of negative ones
  double warp_mass[kWarps];
  uint32_t warp_count[kWarps];
  uint32_t heavy_key[kHeavy], heavy_count[kHeavy], heavies;
  uint32_t top[8], bad[8];  // of each block of the cluster
  uint32_t answer_key, answer_at;  // the token: its value, and which occurrence; kKeys: none
  uint32_t answer_joined;          // whether block 0's counter of that value is the row's
  uint32_t counted, listed, bounds[2][8];
  uint32_t coarse[2], wanted[2], fine[2][32];  // group of a bound, how many of its threads, their values
  uint32_t heavy_enough;  // tokens that min-p keeps
  double total;
};

template <int SIZE>
__device__ __forceinline__ void row_sync() {
  if (SIZE == 1) __syncthreads();
  else cluster_sync();
}

// Place of a value's 16-bit counter: a word for each magnitude, its lower half for the positive value, so that values side by side
// have words of their own and counting needs no order.
__device__ __forceinline__ uint32_t counter(uint32_t key) { return key & 0x8000u ? (key & 0x7fffu) << 1 : (key ^ 0x7fffu) << 1 | 1; }

// Occurrences of a value in block r's run.
template <int SIZE>
__device__ __forceinline__ uint32_t occurrences(const uint16_t *histogram, const Shared *sh, uint32_t key, uint32_t r, bool any_heavy) {
  uint32_t n;
  if (SIZE == 1) n = histogram[counter(key)];
  else asm volatile("{\n .reg .u16 t;\n ld.shared::cluster.u16 t, [%1];\n cvt.u32.u16 %0, t;\n}" : "=r"(n) : "r"(cluster_addr(histogram + counter(key), r)) : "memory");
  if (any_heavy) {
    for (uint32_t i = 0; i < kHeavy; ++i) {
      uint32_t k, c, many;
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(many) : "r"(cluster_addr(&sh->heavies, r)) : "memory");
      if (i >= many) break;
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(k) : "r"(cluster_addr(&sh->heavy_key[i], r)) : "memory");
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c) : "r"(cluster_addr(&sh->heavy_count[i], r)) : "memory");
      if (k == key) n += c;
    }
  }
  return n;
}

// Inclusive sum over a warp, in a fixed order.
template <typename V>
__device__ __forceinline__ V warp_scan(V v) {
  const uint32_t lane = threadIdx.x & 31;
#pragma unroll
  for (uint32_t o = 1; o < 32; o <<= 1) {
    const V up = __shfl_up_sync(kFullMask, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

struct Bin {  // one value of a group, a lane each, the largest in lane 0
  uint32_t key, count, before;  // occurrences, and tokens before them in the order
  double weight, mass;          // of one, and of all before
  bool joined;                  // counted in block 0 for all blocks
};

__device__ __forceinline__ uint32_t last_lane(bool yes) {
  const uint32_t votes = __ballot_sync(kFullMask, yes);
  return votes ? 31 - __clz(votes) : 0;
}

// Chooses among `listed` (up to kListed) tokens, thread i's being `mine` (key << 32 | ~id, 0 behind the last), which hold all
// that top-k keeps: put in order, one a thread. sh.counts are 0.
template <typename T>
__device__ void choose_listed(Shared &sh, uint64_t mine, uint32_t listed, uint32_t most, double slope, float top_p, float min_p,
                              float u, int32_t *token, float *logprob) {
  const uint32_t i = threadIdx.x, lane = i & 31, warp = i >> 5;
  if (most == 1) {  // temperature 0, or top-k 1: all listed are the largest value
    const uint32_t lowest = __reduce_max_sync(kFullMask, static_cast<uint32_t>(mine));
    if (lane == 0) atomicMax(&sh.counts[0], lowest);
    __syncthreads();
    if (i == 0) {
      *token = static_cast<int32_t>(~sh.counts[0]);
      if (logprob) *logprob = 0.f;
    }
    return;
  }
  uint32_t size = 32;
  while (size < listed) size *= 2;
  if (size <= kRanked) {  // each one's place is the number of larger ones, counted by several threads
    __syncthreads();
    if (i < size) sh.list[i] = mine;
    __syncthreads();
    const uint32_t entry = i & (size - 1), each = size * size / kThreads;
    const uint64_t own = sh.list[entry];
    uint32_t larger = 0;
    for (uint32_t j = i / size * each, end = j + each; j < end; ++j) larger += sh.list[j] > own;
    if (larger) atomicAdd(&sh.counts[entry], larger);
    __syncthreads();
    if (i < listed) sh.list[sh.counts[i]] = mine;
    __syncthreads();
    mine = i < listed ? sh.list[i] : 0;
  } else {
    for (uint32_t run = 2; run <= size; run *= 2) {  // bitonic, the largest first
      for (uint32_t stride = run / 2; stride > 0; stride /= 2) {
        uint64_t other;
        if (stride >= 32) {
          __syncthreads();
          sh.list[i] = mine;
          __syncthreads();
          other = sh.list[i ^ stride];
        } else {
          other = __shfl_xor_sync(kFullMask, mine, stride);
        }
        const bool larger = ((i & run) == 0) == ((i & stride) == 0);
        mine = larger == (mine > other) ? mine : other;
      }
    }
  }
  if (i == 0) sh.answer_key = static_cast<uint32_t>(mine >> 32);
  __syncthreads();
  const bool counts = i < listed && i < most;
  double z = 0.0, weight = 0.0;
  if (counts) {
    z = (value_of<T>(static_cast<uint32_t>(mine >> 32)) - value_of<T>(sh.answer_key)) * slope;
    weight = exp(z);
  }
  double sum = warp_scan(weight);
  if (lane == 31) sh.warp_mass[warp] = sum;
  const double up = __shfl_up_sync(kFullMask, sum, 1);
  __syncthreads();
  const double warps = warp_scan(sh.warp_mass[lane]), all = __shfl_sync(kFullMask, warps, 31);
  const double lower = warp ? __shfl_sync(kFullMask, warps, warp - 1) : 0.0;
  sum += lower;
  const double before = lower + (lane ? up : 0.0);
  const bool keep = counts && (i == 0 || ((top_p >= 1.f || before < static_cast<double>(top_p) * all) &&
                                          weight >= static_cast<double>(min_p) && weight > 0.0));
  const uint32_t kept = __syncthreads_count(keep);
  if (i + 1 == kept) sh.total = sum;
  __syncthreads();
  const uint32_t at = min(static_cast<uint32_t>(__syncthreads_count(keep && sum <= static_cast<double>(u) * sh.total)), kept - 1);
  if (i == at) {
    *token = static_cast<int32_t>(~static_cast<uint32_t>(mine));
    if (logprob) *logprob = static_cast<float>(z - log(sh.total));
  }
}

template <typename T, int SIZE>
__global__ void __launch_bounds__(kThreads, 1)
k_sample(const uint16_t *logits, uint64_t stride, const float *temperatures, const int32_t *top_ks, const float *top_ps,
         const float *min_ps, const float *us, int32_t *tokens, float *logprobs, uint32_t vocabulary) {
  extern __shared__ __align__(16) uint16_t histogram[];
  __shared__ Shared sh;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = SIZE == 1 ? 0 : cluster_rank(), row = blockIdx.x / SIZE;
  uint4 *const words = reinterpret_cast<uint4 *>(histogram);
  const auto clear_histogram = [&] {
    for (uint32_t i = threadIdx.x; i < kSmem / 16; i += kThreads) words[i] = make_uint4(0, 0, 0, 0);
  };
  for (uint32_t i = threadIdx.x; i < kGroups; i += kThreads) {
    sh.counts[i] = 0;
    sh.masses[i] = 0.0;
  }
  if (threadIdx.x == 0) {
    sh.heavies = sh.counted = sh.listed = 0;
    for (int i = 0; i < 8; ++i) sh.top[i] = sh.bad[i] = sh.bounds[0][i] = sh.bounds[1][i] = 0;
    sh.coarse[0] = sh.coarse[1] = kGroups;
  }
  if (threadIdx.x < 64) sh.fine[threadIdx.x / 32][lane] = 0;
  grid_dep_launch();
  grid_dep_wait();
  row_sync<SIZE>();

  const volatile float *const vt = temperatures, *const vp = top_ps, *const vm = min_ps, *const vu = us;
  const volatile int32_t *const vk = top_ks;
  const float temperature = temperatures ? vt[row] : 1.f, top_p = top_ps ? vp[row] : 1.f, min_p = min_ps ? vm[row] : 0.f;
  const int32_t top_k = top_ks ? vk[row] : 0;
  const float u = vu[row];
  const Run<T, (SIZE >= 4)> r(logits + row * stride, vocabulary, rank, SIZE);
  const bool asked = temperature >= 0.f && top_p == top_p && min_p == min_p && u >= 0.f && u < 1.f && top_k >= 0;
  const bool greedy = temperature == 0.f;
  const uint32_t most = greedy ? 1 : (top_k == 0 ? UINT32_MAX : static_cast<uint32_t>(top_k));
  const double slope = greedy ? 1.0 : 1.0 / static_cast<double>(temperature);
  const uint32_t begin = r.begin, end = r.end;

  uint32_t most2 = Keys<T>::kMask;  // the largest of this thread's logits, in each half
  const auto look = [&](const uint4 &v) { most2 = larger2<T>(larger2<T>(most2, larger2<T>(v.x, v.y)), larger2<T>(v.z, v.w)); };
  const auto top_of = [&] { return max(key_of(most2 & 0xffffu), key_of(most2 >> 16)); };
  // use(piece, its number) for the pieces of some of the warp's threads, spread over its lanes.
  const auto over_lanes = [&](uint32_t threads, auto use) {
    const uint32_t turns = (end - begin + kThreads - 1) / kThreads, items = __popc(threads) * turns;
    for (uint32_t item = lane; item < items; item += 32) {
      uint32_t left = threads;
      for (uint32_t skip = item / turns; skip; --skip) left &= left - 1;
      const uint32_t p = begin + 32 * warp + __ffs(left) - 1 + item % turns * kThreads;
      if (p < end) use(r.row.piece(p), p);
    }
  };
  const auto is_bad = [&] { return top_of() >= Keys<T>::kPlusInf; };  // the NaN of a maximum is positive

  if (most <= kMostListed) {
    r.each(begin, end, [&](const uint4 &v, uint32_t) { look(v); });
    const uint32_t mine = top_of();
    if (most > 1) {
      if (mine > Keys<T>::kMinusInf) atomicAdd(&sh.counts[mine / 32], 1u);
    } else {
      const uint32_t warp_top = __reduce_max_sync(kFullMask, mine);
      if (lane == 0) atomicMax(&sh.bounds[0][rank], warp_top);
    }
    const bool any_bad = __syncthreads_or(is_bad());
    if (most > 1) {
      // Lower bounds of the `most`-th largest logit: this block's `most`-th of the threads' largest; and the least of all blocks'
      // such values for their part of `most`. First the group of 32 values, thread i looking at groups 2047 - 2 i and
      // 2046 - 2 i, then the value.
      const uint32_t hi = kGroups - 1 - 2 * threadIdx.x, a = sh.counts[hi], b = sh.counts[hi - 1];
      const uint32_t inc = warp_scan(a + b);
      if (lane == 31) sh.warp_count[warp] = inc;
      __syncthreads();
      const uint32_t before = __reduce_add_sync(kFullMask, lane < warp ? sh.warp_count[lane] : 0) + inc - a - b;
      constexpr uint32_t kParts = SIZE == 1 ? 1 : 2;
#pragma unroll
      for (uint32_t part = 0; part < kParts; ++part) {
        const uint32_t n = part ? (most + SIZE - 1) / SIZE : most;
        const bool first = before < n && before + a >= n, second = before + a < n && before + a + b >= n;
        if (first || second) {
          sh.coarse[part] = first ? hi : hi - 1;
          sh.wanted[part] = n - before - (first ? 0 : a);
        }
      }
      __syncthreads();
#pragma unroll
      for (uint32_t part = 0; part < kParts; ++part)
        if (mine / 32 == sh.coarse[part]) atomicAdd(&sh.fine[part][31 - mine % 32], 1u);
      __syncthreads();
      if (warp < kParts && sh.coarse[warp] < kGroups) {
        const uint32_t votes = __ballot_sync(kFullMask, warp_scan(sh.fine[warp][lane]) >= sh.wanted[warp]);
        const uint32_t bound = 32 * sh.coarse[warp] + 32 - __ffs(votes);
        if (SIZE == 1) {
          if (lane == 0) sh.bounds[0][0] = bound;
        } else if (lane < SIZE) {
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(&sh.bounds[warp][rank], lane)), "r"(bound) : "memory");
        }
      }
      sh.counts[hi] = sh.counts[hi - 1] = 0;
    } else if (SIZE > 1 && threadIdx.x < SIZE && threadIdx.x != rank) {
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(&sh.bounds[0][rank], threadIdx.x)), "r"(sh.bounds[0][rank]) : "memory");
    }
    row_sync<SIZE>();
    uint32_t bound = Keys<T>::kMinusInf + 1, least = ~0u;
#pragma unroll
    for (int q = 0; q < SIZE; ++q) {
      bound = max(bound, sh.bounds[0][q]);
      least = min(least, sh.bounds[1][q]);
    }
    if (SIZE > 1 && most > 1) bound = max(bound, least);
    const auto list = [&](const uint4 &v, uint32_t p) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t key = key_of(element(v, i));
        if (key < bound) continue;
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < kListed) sh.list[at] = static_cast<uint64_t>(key) << 32 | ~(8 * p + i - r.row.skipped);
      }
    };
    if (SIZE >= 4) {
      if (mine >= bound) r.each(begin, end, list);
    } else {
      over_lanes(__ballot_sync(kFullMask, mine >= bound), list);
    }
    if (threadIdx.x == 0) sh.bad[0] = any_bad;
    row_sync<SIZE>();
    uint32_t listed = 0, none = !asked, from = 0, at = threadIdx.x;
#pragma unroll
    for (uint32_t q = 0; q < SIZE; ++q) {
      uint32_t n = sh.listed, bad = sh.bad[0];
      if (SIZE > 1) {
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(n) : "r"(cluster_addr(&sh.listed, q)) : "memory");
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(bad) : "r"(cluster_addr(&sh.bad[0], q)) : "memory");
      }
      if (threadIdx.x >= listed && threadIdx.x < listed + n) from = q, at = threadIdx.x - listed;
      listed += n;
      none |= bad;
    }
    none |= listed == 0;
    if (none || listed <= kListed) {  // the same for every block of the row
      if (rank == 0) {
        if (none) {
          if (threadIdx.x == 0) {
            tokens[row] = -1;
            if (logprobs) logprobs[row] = -INFINITY;
          }
        } else {
          uint64_t entry = 0;
          if (threadIdx.x < listed) {
            if (SIZE == 1) entry = sh.list[at];
            else asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(entry) : "r"(cluster_addr(&sh.list[at], from)) : "memory");
          }
          choose_listed<T>(sh, entry, listed, most, slope, top_p, min_p, u, tokens + row, logprobs ? logprobs + row : nullptr);
        }
      }
      if (SIZE > 1) cluster_sync();  // no block leaves while its list is read
      return;
    }
    row_sync<SIZE>();  // every block has seen the others' numbers
    if (threadIdx.x == 0) sh.bad[0] = 0;
  }

  clear_histogram();
  if (threadIdx.x < kWarps) sh.occupied[0][threadIdx.x] = sh.occupied[1][threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    sh.heavy_key[0] = Keys<T>::kMinusInf + 1;
    sh.heavy_count[0] = 0;
    sh.answer_joined = 0;
  }
  row_sync<SIZE>();  // what was cleared is, before another block writes there
  constexpr uint32_t kLowest = Keys<T>::kMinusInf + 1;  // the lowest finite value masks too: counted without the histogram

  uint32_t counted = 0, lowest = 0;
  const auto add = [&](uint32_t at_top) {  // a logit in the upper half of a word
    atomicAdd(reinterpret_cast<uint32_t *>(reinterpret_cast<char *>(histogram) + (at_top >> 14 & 0x1fffcu)),
              static_cast<int32_t>(at_top) < 0 ? 0x10000u : 1u);
  };
  const auto count = [&](uint32_t from, uint32_t to) {
    r.each(from, to, [&](const uint4 &v, uint32_t) {
      look(v);
      if (all_above_lowest<T>(v)) {
        counted += 8;
        add(v.x << 16), add(v.x), add(v.y << 16), add(v.y), add(v.z << 16), add(v.z), add(v.w << 16), add(v.w);
        return;
      }
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        const uint32_t word = i < 4 ? (i < 2 ? v.x : v.y) : (i < 6 ? v.z : v.w), bits = word >> (16 * (i % 2)) & 0xffffu, key = key_of(bits);
        if (key > kLowest) {
          ++counted;
          add(bits << 16);
        } else if (key == kLowest) {
          ++lowest;
        }
      }
    });
  };
  count(begin, end);
  __syncthreads();
  {
    const uint32_t n = __reduce_add_sync(kFullMask, lowest);
    if (lane == 0 && n) atomicAdd(&sh.heavy_count[0], n);
  }
  if (8 * (end - begin) > 65535) {
    // A counter may have passed 65535: then the sum of all is too small by a multiple of 65535 or 65536.
    uint32_t sum = 0;
    for (uint32_t i = threadIdx.x; i < kSmem / 16; i += kThreads) {
      const uint4 v = words[i];
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += element(v, e);
    }
    const uint32_t missing = __reduce_add_sync(kFullMask, counted - sum);
    if (lane == 0) atomicAdd(&sh.counted, missing);
    __syncthreads();
    if (sh.counted) {  // once more, emptying counters of 32768 and more after every 32768 logits
      clear_histogram();
      if (threadIdx.x == 0) sh.heavies = 1;
      __syncthreads();
      for (uint32_t from = begin; from < end; from += kRound / 8) {  // four whole turns
        count(from, min(end, from + kRound / 8));
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < kKeys; i += kThreads) {
          uint16_t *const held = histogram + counter(i);
          if (*held < kRound) continue;
          const uint32_t at = atomicAdd(&sh.heavies, 1u);
          sh.heavy_key[at] = i;
          sh.heavy_count[at] = *held;
          *held = 0;
          const uint32_t key = i == 0x7fff ? 0x8000 : i;
          const uint32_t magnitudes = counter(key) / 64;
          atomicOr(&sh.occupied[counter(key) & 1][magnitudes / 32], 1u << (magnitudes & 31));
        }
        __syncthreads();
      }
    }
  }
  uint32_t top = __reduce_max_sync(kFullMask, top_of()), bad = __any_sync(kFullMask, is_bad());
  if (lane == 0) {
    atomicMax(&sh.top[rank], top);
    atomicOr(&sh.bad[rank], bad);
  }
  __syncthreads();
  if (threadIdx.x == 0 && histogram[counter(0x7fff)]) {  // -0 is 0; a sum of more than 16 bits becomes a heavy one
    uint16_t *const zero = histogram + counter(0x8000), *const minus = histogram + counter(0x7fff);
    const uint32_t zeros = static_cast<uint32_t>(*zero) + *minus;
    *minus = 0;
    *zero = static_cast<uint16_t>(min(zeros, 65535u));
    if (zeros > 65535) {
      sh.heavies = max(sh.heavies, 1u);
      sh.heavy_key[sh.heavies] = 0x8000;
      sh.heavy_count[sh.heavies++] = zeros - 65535;
    }
  }
  if (sh.heavies && threadIdx.x < sh.heavies && sh.heavy_key[threadIdx.x] == 0x7fff) sh.heavy_key[threadIdx.x] = 0x8000;
  __syncthreads();
  {
    // Thread i looks at 32 magnitudes, from another 16 bytes on in each lane (banks).
    uint32_t has[2] = {0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint4 v = words[8 * threadIdx.x + ((i + lane) & 7)];
      const uint32_t any = v.x | v.y | v.z | v.w;
      has[0] |= any & 0xffffu;
      has[1] |= any >> 16;
    }
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const uint32_t votes = __ballot_sync(kFullMask, has[i]);
      if (lane == 0 && votes) atomicOr(&sh.occupied[i][warp], votes);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && sh.heavy_count[0]) {
    sh.heavies = max(sh.heavies, 1u);
    sh.occupied[1][counter(kLowest) / 64 / 32] |= 1u << (counter(kLowest) / 64 & 31);
  }
  if (SIZE > 1 && threadIdx.x < SIZE && threadIdx.x != rank) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(&sh.top[rank], threadIdx.x)), "r"(sh.top[rank]) : "memory");
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(&sh.bad[rank], threadIdx.x)), "r"(sh.bad[rank]) : "memory");
  }
  row_sync<SIZE>();

  uint32_t any_heavy = 0;
  top = bad = 0;
  uint32_t has[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < SIZE; ++i) {
    top = max(top, sh.top[i]);
    bad |= sh.bad[i];
    if (SIZE == 1) {
      any_heavy = sh.heavies;
      has[0] = sh.occupied[0][warp];
      has[1] = sh.occupied[1][warp];
    } else {
      uint32_t h, a, b;
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(h) : "r"(cluster_addr(&sh.heavies, i)) : "memory");
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(a) : "r"(cluster_addr(&sh.occupied[0][warp], i)) : "memory");
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(b) : "r"(cluster_addr(&sh.occupied[1][warp], i)) : "memory");
      any_heavy |= h;
      has[0] |= a;
      has[1] |= b;
    }
  }
  const bool none = bad || !asked || top <= Keys<T>::kMinusInf;
  const double largest = none ? 0.0 : value_of<T>(top);
  const auto log_weight = [&](uint32_t key) { return (value_of<T>(key) - largest) * slope; };

  if (none || greedy) {  // the same for every block of the row
    if (threadIdx.x == 0) {
      sh.answer_key = none ? kKeys : top;
      sh.answer_at = 0;
      if (rank == 0 && logprobs) logprobs[row] = none ? -INFINITY : 0.f;
      if (rank == 0 && none) tokens[row] = -1;
    }
    __syncthreads();
  } else {
    // The groups with values, and each block's share of them, their sums to block 0.
    const uint32_t below[2] = {__popc(has[0] & ((1u << lane) - 1)), __popc(has[1] & ((1u << lane) - 1))};
    if (lane == 0) sh.warp_count[warp] = __popc(has[0]) | __popc(has[1]) << 16;
    __syncthreads();
    const uint32_t of_warp = sh.warp_count[lane], earlier = __reduce_add_sync(kFullMask, lane < warp ? of_warp : 0);
    const uint32_t both = __reduce_add_sync(kFullMask, of_warp), negative = both >> 16, groups = (both & 0xffffu) + negative;
    if (has[1] >> lane & 1) sh.groups[negative - 1 - (earlier >> 16) - below[1]] = static_cast<uint16_t>(1023 - threadIdx.x);
    if (has[0] >> lane & 1) sh.groups[negative + (earlier & 0xffffu) + below[0]] = static_cast<uint16_t>(1024 + threadIdx.x);
    __syncthreads();
    const auto put = [&](uint32_t i, uint32_t n, double mass) {
      if (SIZE == 1) {
        sh.counts[groups - 1 - i] = n;
        sh.masses[groups - 1 - i] = mass;
      } else {
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(&sh.counts[groups - 1 - i], 0)), "r"(n) : "memory");
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(cluster_addr(&sh.masses[groups - 1 - i], 0)), "d"(mass) : "memory");
      }
    };
    if (SIZE == 1 && groups > kMostGroups) {
      // A thread a group: its values are evenly spaced, its weights a geometric series, w n_e + w r n_(e-1) + .. = w (n_e + r
      // (n_(e-1) + ..)) from its highest value e down, taken upwards from another value in each lane (banks): the part from
      // there to e, and the part below it times its power of r. e is the largest logit in its own group, whose weight is 1.
      for (uint32_t i = warp + kWarps * lane; i < groups; i += kThreads) {
        const uint32_t g = sh.groups[i], last = g == top / 32 ? top % 32 : 31, highest = 32 * g + last;
        const double ratio = exp((value_of<T>(highest - 1) - value_of<T>(highest)) * slope);
        double sum = 0.0, upper = 0.0;
        uint32_t many = 0;
#pragma unroll 4
        for (uint32_t k = 0; k < 32; ++k) {
          const uint32_t at = (lane + k) & 31;
          if (at == 0) upper = sum, sum = 0.0;
          const uint32_t n = occurrences<SIZE>(histogram, &sh, 32 * g + at, 0, any_heavy);
          many += n;
          if (at <= last) sum = fma(sum, ratio, __hiloint2double(0x43300000, static_cast<int>(n)) - 4503599627370496.0);  // 2^52 + n
        }
        double power = 1.0, factor = ratio;
        for (uint32_t left = lane && lane <= last ? last + 1 - lane : 0; left; left /= 2) {
          if (left & 1) power *= factor;
          factor *= factor;
        }
        put(i, many, exp(log_weight(highest)) * fma(sum, power, upper));
      }
    } else {
      for (uint32_t i = warp * SIZE + rank; i < groups; i += kWarps * SIZE) {
        const uint32_t key = 32 * sh.groups[i] + lane;
        uint32_t n = 0;
#pragma unroll
        for (int b = 0; b < SIZE; ++b) n += occurrences<SIZE>(histogram, &sh, key, b, any_heavy);
        double mass = n ? n * exp(log_weight(key)) : 0.0;
        // Block 0's counters become the row's, where they hold it: the search would wait 2000 cycles for the others' each time.
        const bool joined = SIZE > 1 && !any_heavy && __all_sync(kFullMask, n < 65536);
        if (joined) asm volatile("st.shared::cluster.u16 [%0], %1;" ::"r"(cluster_addr(histogram + counter(key), 0)), "h"(static_cast<uint16_t>(n)) : "memory");
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(kFullMask, mass, o);
        n = __reduce_add_sync(kFullMask, n);
        if (lane == 0) put(i, n | (joined ? kJoined : 0), mass);
      }
    }
    row_sync<SIZE>();
    if (rank == 0) {
      // Sums over the groups before each; thread i has groups 2 i and 2 i + 1.
      const uint32_t e = 2 * threadIdx.x, c0 = e < groups ? sh.counts[e] : 0, c1 = e + 1 < groups ? sh.counts[e + 1] : 0;
      const uint32_t n0 = c0 & ~kJoined, n1 = c1 & ~kJoined;
      if (c0 & kJoined) sh.groups[groups - 1 - e] |= kJoinedGroup;
      if (c1 & kJoined) sh.groups[groups - 2 - e] |= kJoinedGroup;
      const double m0 = e < groups ? sh.masses[e] : 0.0, m1 = e + 1 < groups ? sh.masses[e + 1] : 0.0;
      const uint32_t inc = warp_scan(n0 + n1);
      const double minc = warp_scan(m0 + m1);
      if (lane == 31) {
        sh.warp_count[warp] = inc;
        sh.warp_mass[warp] = minc;
      }
      __syncthreads();
      const uint32_t counts = warp_scan(sh.warp_count[lane]), all = __shfl_sync(kFullMask, counts, 31);
      const double masses = warp_scan(sh.warp_mass[lane]), all_mass = __shfl_sync(kFullMask, masses, 31);
      uint32_t before = __shfl_up_sync(kFullMask, inc, 1);
      double mass = __shfl_up_sync(kFullMask, minc, 1);
      const uint32_t lower = __shfl_sync(kFullMask, counts, warp ? warp - 1 : 0);
      const double lower_mass = __shfl_sync(kFullMask, masses, warp ? warp - 1 : 0);
      before = (lane ? before : 0) + (warp ? lower : 0);
      mass = (lane ? mass : 0.0) + (warp ? lower_mass : 0.0);
      if (e < groups) {
        sh.counts[e] = before;
        sh.masses[e] = mass;
      }
      if (e + 1 < groups) {
        sh.counts[e + 1] = before + n0;
        sh.masses[e + 1] = mass + m0;
      }
      __syncthreads();
      if (warp < 2) {
        // The last group of which yes(tokens before it, their weight); the first if there is none.
        const auto last_group = [&](auto yes) {
          uint32_t low = 0, many = groups;
          while (many > 1) {  // 32 places of [low, low + many) at once
            const uint32_t step = (many + 31) / 32, at = low + min(lane * step, many - 1);
            const uint32_t votes = __ballot_sync(kFullMask, yes(sh.counts[at], sh.masses[at]));
            const uint32_t run = votes == kFullMask ? 32 : __ffs(~votes) - 1, from = min((run ? run - 1 : 0) * step, many - 1);
            low += from;
            many = min(step, many - from);
          }
          return low;
        };
        const auto bins_of = [&](uint32_t group) {
          Bin bin;
          const uint32_t g = sh.groups[groups - 1 - group];
          bin.key = 32 * (g & (kGroups - 1)) + 31 - lane;
          bin.count = 0;
          bin.joined = SIZE > 1 && (g & kJoinedGroup);
          if (bin.joined) {
            bin.count = histogram[counter(bin.key)];
          } else {
#pragma unroll
            for (int b = 0; b < SIZE; ++b) bin.count += occurrences<SIZE>(histogram, &sh, bin.key, b, any_heavy);
          }
          bin.weight = bin.count ? exp(log_weight(bin.key)) : 0.0;
          const double m = warp_scan(bin.count * bin.weight);
          const double up = __shfl_up_sync(kFullMask, m, 1);
          bin.before = sh.counts[group] + warp_scan(bin.count) - bin.count;
          bin.mass = sh.masses[group] + (lane ? up : 0.0);
          return bin;
        };
        // Weight of the first n tokens.
        const auto weight_of_first = [&](uint32_t n) {
          const Bin b = bins_of(last_group([&](uint32_t c, double) { return c < n; }));
          const uint32_t at = last_lane(b.count && b.before < n);
          return __shfl_sync(kFullMask, b.mass + min(n - b.before, b.count) * b.weight, at);
        };
        if (warp == 1 && min_p > 0.f && min_p <= 1.f) {  // what min-p keeps, while the other warp looks at top-k and top-p
          // The lowest value that is heavy enough: one of the keys [low, low + many).
          uint32_t low = 0, many = top + 1;
          while (many > 1) {
            const uint32_t step = (many + 31) / 32, at = low + min((lane + 1) * step, many) - 1;
            const double weight = at > Keys<T>::kMinusInf ? exp(log_weight(at)) : 0.0;
            const uint32_t votes = __ballot_sync(kFullMask, weight >= static_cast<double>(min_p));
            const uint32_t chosen = votes ? __ffs(votes) - 1 : 31, from = min(chosen * step, many - 1);
            low += from;
            many = min(step, many - from);
          }
          // tokens of that value and above
          uint32_t found = 0, place = groups;  // the first group whose highest value is below it
          for (uint32_t from = 0; from < groups && place == groups; from += 32) {
            const uint32_t at = from + lane;
            const uint32_t votes = __ballot_sync(kFullMask, at < groups && 32u * (sh.groups[groups - 1 - at] & (kGroups - 1)) + 31 < low);
            if (votes) place = from + __ffs(votes) - 1;
          }
          if (place > 0) {
            const Bin b = bins_of(place - 1);
            const uint32_t in = __reduce_add_sync(kFullMask, b.key >= low ? b.count : 0);
            found = sh.counts[place - 1] + in;
          }
          if (lane == 0) sh.heavy_enough = found;
          asm volatile("bar.sync 1, 64;" ::: "memory");
        }
        if (warp == 0) {
          uint32_t kept = min(most, all);
          double total = kept == all ? all_mass : weight_of_first(kept);
          uint32_t fewer = kept;
          if (top_p < 1.f) {
            const double wanted = static_cast<double>(top_p) * total;
            const Bin b = bins_of(last_group([&](uint32_t, double m) { return m < wanted; }));
            const uint32_t at = last_lane(b.count && b.mass < wanted);
            const double need = fmin(fmax(ceil((wanted - b.mass) / b.weight), 1.0), static_cast<double>(b.count));
            fewer = min(fewer, __shfl_sync(kFullMask, b.before + (b.count ? static_cast<uint32_t>(need) : 0), at));
          }
          if (min_p > 1.f) {
            fewer = 1;
          } else if (min_p > 0.f) {
            asm volatile("bar.sync 1, 64;" ::: "memory");
            fewer = min(fewer, sh.heavy_enough);
          }
          fewer = max(fewer, 1u);
          if (fewer < kept) total = weight_of_first(kept = fewer);
          const double wanted = static_cast<double>(u) * total;
          const Bin b = bins_of(last_group([&](uint32_t c, double m) { return c < kept && m <= wanted; }));
          const uint32_t at = last_lane(b.count && b.weight > 0.0 && b.before < kept && b.mass <= wanted);
          if (lane == at) {
            const uint32_t in = max(min(b.count, kept - b.before), 1u);  // of its occurrences are kept
            const double which = floor((wanted - b.mass) / b.weight);
            const uint32_t j = which < in ? static_cast<uint32_t>(which) : in - 1;
            if (logprobs) logprobs[row] = static_cast<float>(log_weight(b.key) - log(total));
            for (int i = 0; i < SIZE; ++i) {
              if (SIZE == 1) {
                sh.answer_key = b.key;
                sh.answer_at = j;
              } else {
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(&sh.answer_key, i)), "r"(b.key) : "memory");
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(&sh.answer_at, i)), "r"(j) : "memory");
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(&sh.answer_joined, i)), "r"(static_cast<uint32_t>(b.joined)) : "memory");
              }
            }
          }
        }
      }
    }
    row_sync<SIZE>();
  }

  // The answer's place in the row: which block's run has that occurrence, then which warp's.
  const uint32_t key = sh.answer_key;
  uint32_t j = sh.answer_at, here = 0, of_block[SIZE];
#pragma unroll
  for (uint32_t b = 0; b < SIZE; ++b) of_block[b] = key < kKeys ? occurrences<SIZE>(histogram, &sh, key, b, any_heavy) : 0;
  if (SIZE > 1 && sh.answer_joined) {
#pragma unroll
    for (uint32_t b = 1; b < SIZE; ++b) of_block[0] -= of_block[b];
  }
  bool mine = key < kKeys;
#pragma unroll
  for (uint32_t b = 0; b < SIZE; ++b) {
    if (b == rank) {
      here = of_block[b];
      mine = mine && j < here;
    } else if (b < rank) {
      mine = mine && j >= of_block[b];
      j -= of_block[b];
    }
  }
  // A bit for each of a piece's logits that has the value; 0 has two forms.
  const uint32_t form = key & 0x8000u ? key & 0x7fffu : key ^ 0xffffu, form2 = form << 16 | form, other2 = form ? form2 : 0x80008000u;
  const auto matches = [&](const uint4 &v) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
    uint32_t equal[4], any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      equal[i] = __vcmpeq2(u[i], form2) | __vcmpeq2(u[i], other2);
      any |= equal[i];
    }
    if (any == 0) return 0u;
    uint32_t mask = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) mask |= (equal[i] & 1u) << 2 * i | (equal[i] >> 31) << (2 * i + 1);
    return mask;
  };
  if (mine && here <= kListed) {  // listed by the threads whose largest logit is not below it, then the j-th in the order of ids
    uint32_t *const ids = reinterpret_cast<uint32_t *>(sh.list);
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    const auto list = [&](const uint4 &v, uint32_t p) {
      for (uint32_t mask = matches(v); mask; mask &= mask - 1) {
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < kListed) ids[at] = 8 * p + __ffs(mask) - 1 - r.row.skipped;
      }
    };
    const bool may = top_of() >= key;
    const uint32_t threads = __ballot_sync(kFullMask, may);
    if (SIZE >= 4 || __popc(threads) > 4) {
      if (may) r.each(begin, end, list);
    } else {
      over_lanes(threads, list);
    }
    __syncthreads();
    const uint32_t id = threadIdx.x < here ? ids[threadIdx.x] : 0;
    uint32_t lower = 0;
    if (threadIdx.x < here)
      for (uint32_t i = 0; i < here; ++i) lower += ids[i] < id;
    if (threadIdx.x < here && lower == j) tokens[row] = static_cast<int32_t>(id);
  } else if (mine) {  // a run of pieces a warp, whose occurrences are counted first
    const uint32_t run = (end - begin + kWarps - 1) / kWarps, from = begin + warp * run, to = min(from + run, end);
    uint32_t n = 0;
    for (uint32_t p = from + lane; p < to; p += 4 * 32) {
      uint4 v[4];
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        if (p + 32 * i < to) v[i] = r.row.piece(p + 32 * i);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        if (p + 32 * i < to) n += __popc(matches(v[i]));
    }
    {
      n = __reduce_add_sync(kFullMask, n);
      if (lane == 0) sh.warp_count[warp] = n;
      __syncthreads();
      uint32_t earlier = 0;
      for (uint32_t w = 0; w < warp; ++w) earlier += sh.warp_count[w];
      if (j >= earlier && j - earlier < n) {
        j -= earlier;
        for (uint32_t p = from; p < to; p += 32) {
          const uint32_t mask = p + lane < to ? matches(r.row.piece(p + lane)) : 0;
          const uint32_t inc = warp_scan(static_cast<uint32_t>(__popc(mask)));
          const uint32_t many = __shfl_sync(kFullMask, inc, 31), before = inc - __popc(mask);
          if (j < many) {
            if (j >= before && j < inc) {
              uint32_t left = mask;
              for (uint32_t skip = j - before; skip; --skip) left &= left - 1;
              tokens[row] = static_cast<int32_t>(8 * (p + lane) + __ffs(left) - 1 - r.row.skipped);
            }
            break;
          }
          j -= many;
        }
      }
    }
  }
  if (SIZE > 1) cluster_sync();  // no block leaves while another may read its counters
}

// Rows of up to kShort logits: all are sorted, four a thread, as key << 16 | ~id (0: none), so that a block needs little shared memory
// and an SM holds several. Without limits, us here and through the histogram: 250 logits, 1 row 3.9 and 10.7, 1024 rows 9.4 and 74;
// 2000 logits 8.0 and 10.3, 42 and 70; 4096 logits 14.6 and 10.3, 102 and 71.
constexpr uint32_t kShort = 2048;

template <typename T>
__global__ void __launch_bounds__(kShort / 4)
k_sample_short(const uint16_t *logits, uint64_t stride, const float *temperatures, const int32_t *top_ks, const float *top_ps,
               const float *min_ps, const float *us, int32_t *tokens, float *logprobs, uint32_t vocabulary) {
  extern __shared__ __align__(16) uint4 exchange[];  // two of blockDim.x
  __shared__ double warp_mass[kWarps], total;
  __shared__ uint32_t warp_most[kWarps], warp_kept[kWarps], warp_below[kWarps];
  const uint32_t i = threadIdx.x, lane = i & 31, warp = i >> 5, row = blockIdx.x;
  if (i < kWarps) {
    warp_mass[i] = 0.0;
    warp_most[i] = warp_kept[i] = warp_below[i] = 0;
  }
  grid_dep_launch();
  grid_dep_wait();
  const volatile float *const vt = temperatures, *const vp = top_ps, *const vm = min_ps, *const vu = us;
  const volatile int32_t *const vk = top_ks;
  const volatile uint16_t *const vl = logits + row * stride;
  uint32_t e[4];
  bool bad = false;
#pragma unroll
  for (uint32_t q = 0; q < 4; ++q) {
    const uint32_t id = q * blockDim.x + i, bits = id < vocabulary ? vl[id] : Keys<T>::kMask & 0xffffu, key = key_of(bits);
    constexpr uint32_t inf = Keys<T>::kPlusInf & 0x7fffu;
    bad |= bits == inf || (bits & 0x7fffu) > inf;
    e[q] = key > Keys<T>::kMinusInf ? key << 16 | (id ^ 0xffffu) : 0;
  }
  const float temperature = temperatures ? vt[row] : 1.f, top_p = top_ps ? vp[row] : 1.f, min_p = min_ps ? vm[row] : 0.f;
  const int32_t top_k = top_ks ? vk[row] : 0;
  const float u = vu[row];
  const bool asked = temperature >= 0.f && top_p == top_p && min_p == min_p && u >= 0.f && u < 1.f && top_k >= 0;
  const bool greedy = temperature == 0.f;
  const uint32_t most = greedy ? 1 : (top_k == 0 ? UINT32_MAX : static_cast<uint32_t>(top_k));
  const double slope = greedy ? 1.0 : 1.0 / static_cast<double>(temperature);
  uint32_t first = __reduce_max_sync(kFullMask, max(max(e[0], e[1]), max(e[2], e[3])));
  if (__syncthreads_or(bad)) first = 0;  // here the sums of absent warps are 0, too
  if (lane == 0) warp_most[warp] = first;
  __syncthreads();
  first = __reduce_max_sync(kFullMask, warp_most[lane]);
  if (!asked || first == 0 || most == 1) {
    if (i == 0) {
      const bool none = !asked || first == 0;
      tokens[row] = none ? -1 : static_cast<int32_t>((first & 0xffffu) ^ 0xffffu);
      if (logprobs) logprobs[row] = none ? -INFINITY : 0.f;
    }
    return;
  }

  // Bitonic, the largest first: thread i has places 4 i to 4 i + 3.
  const auto pick = [](uint32_t &mine, uint32_t other, bool larger) { mine = larger ? max(mine, other) : min(mine, other); };
  const auto both = [](uint32_t &a, uint32_t &b, bool larger_first) {
    const uint32_t hi = max(a, b), lo = min(a, b);
    a = larger_first ? hi : lo;
    b = larger_first ? lo : hi;
  };
  both(e[0], e[1], true);
  both(e[2], e[3], false);
  uint32_t turn = 0;
  for (uint32_t run = 1; run <= blockDim.x; run *= 2) {  // of threads
    const bool falling = (i & run) == 0;
    for (uint32_t far = run / 2; far > 0; far /= 2) {
      const bool larger = falling == ((i & far) == 0);
      if (far >= 32) {
        uint4 *const at = exchange + (turn ^= 1) * blockDim.x;  // the other half may still be read
        at[i] = make_uint4(e[0], e[1], e[2], e[3]);
        __syncthreads();
        const uint4 other = at[i ^ far];
        pick(e[0], other.x, larger), pick(e[1], other.y, larger), pick(e[2], other.z, larger), pick(e[3], other.w, larger);
      } else {
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) pick(e[q], __shfl_xor_sync(kFullMask, e[q], far), larger);
      }
    }
    both(e[0], e[2], falling), both(e[1], e[3], falling);
    both(e[0], e[1], falling), both(e[2], e[3], falling);
  }

  const double largest = value_of<T>(first >> 16);
  double z[4], weight[4], sum[4], thread_sum = 0.0;
#pragma unroll
  for (uint32_t q = 0; q < 4; ++q) {
    z[q] = weight[q] = 0.0;
    if (e[q] && 4 * i + q < most) {
      z[q] = (value_of<T>(e[q] >> 16) - largest) * slope;
      weight[q] = exp(z[q]);
    }
    sum[q] = thread_sum += weight[q];
  }
  const double inc = warp_scan(thread_sum), up = __shfl_up_sync(kFullMask, inc, 1);
  if (lane == 31) warp_mass[warp] = inc;
  __syncthreads();
  const double masses = warp_scan(warp_mass[lane]), all = __shfl_sync(kFullMask, masses, 31);
  const double lower = warp ? __shfl_sync(kFullMask, masses, warp - 1) : 0.0, before = lower + (lane ? up : 0.0);
  uint32_t kept = 0;
  bool keep[4];
#pragma unroll
  for (uint32_t q = 0; q < 4; ++q) {
    sum[q] = fmin(before + sum[q], lower + inc);  // never above the next thread's
    const bool counts = e[q] && 4 * i + q < most;
    keep[q] = counts && (4 * i + q == 0 || ((top_p >= 1.f || (q ? sum[q ? q - 1 : 0] : before) < static_cast<double>(top_p) * all) &&
                                            weight[q] >= static_cast<double>(min_p) && weight[q] > 0.0));
    kept += keep[q];
  }
  kept = __reduce_add_sync(kFullMask, kept);
  if (lane == 0) warp_kept[warp] = kept;
  __syncthreads();
  kept = __reduce_add_sync(kFullMask, warp_kept[lane]);
#pragma unroll
  for (uint32_t q = 0; q < 4; ++q)
    if (4 * i + q + 1 == kept) total = sum[q];
  __syncthreads();
  uint32_t below = 0;
#pragma unroll
  for (uint32_t q = 0; q < 4; ++q) below += keep[q] && sum[q] <= static_cast<double>(u) * total;
  below = __reduce_add_sync(kFullMask, below);
  if (lane == 0) warp_below[warp] = below;
  __syncthreads();
  const uint32_t at = min(__reduce_add_sync(kFullMask, warp_below[lane]), kept - 1);
#pragma unroll
  for (uint32_t q = 0; q < 4; ++q) {
    if (4 * i + q == at) {
      tokens[row] = static_cast<int32_t>((e[q] & 0xffffu) ^ 0xffffu);
      if (logprobs) logprobs[row] = static_cast<float>(z[q] - log(total));
    }
  }
}

template <typename T, int SIZE>
cudaError_t launch(const SampleArgs &a, cudaStream_t s, bool *fits) {
  const auto kernel = k_sample<T, SIZE>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = SIZE;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(a.rows * SIZE);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = SIZE > 1 ? 2 : 1;
  if (SIZE > 1) {
    int device = 0;
    if ((e = cudaGetDevice(&device)) != cudaSuccess) return e;
    static std::atomic<int> resident[64];  // clusters at once
    int clusters = resident[device & 63].load(std::memory_order_relaxed);
    if (clusters == 0) {
      if ((e = cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg)) != cudaSuccess) return e;
      resident[device & 63].store(clusters = std::max(clusters, 1), std::memory_order_relaxed);
    }
    if (!(*fits = a.rows <= static_cast<uint32_t>(clusters))) return cudaSuccess;
  }
  *fits = true;
  return cudaLaunchKernelEx(&cfg, kernel, a.logits, a.stride, a.temperature, a.top_k, a.top_p, a.min_p, a.u, a.tokens, a.logprobs,
                            a.vocabulary);
}

// The most blocks a row with which all rows are resident at once; a run of fewer than 4096 logits a block would not pay for
// the cluster's barriers.
template <typename T>
cudaError_t best_launch(const SampleArgs &a, cudaStream_t s) {
  bool done = false;
  cudaError_t e = cudaSuccess;
  if (a.vocabulary <= kShort) {
    uint32_t threads = 32;
    while (4 * threads < a.vocabulary) threads *= 2;
    return launch_after(k_sample_short<T>, a.rows, threads, 2 * threads * sizeof(uint4), s, a.logits, a.stride, a.temperature, a.top_k,
                        a.top_p, a.min_p, a.u, a.tokens, a.logprobs, a.vocabulary);
  }
  // up to 8 blocks x kHeld x 1024 pieces, one piece more where the row's address is odd
  const uint32_t pieces = (a.vocabulary + 14) / 8;
  if (a.vocabulary >= 8 * 4096 && (pieces + 7) / 8 <= kHeld * kThreads) e = launch<T, 8>(a, s, &done);
  if (e == cudaSuccess && !done && a.vocabulary >= 4 * 4096 && (pieces + 3) / 4 <= kHeld * kThreads) e = launch<T, 4>(a, s, &done);
  if (e == cudaSuccess && !done && a.vocabulary >= 2 * 4096) e = launch<T, 2>(a, s, &done);
  return e != cudaSuccess || done ? e : launch<T, 1>(a, s, &done);
}

}  // namespace

cudaError_t sample_launch(bool fp16, const SampleArgs &a, cudaStream_t s) {
  return fp16 ? best_launch<__half>(a, s) : best_launch<__nv_bfloat16>(a, s);
}

}  // namespace xpu
