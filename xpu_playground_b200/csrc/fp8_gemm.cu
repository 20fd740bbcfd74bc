// Product of 8-bit rows with 8-bit weights (xpu_fp8_gemm in include/xpu_cuda.h):
//
//   c[m][n] = sum_g sa[g][m] sw[n / 128][g] sum_{k in g} a[m][k] w[n][k]
//
// over the groups g of 128 columns. The inner sums run on the tensor cores
// (tcgen05, kind::f8f6f4, four instructions of 32 columns a group) into TMEM; every
// group is its own accumulation there, which other warps read, scale and add up
// in FP32 registers while the tensor cores work on the next group in another
// TMEM buffer.
//
// Few rows (k_skinny): reading the weights bounds it. A block takes 128 rows of w
// as the M side of its products and NT rows of a as the N side, so that a tile of
// weights is read once; the blocks of a cluster share the groups of one
// tile and add their sums up through distributed shared memory, in a fixed order. 16 x 24576 x 4096: 19.6 us (5.2 TB/s);
// 1 x 6144 x 4096: 6.6, of which the memory takes 3.8 and start, first load, cluster sum and end the rest.
//
// Many rows (k_wide): the tensor cores bound it. Two blocks of a cluster work as a pair
// (cta_group::2) on 256 x 256 outputs, each with 128 rows of a and 128 of w in its shared
// memory and 128 x 256 sums in its TMEM, twice. Eight warps a block hold the tile's
// FP32 sums in registers: a thread has one row and the 128 columns of one scale block, so
// that a group's scale is one number a thread. The finished tile leaves through shared
// memory while the next one's products run. 8192 x 24576 x 4096: 878 us in a long run (1.88 PFLOP/s: power), 726 on a cool card
// (2.27), 565 there with the adding up left out; 777 x 4096 x 12288: 57.6 and 48 (1.36 and 1.63 PFLOP/s; 64 tiles for 74 pairs).
#include <cuda.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "serving.h"
#include "stream.cuh"
#include "tcgen05.cuh"

namespace xpu {

__device__ unsigned int g_fp8_error = 0;

namespace {

constexpr uint32_t kGroup = XPU_FP8_BLOCK;
constexpr uint32_t kTileN = 128;                 // rows of w a tile: one row of scale blocks
constexpr uint32_t kTileBytes = kTileN * kGroup;  // 128 swizzled rows of 128 bytes
constexpr unsigned kErrTimeout = 1u;

// kind::f8f6f4, both operands e4m3 and K-major, FP32 accumulator.
constexpr uint32_t instr_desc(uint32_t m, uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((m >> 4) << 24); }

__device__ __forceinline__ void mma1_f8(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ bool has_failed(const int *flag) { return *reinterpret_cast<const volatile int *>(flag) != 0; }

// sums (two of them) += {lo, hi} * scale (twice the same).
__device__ __forceinline__ void fma2(uint64_t &sums, uint32_t lo, uint32_t hi, uint64_t scale) {
  asm("{\n .reg .b64 d;\n mov.b64 d, {%1, %2};\n fma.rn.f32x2 %0, d, %3, %0;\n}" : "+l"(sums) : "r"(lo), "r"(hi), "l"(scale));
}

// The same answer for the whole warp, so that its lanes stay together.
__device__ __forceinline__ bool warp_wait(int *failed, uint64_t *bar, uint32_t parity) {
  if (__all_sync(kFullMask, mbar_wait(bar, parity))) return true;
  *failed = 1;
  return false;
}

// Waits for the TMEM loads in flight, whose registers are usable from here on.
__device__ __forceinline__ void tmem_landed(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// Arrives on a barrier of the even block to say that this warp has read a TMEM buffer. Nothing that it wrote is passed on: the loads
// have been waited for, and the next products overwrite what they read. So relaxed: a release at cluster scope waits for
// every access of the warp, 1000 cycles a group here. What one warp writes for another passes through a barrier of their own block.
__device__ __forceinline__ void pair_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(uint64_t pair) {
  const T lo = Elem<T>::from_float(__uint_as_float(static_cast<uint32_t>(pair)));
  const T hi = Elem<T>::from_float(__uint_as_float(static_cast<uint32_t>(pair >> 32)));
  return *reinterpret_cast<const uint16_t *>(&lo) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(&hi)) << 16;
}

// A float that the kernel before may have written.
__device__ __forceinline__ float ld_f32(const float *p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}

// ---------------------------------------------------------------- few rows ----

template <int NT>
struct Skinny {
  static constexpr uint32_t kBuffers = 4, kColumns = NT * kBuffers;
  static constexpr uint32_t kStageBytes = kTileBytes + NT * kGroup;
  static constexpr uint32_t kStages = NT <= 32 ? 5 : 4;  // two blocks an SM
  static constexpr uint32_t kChunk = 8;                  // groups whose scales are held, twice
  static constexpr uint32_t kSmem = 1024 + kStages * kStageBytes + 2 * kChunk * NT * 4;
  static_assert(NT * kTileN * 4 <= kStages * kStageBytes, "the sums of a tile take the ring's place");
};
constexpr uint32_t kSkinnyThreads = 192, kSkinnyBlocks = 2;

// Warp 0 loads, warp 1 issues the products (converged, as in k_wide), warps 2 to 5 add up: a thread has one row of w and NT
// sums.
template <typename T, int NT>
__global__ void __launch_bounds__(kSkinnyThreads, kSkinnyBlocks)
k_skinny(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const float *a_scales,
         const float *w_scales, T *c, uint32_t m, uint32_t n, uint32_t groups, uint32_t split) {
  using S = Skinny<NT>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t full[S::kStages], empty[S::kStages], sum_full[S::kBuffers], sum_empty[S::kBuffers], drain;
  __shared__ uint32_t tmem_base;
  __shared__ int failed;
  const uint32_t a0 = smem_addr(smem_raw);
  uint8_t *ring = smem_raw + ((a0 + 1023u) / 1024u * 1024u - a0);
  float *scales = reinterpret_cast<float *>(ring + S::kStages * S::kStageBytes);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = blockIdx.x % split, tile = blockIdx.x / split, tiles_m = (m + NT - 1) / NT;
  const uint32_t tile_n = tile / tiles_m, tile_m = tile % tiles_m;  // tiles of the same weights run side by side
  const uint32_t first = static_cast<uint32_t>(static_cast<uint64_t>(groups) * rank / split);
  const uint32_t count = static_cast<uint32_t>(static_cast<uint64_t>(groups) * (rank + 1) / split) - first;

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (uint32_t i = 0; i < S::kBuffers; ++i) {
      mbar_init(&sum_full[i], 1);
      mbar_init(&sum_empty[i], 4);
    }
    mbar_init(&drain, 1);
    fence_mbar_init();
    failed = 0;
  }
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
  }
  if (warp == 1) tmem_alloc1(&tmem_base, S::kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  grid_dep_launch();  // with the TMEM held: a block of the next kernel cannot take it from one of this
  grid_dep_wait();

  uint64_t sums[NT / 2];
  const uint32_t row = (warp & 3) * 32 + lane;  // of the tile; warps 2 to 5 have the TMEM quarters 2, 3, 0, 1
  const uint32_t held = min(static_cast<uint32_t>(NT), m - tile_m * NT);
  if (warp == 0) {
    if (lane == 0) {
      uint32_t i = 0;
      for (; i < count && !has_failed(&failed); ++i) {
        const uint32_t s = i % S::kStages, use = i / S::kStages;
        if (use > 0 && !mbar_wait(&empty[s], (use - 1) & 1)) { failed = 1; break; }
        mbar_expect_tx(&full[s], S::kStageBytes);
        uint8_t *st = ring + s * S::kStageBytes;
        const int32_t x = static_cast<int32_t>((first + i) * kGroup);
        tma_load_2d_plain(st, &map_w, x, static_cast<int32_t>(tile_n * kTileN), &full[s]);
        tma_load_2d_plain(st + kTileBytes, &map_a, x, static_cast<int32_t>(tile_m * NT), &full[s]);
      }
      if (has_failed(&failed))  // no copy may land once this block's shared memory is another's
        for (uint32_t back = 0; back < S::kStages && back < i; ++back) mbar_wait(&full[(i - 1 - back) % S::kStages], (i - 1 - back) / S::kStages & 1);
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = instr_desc(kTileN, NT);
    for (uint32_t i = 0; i < count; ++i) {
      const uint32_t s = i % S::kStages, b = i % S::kBuffers, use = i / S::kBuffers;
      if (!warp_wait(&failed, &full[s], i / S::kStages & 1)) break;
      if (use > 0 && !warp_wait(&failed, &sum_empty[b], (use - 1) & 1)) break;
      tc_fence_after();
      const uint32_t st = smem_addr(ring + s * S::kStageBytes);
      const uint64_t dw = smem_desc(st, 16, 1024), da = smem_desc(st + kTileBytes, 16, 1024);
      if (elect_one()) {
#pragma unroll
        for (uint32_t kk = 0; kk < 4; ++kk) mma1_f8(tmem + b * NT, dw + 2 * kk, da + 2 * kk, idesc, kk != 0);
        mma1_commit(&empty[s]);
        mma1_commit(&sum_full[b]);
      }
      __syncwarp();
    }
    if (elect_one()) mma1_commit(&drain);
    warp_wait(&failed, &drain, 0);
  } else {
    const uint32_t et = threadIdx.x - 64;
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) sums[j] = 0;
    constexpr uint32_t kEach = S::kChunk * NT / 128;  // scales a thread brings
    float next[kEach];
    const auto fetch = [&](uint32_t at) {  // of groups first + at ..
#pragma unroll
      for (uint32_t e = 0; e < kEach; ++e) {
        const uint32_t i = e * 128 + et, g = at + i / NT, j = i % NT;
        next[e] = 0.f;
        if (g < count && j < held)
          next[e] = ld_f32(a_scales + static_cast<uint64_t>(first + g) * m + tile_m * NT + j) *
                    ld_f32(w_scales + static_cast<uint64_t>(tile_n) * groups + first + g);
      }
    };
    fetch(0);
    for (uint32_t i = 0; i < count; ++i) {
      float *const chunk = scales + (i / S::kChunk & 1) * S::kChunk * NT;
      if (i % S::kChunk == 0) {
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) chunk[e * 128 + et] = next[e];
        asm volatile("bar.sync 1, 128;" ::: "memory");  // the other half was read before this one's last barrier
        fetch(i + S::kChunk);
      }
      const uint32_t b = i % S::kBuffers;
      // A warp that gives up goes on without waiting: the others count on it at the barrier above.
      if (!has_failed(&failed) && !mbar_wait(&sum_full[b], i / S::kBuffers & 1)) failed = 1;
      __syncwarp();
      tc_fence_after();
      const ulonglong2 *const by = reinterpret_cast<const ulonglong2 *>(chunk + i % S::kChunk * NT);
      const uint32_t taddr = tmem + ((warp & 3) * 32u << 16) + b * NT;
      uint32_t d[2][16];
      tmem_ld16_nowait(taddr, d[0]);
#pragma unroll
      for (int piece = 0; piece < NT / 16; ++piece) {
        uint32_t(&now)[16] = d[piece & 1];
        tmem_landed(now);
        if (piece + 1 < NT / 16) {
          tmem_ld16_nowait(taddr + 16 * (piece + 1), d[(piece + 1) & 1]);
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sum_empty[b]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const ulonglong2 s = by[4 * piece + q];
          fma2(sums[8 * piece + 2 * q], now[4 * q], now[4 * q + 1], s.x);
          fma2(sums[8 * piece + 2 * q + 1], now[4 * q + 2], now[4 * q + 3], s.y);
        }
      }
    }
    const auto sum = [&](int j) { return __uint_as_float(static_cast<uint32_t>(sums[j / 2] >> (32 * (j % 2)))); };
    if (split == 1) {
      T *const out = c + static_cast<uint64_t>(tile_m) * NT * n + tile_n * kTileN + row;
      if (tile_n * kTileN + row < n) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
          if (static_cast<uint32_t>(j) < held) out[static_cast<uint64_t>(j) * n] = Elem<T>::from_float(sum(j));
      }
    } else {
      // Every copy has landed and every product has read it: the ring is free.
      float *const part = reinterpret_cast<float *>(ring);
#pragma unroll
      for (int j = 0; j < NT; ++j)
        if (static_cast<uint32_t>(j) < held) part[j * kTileN + row] = sum(j);
    }
  }
  tc_fence_before();
  if (split == 1) {
    __syncthreads();
  } else {
    cluster_sync();
    // Four outputs of one row a thread, the blocks' sums added in their order.
    uint32_t from[8];
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) from[q] = cluster_addr(ring, min(q, split - 1));
    for (uint32_t i = rank * kSkinnyThreads + threadIdx.x; i < held * (kTileN / 4); i += split * kSkinnyThreads) {
      float4 v[8];
#pragma unroll
      for (uint32_t q = 0; q < 8; ++q)
        if (q < split)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v[q].x), "=f"(v[q].y), "=f"(v[q].z), "=f"(v[q].w)
                       : "r"(from[q] + 16 * i)
                       : "memory");
      float4 total = v[0];
#pragma unroll
      for (uint32_t q = 1; q < 8; ++q)
        if (q < split) total.x += v[q].x, total.y += v[q].y, total.z += v[q].z, total.w += v[q].w;
      const uint32_t j = i / (kTileN / 4), col = tile_n * kTileN + 4 * (i % (kTileN / 4));
      T *const out = c + (static_cast<uint64_t>(tile_m) * NT + j) * n + col;
      const T r[4] = {Elem<T>::from_float(total.x), Elem<T>::from_float(total.y), Elem<T>::from_float(total.z), Elem<T>::from_float(total.w)};
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e)
        if (col + e < n) out[e] = r[e];
    }
    cluster_sync();  // no block leaves while another reads its sums
  }
  if (threadIdx.x == 0 && failed) atomicOr(&g_fp8_error, kErrTimeout);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc1(tmem, S::kColumns);
  }
}

// Blocks that share a tile's groups: as many as can be resident at once for all tiles, two an SM. A second wave of smaller shares
// costs more than it brings: 16 x 24576 x 4096 (192 tiles) 19 us unsplit, 25 and 31 in two and three; 1 x 6144 x 4096
// (48) 13.1 unsplit, 8.7, 7.9, 6.9 and 6.6 in two to five, where six no longer fit the GPCs: 10.6.
template <typename Kernel>
uint32_t pick_split(Kernel kernel, int kind, cudaLaunchConfig_t cfg, uint64_t tiles, uint32_t groups) {
  static std::mutex mutex;
  static int resident[6][64][9] = {};  // clusters of each size at once, an SM having one block: 0 not known yet, -1 none
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return 1;
  std::lock_guard<std::mutex> lock(mutex);
  for (uint32_t split = std::min(8u, groups); split > 1; --split) {
    int &clusters = resident[kind][device & 63][split];
    if (clusters == 0) {
      cfg.gridDim = dim3(split);
      cfg.attrs[1].val.clusterDim.x = split;
      cfg.numAttrs = 2;
      if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess || clusters <= 0) clusters = -1;
    }
    if (clusters > 0 && tiles <= static_cast<uint64_t>(clusters) * kSkinnyBlocks) return split;
  }
  return 1;
}

template <typename T, int NT>
cudaError_t skinny_launch(const Fp8Product &p, cudaStream_t s) {
  using S = Skinny<NT>;
  CUtensorMap map_w, map_a;
  cudaError_t e = make_tmap_2d_u8_swizzled(&map_w, p.w, p.k, p.n, kTileN);
  if (e == cudaSuccess) e = make_tmap_2d_u8_swizzled(&map_a, p.a, p.k, p.m, NT);
  const auto kernel = k_skinny<T, NT>;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  const uint32_t groups = (p.k + kGroup - 1) / kGroup;
  const uint64_t tiles = static_cast<uint64_t>((p.n + kTileN - 1) / kTileN) * ((p.m + NT - 1) / NT);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.blockDim = dim3(kSkinnyThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.attrs = attr;
  const int kind = (NT == 16 ? 0 : NT == 32 ? 1 : 2) + (std::is_same<T, __half>::value ? 3 : 0);
  const uint32_t split = pick_split(kernel, kind, cfg, tiles, groups);
  if (tiles * split >= (1ull << 31)) return cudaErrorInvalidConfiguration;
  attr[1].val.clusterDim.x = split;
  cfg.gridDim = dim3(static_cast<uint32_t>(tiles) * split);
  cfg.stream = s;
  cfg.numAttrs = split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, map_w, map_a, p.a_scales, p.w_scales, static_cast<T *>(p.c), p.m, p.n, groups, split);
}

// --------------------------------------------------------------- many rows ----

constexpr uint32_t kPair = 256;                     // rows and columns of a pair's tile
constexpr uint32_t kWideStages = 4, kWideStage = 2 * kTileBytes;
constexpr uint32_t kSumWarps = 8, kWideThreads = 128 + 32 * kSumWarps;
constexpr uint32_t kOutBox = 32 * 128;              // bytes of 32 rows x 64 outputs, swizzled; two a warp
constexpr uint32_t kScaleGroups = 4;                // groups whose scales are handed over at once, twice
constexpr uint32_t kScalesAt = kWideStages * kWideStage + kSumWarps * 2 * kOutBox;
constexpr uint32_t kWideSmem = 1024 + kScalesAt + 2 * kScaleGroups * kPair * 4;
constexpr uint32_t kGroupRows = 8;                  // tile rows whose tiles follow one another, for the L2; 16 is no faster, 4 3% slower

// Into this block's shared memory, completing on the even block's barrier.
__device__ __forceinline__ void tma_load_pair(void *dst, const CUtensorMap *map, int32_t x, int32_t y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void mma2_f8(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrives on the barrier of this offset in both blocks when the products issued so far are done.
__device__ __forceinline__ void mma2_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}

struct WideTile {
  uint32_t m, n;
};

__device__ __forceinline__ WideTile wide_tile(uint32_t t, uint32_t tiles_m, uint32_t tiles_n) {
  const uint32_t in_group = kGroupRows * tiles_n, group = t / in_group, first = group * kGroupRows;
  const uint32_t rows = min(kGroupRows, tiles_m - first), local = t - group * in_group;
  return {first + local % rows, local / rows};
}

// Warp 0 loads, warp 1 (of the even block) issues the products, warps 2 and 3 bring the scales, warps 4 to 11 add up and have
// most of the registers. TMA_OUT: rows of c are 16-byte aligned.
//
// The sums of a group can only be taken out of TMEM when they are complete, and TMEM holds two groups: a group's time is half of
// its products (512 cycles) and of the way round: their completion seen (200), 128 columns read and added up (450), the buffer
// known to be free (150), the next products issued. So the loop of the adding warps has little in it that can stand elsewhere:
// another pair of warps multiplies the scales of row and block ahead of their use and hands over four groups at a time, through
// barriers of this block alone; from there on the adding warps hold them in registers. The issuing warp stays converged and an
// elected lane issues, so that operands are in uniform registers: from one lane's branch a group took 1.3 times as long.
template <typename T, bool TMA_OUT>
__global__ void __launch_bounds__(kWideThreads, 1)
k_wide(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_c,
       const float *a_scales, const float *w_scales, T *c, uint32_t m, uint32_t n, uint32_t groups) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t full[kWideStages], empty[kWideStages], sum_full[2], sum_empty[2], scale_full[2], scale_empty[2], drain;
  __shared__ uint32_t tmem_base;
  __shared__ int failed;
  const uint32_t a0 = smem_addr(smem_raw);
  uint8_t *const ring = smem_raw + ((a0 + 1023u) / 1024u * 1024u - a0);
  float *const scales = reinterpret_cast<float *>(ring + kScalesAt);  // [half of the places][group of four][column half][row]
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const uint32_t tiles_m = (m + kPair - 1) / kPair, tiles_n = (n + kPair - 1) / kPair, tiles = tiles_m * tiles_n;

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < kWideStages; ++i) {
      mbar_init(&full[i], 1);  // the even block's, for both blocks' operands
      mbar_init(&empty[i], 1);
    }
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(&sum_full[i], 1);
      mbar_init(&sum_empty[i], 2 * kSumWarps);
      mbar_init(&scale_full[i], 2);
      mbar_init(&scale_empty[i], kSumWarps);
    }
    mbar_init(&drain, 1);
    fence_mbar_init();
    failed = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  grid_dep_launch();
  grid_dep_wait();

  const uint32_t full_bars = cluster_addr(&full[0], 0);
  // 384 threads x 168 registers at launch = 128 x 72 + 256 x 216.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      if (lane == 0) {
        uint32_t i = 0;
        for (uint32_t t = pair; t < tiles && !has_failed(&failed); t += pairs) {
          const WideTile tile = wide_tile(t, tiles_m, tiles_n);
          const int32_t ya = static_cast<int32_t>(tile.m * kPair + rank * 128), yw = static_cast<int32_t>(tile.n * kPair + rank * 128);
          for (uint32_t g = 0; g < groups; ++g, ++i) {
            const uint32_t s = i % kWideStages, use = i / kWideStages;
            if (use > 0 && !mbar_wait(&empty[s], (use - 1) & 1)) { failed = 1; break; }
            if (rank == 0) mbar_expect_tx(&full[s], 2 * kWideStage);
            uint8_t *const st = ring + s * kWideStage;
            tma_load_pair(st, &map_a, static_cast<int32_t>(g * kGroup), ya, full_bars + 8 * s);
            tma_load_pair(st + kTileBytes, &map_w, static_cast<int32_t>(g * kGroup), yw, full_bars + 8 * s);
          }
        }
        if (has_failed(&failed) && rank == 0)  // no copy may land once this shared memory is another block's
          for (uint32_t back = 0; back < kWideStages && back < i; ++back)
            mbar_wait(&full[(i - 1 - back) % kWideStages], (i - 1 - back) / kWideStages & 1);
        // The products' last arrivals in this block, before it leaves with its barriers.
        for (uint32_t back = min(i, kWideStages); back > 0 && !has_failed(&failed); --back)
          if (!mbar_wait(&empty[(i - back) % kWideStages], (i - back) / kWideStages & 1)) failed = 1;
        if (!mbar_wait(&drain, 0)) failed = 1;
      }
    } else if (warp == 1) {
      if (rank == 0) {
        constexpr uint32_t idesc = instr_desc(kPair, kPair);
        uint32_t i = 0;
        bool ok = true;
        for (uint32_t t = pair; ok && t < tiles; t += pairs) {
          for (uint32_t g = 0; g < groups; ++g, ++i) {
            const uint32_t s = i % kWideStages, b = i & 1, use = i >> 1;
            if (!(ok = warp_wait(&failed, &full[s], i / kWideStages & 1))) break;
            if (!(ok = use == 0 || warp_wait(&failed, &sum_empty[b], (use - 1) & 1))) break;
            tc_fence_after();
            const uint32_t st = smem_addr(ring + s * kWideStage);
            const uint64_t da = smem_desc(st, 16, 1024), dw = smem_desc(st + kTileBytes, 16, 1024);
            if (elect_one()) {
#pragma unroll
              for (uint32_t kk = 0; kk < 4; ++kk) mma2_f8(tmem + b * kPair, da + 2 * kk, dw + 2 * kk, idesc, kk != 0);
              mma2_commit(&empty[s]);
              mma2_commit(&sum_full[b]);
            }
            __syncwarp();
          }
        }
        if (elect_one()) mma2_commit(&drain);
        warp_wait(&failed, &drain, 0);
      }
    } else {
      const uint32_t half = warp - 2;
      uint32_t chunk = 0;  // of four groups, of all tiles
      bool ok = true;
      for (uint32_t t = pair; ok && t < tiles; t += pairs) {
        const WideTile tile = wide_tile(t, tiles_m, tiles_n);
        const uint32_t row0 = tile.m * kPair + rank * 128 + lane, block = tile.n * 2 + half;
        const bool real = block * kGroup < n;
        const float *const sw = w_scales + static_cast<uint64_t>(block) * groups;
        float row_scale[kScaleGroups][4], block_scale[kScaleGroups];  // on their way; 0 behind the last group
        const auto bring = [&](uint32_t g, uint32_t at) {
          block_scale[at] = real && g < groups ? ld_f32(sw + g) : 0.f;
#pragma unroll
          for (uint32_t q = 0; q < 4; ++q)
            row_scale[at][q] = real && g < groups && row0 + 32 * q < m ? ld_f32(a_scales + static_cast<uint64_t>(g) * m + row0 + 32 * q) : 0.f;
        };
#pragma unroll
        for (uint32_t at = 0; at < kScaleGroups; ++at) bring(at, at);
        for (uint32_t g0 = 0; g0 < groups; g0 += kScaleGroups, ++chunk) {
          if (!(ok = chunk < 2 || warp_wait(&failed, &scale_empty[chunk & 1], ((chunk >> 1) - 1) & 1))) break;
          float *const place = scales + (chunk & 1) * kScaleGroups * kPair + half * 128 + lane;
#pragma unroll
          for (uint32_t at = 0; at < kScaleGroups; ++at) {
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q) place[at * kPair + 32 * q] = row_scale[at][q] * block_scale[at];
            bring(g0 + kScaleGroups + at, at);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&scale_full[chunk & 1]);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const uint32_t quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t release = cluster_addr(&sum_empty[0], 0), taddr = tmem + (quarter * 32u << 16) + half * 128;
    const uint32_t scale_at = smem_addr(scales + half * 128 + quarter * 32 + lane);
    uint8_t *const stage = ring + kWideStages * kWideStage + (warp - 4) * 2 * kOutBox;
    bool ok = true;  // a warp that gives up goes on without waiting, to the end of its tile
    uint32_t i = 0, chunk = 0;
    for (uint32_t t = pair; t < tiles; t += pairs) {
      if (__any_sync(kFullMask, has_failed(&failed))) break;
      const WideTile tile = wide_tile(t, tiles_m, tiles_n);
      const uint32_t row0 = tile.m * kPair + rank * 128 + quarter * 32, col0 = tile.n * kPair + half * 128;
      uint64_t sums[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) sums[j] = 0;
      uint32_t held[kScaleGroups];  // this row's scales of the next groups
      for (uint32_t g = 0; g < groups; ++g, ++i) {
        const uint32_t b = i & 1;
        if (g % kScaleGroups == 0) {
          if (ok && !mbar_wait(&scale_full[chunk & 1], chunk >> 1 & 1)) failed = 1, ok = false;
#pragma unroll
          for (uint32_t at = 0; at < kScaleGroups; ++at)
            asm volatile("ld.shared.b32 %0, [%1];"
                         : "=r"(held[at])
                         : "r"(scale_at + ((chunk & 1) * kScaleGroups + at) * (kPair * 4))
                         : "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&scale_empty[chunk & 1]);
          ++chunk;
        }
        const uint32_t scale = held[0];
#pragma unroll
        for (uint32_t at = 0; at + 1 < kScaleGroups; ++at) held[at] = held[at + 1];
        if (ok && !mbar_wait(&sum_full[b], i >> 1 & 1)) failed = 1, ok = false;
        __syncwarp();
        tc_fence_after();
        uint32_t d[2][16];
        tmem_ld16_nowait(taddr + b * kPair, d[0]);
        const uint64_t both = static_cast<uint64_t>(scale) << 32 | scale;
#pragma unroll
        for (int piece = 0; piece < 8; ++piece) {
          uint32_t(&now)[16] = d[piece & 1];
          tmem_landed(now);
          if (piece < 7) {
            tmem_ld16_nowait(taddr + b * kPair + 16 * (piece + 1), d[(piece + 1) & 1]);
          } else {  // all read: the products after next may overwrite them
            tc_fence_before();
            __syncwarp();
            if (lane == 0) pair_arrive(release + 8 * b);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) fma2(sums[8 * piece + j], now[2 * j], now[2 * j + 1], both);
        }
      }
      if (row0 >= m || col0 >= n) continue;
      if (TMA_OUT) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the last tile has left
        __syncwarp();
      }
#pragma unroll
      for (uint32_t j = 0; j < 16; ++j) {
        const uint4 v = make_uint4(pack2<T>(sums[4 * j]), pack2<T>(sums[4 * j + 1]), pack2<T>(sums[4 * j + 2]), pack2<T>(sums[4 * j + 3]));
        *reinterpret_cast<uint4 *>(stage + j / 8 * kOutBox + lane * 128 + ((j % 8 ^ (lane & 7)) * 16)) = v;
      }
      if (TMA_OUT) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
#pragma unroll
          for (uint32_t box = 0; box < 2; ++box)
            if (col0 + 64 * box < n)
              asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(&map_c),
                           "r"(static_cast<int32_t>(col0 + 64 * box)), "r"(static_cast<int32_t>(row0)), "r"(smem_addr(stage + box * kOutBox))
                           : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      } else {
        __syncwarp();
        const uint32_t rows = min(32u, m - row0);
        for (uint32_t r = 0; r < rows; ++r)
#pragma unroll
          for (uint32_t q = 0; q < 4; ++q) {
            const uint32_t col = 32 * q + lane, in = col % 64;
            if (col0 + col < n)
              c[static_cast<uint64_t>(row0 + r) * n + col0 + col] =
                  *reinterpret_cast<const T *>(stage + col / 64 * kOutBox + r * 128 + ((in / 8 ^ (r & 7)) * 16) + in % 8 * 2);
          }
        __syncwarp();
      }
    }
    if (TMA_OUT && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && failed) atomicOr(&g_fp8_error, kErrTimeout);
  cluster_sync();  // neither block touches the other's barriers, shared memory or TMEM after this
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  cluster_sync();
}

template <typename T>
cudaError_t wide_launch(const Fp8Product &p, cudaStream_t s) {
  const bool tma_out = p.n % 8 == 0;
  CUtensorMap map_a, map_w, map_c;
  cudaError_t e = make_tmap_2d_u8_swizzled(&map_a, p.a, p.k, p.m, 128);
  if (e == cudaSuccess) e = make_tmap_2d_u8_swizzled(&map_w, p.w, p.k, p.n, 128);
  map_c = map_a;
  if (e == cudaSuccess && tma_out) e = make_tmap_2d_u16_swizzled(&map_c, p.c, p.n, p.m, p.n, 64, 32);
  const auto kernel = tma_out ? k_wide<T, true> : k_wide<T, false>;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kWideSmem);
  if (e != cudaSuccess) return e;
  const uint64_t tiles = static_cast<uint64_t>((p.m + kPair - 1) / kPair) * ((p.n + kPair - 1) / kPair);
  if (tiles >= (1ull << 31)) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  // The pairs do not wait for one another: any number of them is right.
  cfg.gridDim = dim3(2 * static_cast<uint32_t>(std::min<uint64_t>(tiles, sm_count() / 2)));
  cfg.blockDim = dim3(kWideThreads);
  cfg.dynamicSmemBytes = kWideSmem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, map_a, map_w, map_c, p.a_scales, p.w_scales, static_cast<T *>(p.c), p.m, p.n,
                            (p.k + kGroup - 1) / kGroup);
}

// k_skinny with 64 rows a tile takes 0.31 us for a group of as many tiles as there are SMs, k_wide 0.4 us for one of half as many
// of its tiles, whether there are that many or not: 128 x 4096 x 12288 17.8 and 46 us, 300 x 4096 x 4096 20.0 and
// 19.2, 256 x 24576 x 4096 57 and 39.
bool is_wide(const Fp8Product &p) {
  const uint64_t sms = sm_count(), small = static_cast<uint64_t>((p.n + kTileN - 1) / kTileN) * ((p.m + 63) / 64);
  const uint64_t large = static_cast<uint64_t>((p.n + kPair - 1) / kPair) * ((p.m + kPair - 1) / kPair);
  const uint64_t rounds = (large + sms / 2 - 1) / (sms / 2);
  return 4 * small >= 5 * sms * rounds;
}

template <typename T>
cudaError_t product_launch(const Fp8Product &p, cudaStream_t s) {
  if (p.m <= 16) return skinny_launch<T, 16>(p, s);
  if (p.m <= 32) return skinny_launch<T, 32>(p, s);
  return p.m > 64 && is_wide(p) ? wide_launch<T>(p, s) : skinny_launch<T, 64>(p, s);
}

}  // namespace

cudaError_t fp8_gemm_launch(bool fp16, const Fp8Product &p, cudaStream_t s) {
  return fp16 ? product_launch<__half>(p, s) : product_launch<__nv_bfloat16>(p, s);
}

unsigned take_fp8_error() {
  unsigned v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_fp8_error, sizeof(v)) != cudaSuccess) return 0;
  if (v) cudaMemcpyToSymbol(g_fp8_error, &zero, sizeof(zero));
  return v;
}

}  // namespace xpu
