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
// tile and add their sums up through distributed shared memory, in a fixed order.
#include <cuda.h>

#include <algorithm>

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

// A float that the kernel before may have written.
__device__ __forceinline__ float ld_f32(const float *p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}

// ---------------------------------------------------------------- few rows ----

template <int NT>
struct Skinny {
  static constexpr uint32_t kBuffers = NT <= 64 ? 4 : 2, kColumns = NT * kBuffers;
  static constexpr uint32_t kStageBytes = kTileBytes + NT * kGroup;
  static constexpr uint32_t kStages = NT <= 32 ? 5 : NT == 64 ? 4 : 3;  // two blocks an SM
  static constexpr uint32_t kChunk = 8;                                 // groups whose scales are held
  static constexpr uint32_t kScales = 2 * kChunk * NT;
  static constexpr uint32_t kSmem = 1024 + kStages * kStageBytes + 4 * kScales;
  static_assert(NT * kTileN * 4 <= kStages * kStageBytes, "the sums of a tile take the ring's place");
};
constexpr uint32_t kSkinnyThreads = 192;

// Warp 0 loads, warp 1 issues the products, warps 2 to 5 add up: a thread has one row of w and NT sums.
template <typename T, int NT>
__global__ void __launch_bounds__(kSkinnyThreads, 2)
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
  if (warp == 1) tmem_alloc1(&tmem_base, S::kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  grid_dep_launch();  // with the TMEM held: a block of the next kernel cannot take it from one of this
  grid_dep_wait();

  float sums[NT];
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
    if (lane == 0) {
      constexpr uint32_t idesc = instr_desc(kTileN, NT);
      for (uint32_t i = 0; i < count && !has_failed(&failed); ++i) {
        const uint32_t s = i % S::kStages, b = i % S::kBuffers, use = i / S::kBuffers;
        if (use > 0 && !mbar_wait(&sum_empty[b], (use - 1) & 1)) { failed = 1; break; }
        if (!mbar_wait(&full[s], i / S::kStages & 1)) { failed = 1; break; }
        tc_fence_after();
        const uint32_t st = smem_addr(ring + s * S::kStageBytes);
        const uint64_t dw = smem_desc(st, 16, 1024), da = smem_desc(st + kTileBytes, 16, 1024);
#pragma unroll
        for (uint32_t kk = 0; kk < 4; ++kk) mma1_f8(tmem + b * NT, dw + 2 * kk, da + 2 * kk, idesc, kk != 0);
        mma1_commit(&empty[s]);
        mma1_commit(&sum_full[b]);
      }
      mma1_commit(&drain);
      if (!mbar_wait(&drain, 0)) failed = 1;
    }
  } else {
    const uint32_t et = threadIdx.x - 64;
#pragma unroll
    for (int j = 0; j < NT; ++j) sums[j] = 0.f;
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
      const float4 *const by = reinterpret_cast<const float4 *>(chunk + i % S::kChunk * NT);
#pragma unroll
      for (int at = 0; at < NT; at += 16) {
        float d[16];
        tmem_ld16(tmem + ((warp & 3) * 32u << 16) + b * NT + at, d);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 s = by[at / 4 + q];
          sums[at + 4 * q] = fmaf(d[4 * q], s.x, sums[at + 4 * q]);
          sums[at + 4 * q + 1] = fmaf(d[4 * q + 1], s.y, sums[at + 4 * q + 1]);
          sums[at + 4 * q + 2] = fmaf(d[4 * q + 2], s.z, sums[at + 4 * q + 2]);
          sums[at + 4 * q + 3] = fmaf(d[4 * q + 3], s.w, sums[at + 4 * q + 3]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sum_empty[b]);
    }
    T *const out = c + static_cast<uint64_t>(tile_m) * NT * n + tile_n * kTileN + row;
    if (split == 1) {
      if (tile_n * kTileN + row < n) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
          if (static_cast<uint32_t>(j) < held) out[static_cast<uint64_t>(j) * n] = Elem<T>::from_float(sums[j]);
      }
    } else {
      // Every copy has landed and every product has read it: the ring is free.
      float *const part = reinterpret_cast<float *>(ring);
#pragma unroll
      for (int j = 0; j < NT; ++j)
        if (static_cast<uint32_t>(j) < held) part[j * kTileN + row] = sums[j];
    }
  }
  tc_fence_before();
  if (split == 1) {
    __syncthreads();
  } else {
    cluster_sync();
    if (threadIdx.x >= 64 && tile_n * kTileN + row < n) {  // rank r adds up rows r, r + split, .. of a
      for (uint32_t j = rank; j < held; j += split) {
        float total = 0.f;
        for (uint32_t q = 0; q < split; ++q) {
          float v;
          asm volatile("ld.shared::cluster.f32 %0, [%1];"
                       : "=f"(v)
                       : "r"(cluster_addr(reinterpret_cast<float *>(ring) + j * kTileN + row, q))
                       : "memory");
          total += v;
        }
        c[(static_cast<uint64_t>(tile_m) * NT + j) * n + tile_n * kTileN + row] = Elem<T>::from_float(total);
      }
    }
    cluster_sync();  // no block leaves while another reads its sums
  }
  if (threadIdx.x == 0 && failed) atomicOr(&g_fp8_error, kErrTimeout);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc1(tmem, S::kColumns);
  }
}

// Blocks that share a tile's groups. Time in groups that one SM reads: a block's share, and about four for beginning and
// ending; two blocks an SM share its bandwidth.
uint32_t pick_split(uint64_t tiles, uint32_t groups) {
  const uint64_t slots = 2ull * sm_count();
  uint32_t best = 1;
  uint64_t least = UINT64_MAX;
  for (uint32_t split = 1; split <= std::min(8u, groups); ++split) {
    const uint64_t waves = (tiles * split + slots - 1) / slots, share = (groups + split - 1) / split;
    const uint64_t cost = waves * (2 * share + 4);
    if (cost < least) {
      least = cost;
      best = split;
    }
  }
  return best;
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
  const uint32_t split = pick_split(tiles, groups);
  if (tiles * split >= (1ull << 31)) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<uint32_t>(tiles) * split);
  cfg.blockDim = dim3(kSkinnyThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, map_w, map_a, p.a_scales, p.w_scales, static_cast<T *>(p.c), p.m, p.n, groups, split);
}

template <typename T>
cudaError_t product_launch(const Fp8Product &p, cudaStream_t s) {
  if (p.m <= 16) return skinny_launch<T, 16>(p, s);
  if (p.m <= 32) return skinny_launch<T, 32>(p, s);
  if (p.m <= 64) return skinny_launch<T, 64>(p, s);
  return skinny_launch<T, 128>(p, s);
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
