// Product of 8-bit rows with 8-bit weights (xpu_fp8_gemm in include/xpu_cuda.h):
//
//   c[m][n] = sum_g sa[g][m] sw[n / 128][g] sum_{k in g} a[m][k] w[n][k]
//
// over the groups g of 128 columns, FP32 sums.
#include <cuda_fp8.h>

#include "common.cuh"
#include "serving.h"
#include "stream.cuh"

namespace xpu {
namespace {

constexpr uint32_t kGroup = XPU_FP8_BLOCK;

__device__ __forceinline__ float widen(uint8_t v) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)));
}

// 32 x 32 outputs a block through shared memory, four rows a thread.
template <typename T>
__global__ void __launch_bounds__(256) k_fp8_gemm_simple(const uint8_t *a, const float *a_scales, const uint8_t *w,
                                                         const float *w_scales, T *c, uint32_t m, uint32_t n, uint32_t k) {
  __shared__ float as[32][33], ws[32][33];
  grid_dep_launch();
  grid_dep_wait();
  const uint32_t tx = threadIdx.x % 32, ty = threadIdx.x / 32, groups = (k + kGroup - 1) / kGroup;
  const uint32_t across = (n + 31) / 32, row0 = blockIdx.x / across * 32, col0 = blockIdx.x % across * 32, col = col0 + tx;
  float total[4] = {};
  for (uint32_t g = 0; g < groups; ++g) {
    float sum[4] = {};
    for (uint32_t k0 = g * kGroup; k0 < min(k, (g + 1) * kGroup); k0 += 32) {
      __syncthreads();
      for (uint32_t i = ty; i < 32; i += 8) {
        as[i][tx] = row0 + i < m && k0 + tx < k ? widen(a[static_cast<size_t>(row0 + i) * k + k0 + tx]) : 0.f;
        ws[i][tx] = col0 + i < n && k0 + tx < k ? widen(w[static_cast<size_t>(col0 + i) * k + k0 + tx]) : 0.f;
      }
      __syncthreads();
#pragma unroll 8
      for (uint32_t kk = 0; kk < 32; ++kk)
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) sum[j] = fmaf(as[ty + 8 * j][kk], ws[tx][kk], sum[j]);
    }
    if (col >= n) continue;
    const float sw = w_scales[static_cast<size_t>(col / kGroup) * groups + g];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const uint32_t row = row0 + ty + 8 * j;
      if (row < m) total[j] = fmaf(sum[j], a_scales[static_cast<size_t>(g) * m + row] * sw, total[j]);
    }
  }
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    const uint32_t row = row0 + ty + 8 * j;
    if (row < m && col < n) c[static_cast<size_t>(row) * n + col] = Elem<T>::from_float(total[j]);
  }
}

}  // namespace

cudaError_t fp8_gemm_launch(bool fp16, const Fp8Product &p, cudaStream_t s) {
  const uint64_t blocks = static_cast<uint64_t>((p.m + 31) / 32) * ((p.n + 31) / 32);
  if (blocks >= (1ull << 31)) return cudaErrorInvalidConfiguration;
  const auto go = [&](auto kernel, auto *c) {
    return launch_after(kernel, static_cast<uint32_t>(blocks), 256, 0, s, p.a, p.a_scales, p.w, p.w_scales, c, p.m, p.n, p.k);
  };
  return fp16 ? go(k_fp8_gemm_simple<__half>, static_cast<__half *>(p.c))
              : go(k_fp8_gemm_simple<__nv_bfloat16>, static_cast<__nv_bfloat16 *>(p.c));
}

}  // namespace xpu
