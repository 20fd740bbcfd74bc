// Rows that enter an 8-bit product (xpu_fp8_quantize, xpu_fp8_silu_multiply and
// xpu_fp8_rms_norm in include/xpu_cuda.h): each 128 columns of a row get the
// scale s = max(max |y| / 448, 2^-126) and leave as e4m3(y / s).
//
// All of it is bound by memory. Sixteen lanes hold one group of 128 columns, eight
// each (a 16-byte load, an 8-byte store), and find its largest value with four
// shuffles. The floor of 2^-126 keeps 1 / s finite, so that a group of zeros
// needs no case of its own. NaN and infinities pass on: their group's products
// are NaN.
#include <cuda_fp8.h>

#include "common.cuh"
#include "serving.h"
#include "stream.cuh"

namespace xpu {
namespace {

constexpr uint32_t kGroup = XPU_FP8_BLOCK, kLanes = kGroup / 8;  // lanes of a group
constexpr uint32_t kHalves = 16;                        // half warps a block
__host__ __device__ constexpr uint32_t at_once(bool gated) { return gated ? 2 : 3; }  // groups a half warp takes at once
constexpr float kLargest = 448.f, kSmallestScale = 1.17549435e-38f;

// 16 bytes of a row that is read once, behind the wait for the kernel before.
__device__ __forceinline__ uint4 ld_once(const uint16_t *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ void widen(const uint4 &v, float (&y)[8]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[2 * i] = Elem<T>::lo(u[i]);
    y[2 * i + 1] = Elem<T>::hi(u[i]);
  }
}

// Two FP32 values rounded to T, side by side.
template <typename T>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t narrow2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <>
__device__ __forceinline__ uint32_t narrow2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// The special function unit's reciprocal and power of two, off by 2^-23 and 2^-22; subnormal numbers are 0.
__device__ __forceinline__ float fast_reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Scale and 8-bit values of a group that 16 lanes hold, 8 columns each. The instructions bound these kernels beside the memory
// (24 a value with true divisions), so the scale is a product with 1 / 448, within 2^-23 of the quotient, and a value a product
// with the scale's fast reciprocal, within 2^-22 of its quotient; e4m3 keeps 2^-4.
__device__ __forceinline__ float encode(const float (&y)[8], uint2 *q) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(y[i]));
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
  const float scale = fmaxf(top * (1.f / kLargest), kSmallestScale), inverse = fast_reciprocal(scale);
  uint32_t half[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    half[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i] * inverse, y[2 * i + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
  *q = make_uint2(half[0] | half[1] << 16, half[2] | half[3] << 16);
  return scale;
}

// ------------------------------------------------- plain and gated rows ----

// silu(g) u = g u / (1 + 2^(-g log2 e)). The exponent's rounding is 2^-24 of itself, so results are within 2^-16 down to g =
// -87, below which 1 + 2^x passes 2^126 and its reciprocal is 0: then so is the result, less than 1e-36 u.
__device__ __forceinline__ float gated(float g, float u) { return g * fast_reciprocal(1.f + fast_exp2(g * -1.4426950408889634f)) * u; }

// A half warp takes kAtOnce groups, so that as many loads are in flight, a block 16 kAtOnce in the order of rows and columns.
// 8192 x 12288 gated: fp16 80 us (6.3 TB/s), bf16 83; 84 with three groups, 85 with four, 99 with one; 114 with a loop over
// resident blocks, whose last turn leaves some idle. Plain 8192 x 4096: 17.6 us (5.7 TB/s, from the L2 in part).
// Blocks of 16 rows, whose scales are side by side, were no faster.
template <typename T, bool GATED>
__global__ void __launch_bounds__(16 * kHalves) k_fp8_rows(const uint16_t *x, const uint16_t *up, uint64_t stride, uint8_t *q,
                                                  float *scales, uint32_t rows, uint32_t width) {
  constexpr uint32_t kAtOnce = at_once(GATED);
  grid_dep_launch();
  grid_dep_wait();
  const uint32_t groups = (width + kGroup - 1) / kGroup, lane = threadIdx.x % kLanes, half = threadIdx.x / kLanes;
  const uint32_t first = blockIdx.x * (kAtOnce * kHalves), row0 = first / groups, group0 = first - row0 * groups;
  uint4 a[kAtOnce], b[kAtOnce];
  uint32_t row[kAtOnce], group[kAtOnce];
  bool inside[kAtOnce];
#pragma unroll
  for (uint32_t i = 0; i < kAtOnce; ++i) {
    row[i] = row0;
    group[i] = group0 + i * kHalves + half;
    if (group[i] >= groups) {
      const uint32_t over = group[i] / groups;
      row[i] += over;
      group[i] -= over * groups;
    }
    const uint32_t column = group[i] * kGroup + 8 * lane;
    inside[i] = row[i] < rows && column < width;
    a[i] = b[i] = make_uint4(0, 0, 0, 0);
    if (inside[i]) {
      a[i] = ld_once(x + row[i] * stride + column);
      if (GATED) b[i] = ld_once(up + row[i] * stride + column);
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < kAtOnce; ++i) {
    float y[8];
    widen<T>(a[i], y);
    if (GATED) {
      float u[8];
      widen<T>(b[i], u);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = gated(y[j], u[j]);
    }
    uint2 packed;
    const float scale = encode(y, &packed);
    if (inside[i]) {
      *reinterpret_cast<uint2 *>(q + static_cast<uint64_t>(row[i]) * width + group[i] * kGroup + 8 * lane) = packed;
      if (lane == 0) scales[static_cast<uint64_t>(group[i]) * rows + row[i]] = scale;
    }
  }
}

// ------------------------------------------------------------------ norm ----

// One block a row, CHUNKS pieces of 8 columns a thread. The sum x + residual is rounded to T, as the stream is held,
// and the norm is that of the rounded sum; squares and their mean are FP32 in a fixed order.
template <typename T, int CHUNKS>
__global__ void __launch_bounds__(1024) k_fp8_rms_norm(const uint16_t *x, uint64_t x_stride, const uint16_t *residual,
                                                       uint64_t residual_stride, const uint16_t *weight, uint16_t *total,
                                                       uint64_t total_stride, uint8_t *q, float *scales, uint32_t rows,
                                                       uint32_t width, float epsilon) {
  __shared__ float sums[32];
  grid_dep_launch();
  grid_dep_wait();
  const uint32_t row = blockIdx.x, warps = blockDim.x / 32;
  uint4 t[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const uint32_t column = 8 * (c * blockDim.x + threadIdx.x);
    t[c] = make_uint4(0, 0, 0, 0);
    if (column < width) t[c] = ld_once(x + row * x_stride + column);
  }
  if (residual) {
    uint4 r[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const uint32_t column = 8 * (c * blockDim.x + threadIdx.x);
      r[c] = make_uint4(0, 0, 0, 0);
      if (column < width) r[c] = ld_once(residual + row * residual_stride + column);
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      float a[8], b[8];
      widen<T>(t[c], a);
      widen<T>(r[c], b);
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u[i] = narrow2<T>(a[2 * i] + b[2 * i], a[2 * i + 1] + b[2 * i + 1]);
      }
      t[c] = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
  uint4 scale_by[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const uint32_t column = 8 * (c * blockDim.x + threadIdx.x);
    scale_by[c] = make_uint4(0, 0, 0, 0);
    if (column < width) scale_by[c] = *reinterpret_cast<const uint4 *>(weight + column);
  }
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const uint32_t column = 8 * (c * blockDim.x + threadIdx.x);
    if (total && column < width) *reinterpret_cast<uint4 *>(total + row * total_stride + column) = t[c];
    float y[8];
    widen<T>(t[c], y);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(y[i], y[i], sum);
  }
  sum = warp_sum(sum);
  if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = sum;
  __syncthreads();
  sum = threadIdx.x % 32 < warps ? sums[threadIdx.x % 32] : 0.f;
  const float factor = exact_rsqrt(warp_sum(sum) / static_cast<float>(width) + epsilon);
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const uint32_t column = 8 * (c * blockDim.x + threadIdx.x);
    float y[8], w[8];  // zeros behind the last column
    widen<T>(t[c], y);
    widen<T>(scale_by[c], w);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = y[i] * factor * w[i];
    uint2 packed;
    const float scale = encode(y, &packed);
    if (column < width) {
      *reinterpret_cast<uint2 *>(q + static_cast<uint64_t>(row) * width + column) = packed;
      if (threadIdx.x % kLanes == 0) scales[static_cast<uint64_t>(column / kGroup) * rows + row] = scale;
    }
  }
}

template <typename T>
cudaError_t norm_launch(const Fp8Norm &n, cudaStream_t s) {
  const uint32_t pieces = n.width / 8;
  const auto threads = [&](uint32_t chunks) { return (pieces + 32 * chunks - 1) / (32 * chunks) * 32; };
  const auto go = [&](auto kernel, uint32_t chunks) {
    return launch_after(kernel, n.rows, threads(chunks), 0, s, n.x, n.x_stride, n.residual, n.residual_stride, n.weight, n.total,
                        n.total_stride, n.q, n.scales, n.rows, n.width, n.epsilon);
  };
  // Few rows: the most threads, for the latency (64 x 4096 2.5 us, 2.7 with two pieces a thread, 3.4 with four). Many: blocks of
  // about 256 threads, so that several are resident and one's sum is another's load (8192 x 4096 39.5 us, 5.9 TB/s, with
  // two pieces, 3 more with one; 2048 x 12288 33.4 with four, 7 more with two).
  const bool many = n.rows > 2 * sm_count();
  if (pieces <= 256 || (!many && pieces <= 1024)) return go(k_fp8_rms_norm<T, 1>, 1);
  if (pieces <= 512 || (!many && pieces <= 2048)) return go(k_fp8_rms_norm<T, 2>, 2);
  return go(k_fp8_rms_norm<T, 4>, 4);
}

}  // namespace

cudaError_t fp8_rows_launch(bool fp16, const uint16_t *x, const uint16_t *up, uint64_t stride, uint8_t *q, float *scales,
                            uint32_t rows, uint32_t width, cudaStream_t s) {
  const uint32_t halves = (width + kGroup - 1) / kGroup * rows, each = kHalves * at_once(up != nullptr);
  const uint32_t blocks = halves / each + (halves % each != 0);
  const auto go = [&](auto kernel) { return launch_after(kernel, blocks, 16 * kHalves, 0, s, x, up, stride, q, scales, rows, width); };
  if (fp16) return up ? go(k_fp8_rows<__half, true>) : go(k_fp8_rows<__half, false>);
  return up ? go(k_fp8_rows<__nv_bfloat16, true>) : go(k_fp8_rows<__nv_bfloat16, false>);
}

cudaError_t fp8_rms_norm_launch(bool fp16, const Fp8Norm &n, cudaStream_t s) {
  return fp16 ? norm_launch<__half>(n, s) : norm_launch<__nv_bfloat16>(n, s);
}

}  // namespace xpu
