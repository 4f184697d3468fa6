// Kernels that make block-scaled rows (formats and rounding: block_scale.h) and read them back:
//   block_quantize       out, scales <- x
//   block_dequantize     out <- values of (x, scales)
//   rms_norm_quantize    out, scales <- c r w with c = x or residual + x, r = 1 / sqrt(mean(c^2) + eps); residual_out <- c
//   silu_mul_quantize    out, scales <- gate / (1 + exp(-gate)) * up
// Everything between the loads and the quantised store is f32 and stays in registers: the 16-bit rows that separate kernels would
// hand on are neither written nor rounded to.  Rows of N values fill the first N columns of out, the columns behind them
// (up to whole blocks, or to the K of the product that reads them) are zeros.
//
// A lane holds a unit of 8 consecutive values, the lanes of a block are neighbours (4, or 2 for nvfp4), and its scale is found
// with one or two DPP steps.
#include <hip/hip_runtime.h>

#include "block_scale.h"
#include "kernel_args.h"

using namespace cutile;
using namespace cutile::blocks;

namespace {

constexpr int kThreads = 256;

// Element j of row r.
template <typename T>
__device__ __forceinline__ const T* at(const TensorArg<2>& t, int64_t r, int64_t j) { return (const T*)t.ptr + r * t.strides[0] + j * t.strides[1]; }
template <typename T, int R>
__device__ __forceinline__ T* at(const PartitionArg<R>& t, int64_t r, int64_t j) { return (T*)t.ptr + r * t.strides[0] + j * t.strides[1]; }

// Where unit u of row r of the quantised rows and its block's scale go.
template <Format F>
__device__ __forceinline__ uint8_t* data_at(const PartitionArg<2>& out, int64_t r, int32_t u) { return (uint8_t*)out.ptr + r * out.strides[0] + (int64_t)u * Traits<F>::kUnitBytes; }
template <Format F>
__device__ __forceinline__ uint8_t* scale_at(const PartitionArg<2>& scales, int64_t r, int32_t u) { return (uint8_t*)scales.ptr + r * scales.strides[0] + u / Traits<F>::kLanes; }

// The eight values of unit u of a row of n, any stride; 0 behind the row.
template <typename T>
__device__ __forceinline__ void load_unit(const TensorArg<2>& t, int64_t r, int32_t u, int32_t n, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = u * 8 + i < n ? (float)*at<T>(t, r, u * 8 + i) : 0.0f;
}

// (expf, not the bare exponential: that loses log2(e) * |g| roundings, and the quotient may as well be exact: the kernel waits for memory)
__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

template <Format F, typename T, bool SILU>
__device__ __forceinline__ void quantize_rows(const TensorArg<2>& x, const TensorArg<2>* up, const PartitionArg<2>& out, const PartitionArg<2>& scales,
                                              TensorScale t, int64_t rows, int32_t units) {
  const int32_t n = x.shape[1];
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows * units; i += (int64_t)gridDim.x * kThreads) {
    const int64_t r = i / units;
    const int32_t u = (int32_t)(i - r * units);
    float v[8];
    load_unit<T>(x, r, u, n, v);
    if constexpr (SILU) {
      float w[8];
      load_unit<T>(*up, r, u, n, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = silu_mul(v[e], w[e]);
    }
    quantize_unit<F>(v, t, data_at<F>(out, r, u), scale_at<F>(scales, r, u));
  }
}

// Sum over the workgroup, in every thread.
__device__ __forceinline__ float workgroup_sum(float v) {
  __shared__ float part[kThreads / 64];
  v = lanes::across_wave<lanes::Sum>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return part[0] + part[1] + part[2] + part[3];
}

template <Format F, typename T, bool ADD>
__device__ __forceinline__ void norm_rows(const TensorArg<2>* residual, const TensorArg<2>& x, const TensorArg<1>& w, const PartitionArg<2>& out,
                                          const PartitionArg<2>& scales, const PartitionArg<2>* residual_out, float eps, TensorScale t, int64_t rows,
                                          int32_t units) {
  const int32_t n = x.shape[1];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    auto load = [&](int32_t u, float (&c)[8]) {
      load_unit<T>(x, r, u, n, c);
      if constexpr (ADD) {
        float a[8];
        load_unit<T>(*residual, r, u, n, a);
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] += a[e];
      }
    };
    float c[8], ss = 0.0f;
    for (int32_t u = threadIdx.x; u < units; u += kThreads) {
      load(u, c);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(c[e], c[e], ss);
    }
    const float inv = 1.0f / sqrtf(workgroup_sum(ss) / (float)n + eps);
    for (int32_t u = threadIdx.x; u < units; u += kThreads) {
      load(u, c);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int32_t j = u * 8 + e;
        if (j >= n) continue;
        if constexpr (ADD) *at<T>(*residual_out, r, j) = (T)c[e];   // (may be residual or x itself: this thread has read the element)
        c[e] = c[e] * inv * (float)((const T*)w.ptr)[(int64_t)j * w.strides[0]];
      }
      quantize_unit<F>(c, t, data_at<F>(out, r, u), scale_at<F>(scales, r, u));
    }
  }
}

template <Format F, typename T>
__device__ __forceinline__ void dequantize_rows(const TensorArg<2>& x, const TensorArg<2>& scales, const PartitionArg<2>& out, float g, int64_t rows,
                                                int32_t units) {
  const int32_t n = out.shape[1];
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows * units; i += (int64_t)gridDim.x * kThreads) {
    const int64_t r = i / units;
    const int32_t u = (int32_t)(i - r * units);
    const uint8_t* d = (const uint8_t*)x.ptr + r * x.strides[0] + (int64_t)u * Traits<F>::kUnitBytes;
    uint32_t word[2] = {0, 0};
#pragma unroll
    for (int b = 0; b < Traits<F>::kUnitBytes; ++b) word[b / 4] |= (uint32_t)d[b] << (8 * (b % 4));
    float v[8];
    unpack_unit<F>(word[0], word[1], ((const uint8_t*)scales.ptr)[r * scales.strides[0] + u / Traits<F>::kLanes], g, v);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (u * 8 + e < n) *at<T>(out, r, u * 8 + e) = (T)v[e];
  }
}

}  // namespace

#define BLOCK_KERNELS(FMT, F, TYPE, T)                                                                                                              \
  extern "C" __global__ void __launch_bounds__(kThreads) block_quantize_entry__##FMT##_##TYPE##_any(                                                \
      TensorArg<2> x, PartitionArg<2> out, PartitionArg<2> scales, TensorScale t, int64_t rows, int32_t units) {                                    \
    quantize_rows<F, T, false>(x, nullptr, out, scales, t, rows, units);                                                                            \
  }                                                                                                                                                 \
  extern "C" __global__ void __launch_bounds__(kThreads) block_dequantize_entry__##FMT##_##TYPE##_any(                                              \
      TensorArg<2> x, TensorArg<2> scales, PartitionArg<2> out, float g, int64_t rows, int32_t units) {                                             \
    dequantize_rows<F, T>(x, scales, out, g, rows, units);                                                                                          \
  }
#define BLOCK_KERNELS_16(FMT, F, TYPE, T)                                                                                                           \
  BLOCK_KERNELS(FMT, F, TYPE, T)                                                                                                                    \
  extern "C" __global__ void __launch_bounds__(kThreads) silu_mul_quantize_entry__##FMT##_##TYPE##_any(                                             \
      TensorArg<2> gate, TensorArg<2> up, PartitionArg<2> out, PartitionArg<2> scales, TensorScale t, int64_t rows, int32_t units) {                \
    quantize_rows<F, T, true>(gate, &up, out, scales, t, rows, units);                                                                              \
  }                                                                                                                                                 \
  extern "C" __global__ void __launch_bounds__(kThreads) rms_norm_quantize_entry__##FMT##_##TYPE##_any(                                             \
      TensorArg<2> x, TensorArg<1> w, PartitionArg<2> out, PartitionArg<2> scales, float eps, TensorScale t, int64_t rows, int32_t units) {         \
    norm_rows<F, T, false>(nullptr, x, w, out, scales, nullptr, eps, t, rows, units);                                                               \
  }                                                                                                                                                 \
  extern "C" __global__ void __launch_bounds__(kThreads) add_rms_norm_quantize_entry__##FMT##_##TYPE##_any(                                         \
      TensorArg<2> residual, TensorArg<2> x, TensorArg<1> w, PartitionArg<2> out, PartitionArg<2> scales, PartitionArg<2> residual_out, float eps,  \
      TensorScale t, int64_t rows, int32_t units) {                                                                                                 \
    norm_rows<F, T, true>(&residual, x, w, out, scales, &residual_out, eps, t, rows, units);                                                        \
  }
#define BLOCK_FORMAT(FMT, F)               \
  BLOCK_KERNELS_16(FMT, F, f16, _Float16)  \
  BLOCK_KERNELS_16(FMT, F, bf16, __bf16)   \
  BLOCK_KERNELS(FMT, F, f32, float)
BLOCK_FORMAT(mxfp8, kMxfp8)
BLOCK_FORMAT(mxfp4, kMxfp4)
BLOCK_FORMAT(nvfp4, kNvfp4)
