// Kernels that make block-scaled rows (formats and rounding: block_scale.h) and read them back:
//   block_quantize       out, scales <- x
//   block_dequantize     out <- values of (x, scales)
//   rms_norm_quantize    out, scales <- c r w with c = x or residual + x, r = 1 / sqrt(mean(c^2) + eps); residual_out <- c
//   silu_mul_quantize    out, scales <- gate / (1 + exp(-gate)) * up
// Everything between the loads and the quantised store is f32 (sums of squares, and values next to a border of their format, f64) and stays in registers: the
// 16-bit rows that separate kernels would hand on are neither written nor rounded to.  Rows of N values fill the first N columns of out, the columns behind them
// (up to whole blocks, or to the K of the product that reads them) are zeros.
//
// A lane holds a unit of 8 consecutive values, the lanes of a block are neighbours (4, or 2 for nvfp4), and its scale is found
// with one or two DPP steps.
#include <hip/hip_runtime.h>

#include "block_scale.h"
#include "gemm_common.h"
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

// The eight values of unit u of a row of n, any stride; 0 behind the row.  (Columns in 64 bits: 4-bit rows of 2^30 bytes and more have 2^31 values.)
template <typename T>
__device__ __forceinline__ void load_unit(const TensorArg<2>& t, int64_t r, int32_t u, int32_t n, float (&v)[8]) {
  const int64_t j = (int64_t)u * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = j + i < n ? (float)*at<T>(t, r, j + i) : 0.0f;
}

// ---- values next to a border ---------------------------------------------------------------------------------------------
// A value that is the result of f32 roundings and lies next to a border between two codes, or next to a power of two, which is a border between two block
// scales, may be on the wrong side of it or on the border itself.  So the fused kernels of the mx formats compute in f32, and what comes within some steps
// of f32 (`slack`, what the f32 result may be off) of a border they compute again in f64: the quantised row is that of the 64-bit results.  A sum residual + x is
// one of f32 in both.  Values below 2^-118, whose blocks have scale bytes 0 and 1, stay as f32 has them: kTiny counts there, and borders among subnormals have no
// zeros.  (nvfp4 elements are products with one more factor, which has borders of its own.)
// Steps from the nearest border below, plus the slack: up to twice the slack within reach.  Borders of the mx formats have zeros in all these
// bits; zeros, which are none, are made 2^-142 (and quantised as zeros).
constexpr float kTiny = 0x1p-142f;
template <Format F>
__device__ __forceinline__ uint32_t border_distance(float v, uint32_t slack) {
  return F == kNvfp4 ? ~0u : (__builtin_bit_cast(uint32_t, v) + slack) & (F == kMxfp8 ? (1u << 19) - 1 : (1u << 21) - 1);
}
// y as a float on the same side of every border; what is not further from one than `tie` of itself is on it.
template <Format F>
__device__ __forceinline__ float settled(double y, double tie) {
  const float f = (float)y;
  const double left = y - (double)f;
  if (border_distance<F>(f, 0) != 0 || !(__builtin_fabs(left) > __builtin_fabs(y) * tie) || !__builtin_isfinite(left)) return f;
  const int32_t b = __builtin_bit_cast(int32_t, f);
  return __builtin_bit_cast(float, b + (((b >> 31) ^ (left < 0.0 ? -1 : 0)) | 1));
}
// The values of the bits in `which` by `again(e)` of them.
template <Format F, class Again>
__device__ __forceinline__ void retake(float (&v)[8], uint32_t which, double tie, Again again) {
#pragma unroll 1
  while (which != 0) {
    const int at = __builtin_ctz(which);
    which &= which - 1;
    const float f = settled<F>(again(at), tie);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e == at ? f : v[e];
  }
}
// Those of a unit within `slack` steps of a border; one or none as a rule.
template <Format F, class Again>
__device__ __forceinline__ void settle(float (&v)[8], uint32_t slack, double tie, Again again) {
  if constexpr (F == kNvfp4) return;
  uint32_t border = ~0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) border = min(border, border_distance<F>(v[e], slack));
  if (border > 2 * slack) return;
  uint32_t near = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) near |= border_distance<F>(v[e], slack) <= 2 * slack ? 1u << e : 0u;
  retake<F>(v, near, tie, again);
}

// g / (1 + exp(-g)) * u, through h = exp(-|g| / 2) <= 1, which nothing overflows: g / (1 + h^2) times u, or u h^2 where g is below 0.  The square leaves f32 at
// |g| = 87, its product with a large u need not, so u is multiplied by h twice; from 174 on h itself is 0 (the product is below 2^-115 there).
// Off by less than 16 + 2 |min(g, 0)| steps: exponential twice 4, the products with it 2, sum 1, reciprocal 2, products 2, and 1.23 |g| where h is a factor of the
// result (the argument's rounding 1, that of log2(e) 0.23).  nvfp4: the quotient is corrected once by its remainder.
// (With the library's exponential and division 45 vector instructions a value, 31 us for 1500 x 14336 where memory takes 17; now 29 and
// 22 us, values in f64 among them.  Of 21.5 million codes none differs from the 64-bit result, of the plain f32 form's 7 to 111.)
template <Format F>
__device__ __forceinline__ float silu_mul(float g, float u) {
  const float h = __builtin_amdgcn_exp2f(__builtin_fabsf(g) * -0.72134752f);   // log2(e) / 2
  const float d = __builtin_fmaf(h, h, 1.0f), q = __builtin_amdgcn_rcpf(d), y = g * q, s = g > 0.0f ? u : u * h * h;
  if constexpr (F != kNvfp4) return __builtin_fmaf(y, s, kTiny);
  return __builtin_fmaf(__builtin_fmaf(-y, d, g), q, y) * s;
}
__device__ __forceinline__ double silu_mul_f64(double g, double u) { return g / (1.0 + exp(-g)) * u; }
// The unit's gates `v` and factors `w` to their products, those next to a border by `again(e)` in f64.  exp(-g) is no rational number, so no product is a border
// but where 1 + exp(-g) is 1 in f64, and there f64 has the product exactly: only what equals a border is on it (gate 36 and factor 1.5 are 2^-52 below one).
template <Format F, class Again>
__device__ __forceinline__ void silu_unit(float (&v)[8], const float (&w)[8], Again again) {
  float low = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) low = fminf(low, v[e]);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = silu_mul<F>(v[e], w[e]);
  settle<F>(v, (uint32_t)__builtin_fmaf(-2.0f, fmaxf(low, -175.0f), 16.0f), 0.0, again);
}

// mean(c^2) + eps = sum * inv_n + eps
struct NormMean {
  double inv_n, eps;
};
// c / sqrt(mean) * w: two products of f32 are off by 4.5 x 2^-24 of themselves at most (the mean's rounding, root, quotient and the products); in f64 two
// Newton steps from there (nvfp4: rounded once, with r in two parts).  Of 134 million values at most one differs from the 64-bit result, through a sum residual + x
// that f32 rounds; 70 where the two f32 products are all.
constexpr uint32_t kNormSlack = 8;
// What the norm in f64 may be off by: half of what the sum of squares collects, 2^-53 for each of the additions that a value passes (held rows 8 + 4 in its lane, 6 + 16
// across lanes and wavefronts; otherwise n / 2048 + 8 and 10), and 4 for mean, root and products: below 2^-44 for rows of up to 2^20 values.
constexpr double kNormTie = 0x1p-44;
struct Scale {
  float r, rest;   // exact = r + rest
  double exact;
  template <Format F>
  __device__ __forceinline__ float times(float c, float w) const {
    const float t = c * r;
    return F == kNvfp4 ? __builtin_fmaf(t, w, __builtin_fmaf(c, rest, __builtin_fmaf(c, r, -t)) * w) : __builtin_fmaf(t, w, kTiny);
  }
  __device__ __forceinline__ double in_f64(float c, float w) const { return (double)c * exact * (double)w; }
};
// The root is taken in f32, of a mean whose f32 is neither 0 nor subnormal: one below 2^-100 (eps = 0) is scaled by an even power of two.  A mean of 2^128 and more,
// of rows whose root mean square is 2^64 and more, is infinite in f32, and the row 0.
__device__ __forceinline__ Scale norm_scale(double mean) {
  const bool small = mean > 0.0 && mean < 0x1p-100;
  const double m = small ? mean * 0x1p200 : mean;
  Scale s;
  const float r = 1.0f / sqrtf((float)m);
  s.exact = (double)r;
  if (r > 0.0f && r < __builtin_inff()) {   // (rows of zeros, infinities and NaN, and beyond f32, stay as they are)
#pragma unroll
    for (int i = 0; i < 2; ++i) s.exact = __builtin_fma(0.5 * s.exact, __builtin_fma(-m * s.exact, s.exact, 1.0), s.exact);
  }
  if (small) s.exact *= 0x1p100;
  s.r = (float)s.exact;
  s.rest = (float)(s.exact - (double)s.r);
  if (!__builtin_isfinite(s.rest)) s.rest = 0.0f;   // (infinity less infinity)
  return s;
}

// Sum over the wavefront, in every lane.
__device__ __forceinline__ double wave_sum(double v) {
  union Words {
    double d;
    int32_t w[2];
  };
  auto add = [&](auto exchange) {
    Words a{v}, b;
    b.w[0] = exchange(a.w[0]), b.w[1] = exchange(a.w[1]);
    v = a.d + b.d;
  };
  add([](int32_t w) { return lanes::dpp<lanes::kQuadXor1>(w); });
  add([](int32_t w) { return lanes::dpp<lanes::kQuadXor2>(w); });
  add([](int32_t w) { return lanes::dpp<lanes::kHalfMirror>(w); });
  add([](int32_t w) { return lanes::dpp<lanes::kRowMirror>(w); });
  Words a{v}, e, o;
  for (int i = 0; i < 2; ++i) lanes::split_row_pairs(a.w[i], &e.w[i], &o.w[i]);
  a.d = e.d + o.d;
  for (int i = 0; i < 2; ++i) lanes::split_halves(a.w[i], &e.w[i], &o.w[i]);
  return e.d + o.d;
}

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
      silu_unit<F>(v, w, [&](int e) {
        const int64_t j = (int64_t)u * 8 + e;
        return j < n ? silu_mul_f64((double)*at<T>(x, r, j), (double)*at<T>(*up, r, j)) : 0.0;
      });
    }
    quantize_unit<F>(v, t, data_at<F>(out, r, u), scale_at<F>(scales, r, u));
  }
}

// ---- rows of unit stride ---------------------------------------------------------------------------------------------
// A unit as it lies in memory: 16 bytes (f32: 32), read with one (two) loads of any alignment; behind the row 0.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 Unaligned __attribute__((aligned(2)));
template <typename T>
struct Unit {
  static constexpr int kVectors = sizeof(T) / 2, kPer = 8 / kVectors;
  union {
    u32x4 raw[kVectors];
    T v[8];
  };
  __device__ __forceinline__ Unit() {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) raw[i] = u32x4{0, 0, 0, 0};
  }
  // `left` values of the row from p on; a unit on the row's end goes value by value.  WHOLE: the row is units without a rest.
  template <bool WHOLE>
  __device__ __forceinline__ void load(const T* p, int64_t left) {
    if (WHOLE || left >= 8) {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) raw[i] = *reinterpret_cast<const Unaligned*>(p + i * kPer);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) v[i] = p[i];
    }
  }
  template <bool WHOLE>
  __device__ __forceinline__ void store(T* p, int64_t left) const {
    if (WHOLE || left >= 8) {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) *reinterpret_cast<Unaligned*>(p + i * kPer) = raw[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) p[i] = v[i];
    }
  }
};

// Units of a launch in one sequence, row after row, neighbours to neighbouring lanes; a workgroup takes U of them for each of its
// threads (the launcher counts with the same U).  Where everything is contiguous the launcher makes one row of it.
// One unit a thread for the quantising kernels: later workgroups read while earlier ones write (us with 1, 2, 4, 8 of them: 16384 x 8192 bf16 to mxfp8
// 71, 75, 73, 78; gated activation of 1500 x 14336, without values in f64, 22.2, 24.6, 25.5, 29.3); four for reading back (16384 x 8192 mxfp4 to bf16 65, 69, 61, 65).
// Loads are ordinary ones: a prompt's rows come out of the memory-side cache, past which nontemporal loads go (1500 x 14336 to mxfp8 13.5 us, so 11.7).
constexpr int kQuantizeUnits = 1, kDequantizeUnits = 4;
struct UnitPlace {
  uint32_t r, u;
  bool live;
};
template <int U>
__device__ __forceinline__ void unit_places(uint32_t rows, uint32_t units, UnitPlace (&at)[U]) {
  const uint32_t f = blockIdx.x * (kThreads * U) + threadIdx.x;
  if (rows == 1) {
#pragma unroll
    for (int i = 0; i < U; ++i) at[i] = {0, f + i * kThreads, f + i * kThreads < units};
    return;
  }
  const uint32_t down = kThreads / units, across = kThreads % units;   // from a unit to the thread's next by addition
  uint32_t r = f / units, u = f % units;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    at[i] = {r, u, r < rows};
    u += across;
    r += down + (u >= units);
    u -= u >= units ? units : 0;
  }
}

template <Format F, typename T, bool SILU, bool WHOLE>
__device__ __forceinline__ void quantize_units(const TensorArg<2>& x, const TensorArg<2>* up, const PartitionArg<2>& out, const PartitionArg<2>& scales,
                                               TensorScale t, uint32_t rows, uint32_t units, int64_t n) {
  UnitPlace at[kQuantizeUnits];
  unit_places(rows, units, at);
  Unit<T> a[kQuantizeUnits], b[SILU ? kQuantizeUnits : 1];
#pragma unroll
  for (int i = 0; i < kQuantizeUnits; ++i) {
    if (!at[i].live) continue;
    const int64_t j = (int64_t)at[i].u * 8;
    a[i].template load<WHOLE>((const T*)x.ptr + (int64_t)at[i].r * x.strides[0] + j, n - j);
    if constexpr (SILU) b[i].template load<WHOLE>((const T*)up->ptr + (int64_t)at[i].r * up->strides[0] + j, n - j);
  }
#pragma unroll
  for (int i = 0; i < kQuantizeUnits; ++i) {
    if (!at[i].live) continue;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)a[i].v[e];
    if constexpr (SILU) {
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = (float)b[i].v[e];
      silu_unit<F>(v, w, [&](int e) {
        const int64_t j = (int64_t)at[i].u * 8 + e;
        return j < n ? silu_mul_f64((double)((const T*)x.ptr)[(int64_t)at[i].r * x.strides[0] + j], (double)((const T*)up->ptr)[(int64_t)at[i].r * up->strides[0] + j]) : 0.0;
      });
    }
    quantize_unit<F>(v, t, data_at<F>(out, at[i].r, at[i].u), scale_at<F>(scales, at[i].r, at[i].u));
  }
}

template <Format F, typename T, bool WHOLE>
__device__ __forceinline__ void dequantize_units(const TensorArg<2>& x, const TensorArg<2>& scales, const PartitionArg<2>& out, float g, uint32_t rows,
                                                 uint32_t units, int64_t n) {
  UnitPlace at[kDequantizeUnits];
  unit_places(rows, units, at);
  uint2 word[kDequantizeUnits];
  uint32_t byte[kDequantizeUnits];
#pragma unroll
  for (int i = 0; i < kDequantizeUnits; ++i) {
    if (!at[i].live) continue;
    const uint8_t* d = (const uint8_t*)x.ptr + (int64_t)at[i].r * x.strides[0] + (int64_t)at[i].u * Traits<F>::kUnitBytes;
    if constexpr (F == kMxfp8)
      word[i] = *reinterpret_cast<const uint2*>(d);
    else
      word[i].x = *reinterpret_cast<const uint32_t*>(d);
    byte[i] = ((const uint8_t*)scales.ptr)[(int64_t)at[i].r * scales.strides[0] + at[i].u / Traits<F>::kLanes];
  }
#pragma unroll
  for (int i = 0; i < kDequantizeUnits; ++i) {
    if (!at[i].live) continue;
    float v[8];
    unpack_unit<F>(word[i].x, word[i].y, byte[i], g, v);
    Unit<T> o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o.v[e] = (T)v[e];
    const int64_t j = (int64_t)at[i].u * 8;
    o.template store<WHOLE>((T*)out.ptr + (int64_t)at[i].r * out.strides[0] + j, n - j);
  }
}

// Columns of unit stride: a weight that is kept [K, N], quantised along K.  A lane reads eight neighbouring rows of eight columns, 16 bytes a
// column (16 lanes: 256 bytes), and so holds a unit of each of the eight rows; no exchange is needed but the one for the scale.
// A wavefront covers 128 rows of four units, the eight of a workgroup lie side by side along the row.  Quantised units and scales
// go through LDS, so that a row's 32 units leave as whole lines and its scale bytes at once (straight from the lanes, 16 or 32 bytes to a
// line and byte by byte: 14336 x 4096 bf16 to mxfp4 out of [4096, 14336] 51 us, value by value 242).
constexpr int kColThreads = 512, kColRows = 128, kColUnits = 32;   // of a workgroup
template <Format F>
struct ColumnStage {
  static constexpr int kRowBytes = kColUnits * Traits<F>::kUnitBytes, kScales = kColUnits / Traits<F>::kLanes;
  uint8_t data[kColRows * kRowBytes], scale[kColRows * kScales];
  // unit u of row r; the rows that a store instruction's lanes write are 8 apart: each starts at another place
  __device__ __forceinline__ uint8_t* unit(int r, int u) { return data + r * kRowBytes + (u * Traits<F>::kUnitBytes + (r >> 3) * (kRowBytes / 8)) % kRowBytes; }
};
template <Format F, typename T, bool WHOLE>
__device__ __forceinline__ void quantize_columns(const TensorArg<2>& x, const PartitionArg<2>& out, const PartitionArg<2>& scales, TensorScale t, int64_t rows,
                                                 int32_t units, uint32_t groups, ColumnStage<F>& stage) {
  const uint32_t id = gemm::xcd_contiguous(blockIdx.x, gridDim.x);
  const int lane = threadIdx.x & 63, r_in = (lane >> 2) * 8, u_in = (int)(threadIdx.x >> 6) * 4 + (lane & 3);
  const int64_t r0 = (int64_t)(id / groups) * kColRows;
  const int32_t u0 = (int32_t)(id % groups) * kColUnits, n = x.shape[1];
  if (u0 + u_in < units && r0 + r_in < rows) {
    Unit<T> a[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t j = (int64_t)(u0 + u_in) * 8 + e;
      if (j < n) a[e].template load<WHOLE>((const T*)x.ptr + j * x.strides[1] + r0 + r_in, rows - r0 - r_in);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (float)a[e].v[i];
      quantize_unit<F>(v, t, stage.unit(r_in + i, u_in), stage.scale + (r_in + i) * ColumnStage<F>::kScales + u_in / Traits<F>::kLanes);
    }
  }
  __syncthreads();
  constexpr int kChunks = ColumnStage<F>::kRowBytes / 8, kUnitsOf8 = 8 / Traits<F>::kUnitBytes;   // 8 bytes to a lane
#pragma unroll
  for (int p = 0; p < kColRows * kChunks / kColThreads; ++p) {
    const int r = p * (kColThreads / kChunks) + threadIdx.x / kChunks, c = threadIdx.x % kChunks;
    if (r0 + r < rows && u0 + c * kUnitsOf8 < units) *reinterpret_cast<uint2*>(data_at<F>(out, r0 + r, u0 + c * kUnitsOf8)) = *reinterpret_cast<const uint2*>(stage.unit(r, c * kUnitsOf8));
  }
  constexpr int kScales = ColumnStage<F>::kScales, kLanes = Traits<F>::kLanes;
  for (int s = threadIdx.x; s < kColRows * kScales; s += kColThreads) {
    const int r = s / kScales, b = s % kScales;
    if (r0 + r < rows && u0 + b * kLanes < units) *scale_at<F>(scales, r0 + r, u0 + b * kLanes) = stage.scale[s];
  }
}

// A row of up to WPR * 64 * VPL units in the registers of WPR wavefronts: read once, summed, scaled, quantised.  Bound by memory;
// what the shapes are for, bf16 with residual to mxfp8, us (rows read and written once at the rate of a large copy in front): 16384 x 512 9.3: 11.7 with a
// wavefront of one unit a lane, 12.3 with two, 23 with four wavefronts; 4096 x 1024 4.7: 7.9 with one wavefront, 9.7 with four; 2048 x 2048 4.7: 8.4 with four
// of two units, 8.9 of three; 1500 x 5120 8.5: 11.6 with four of three, 14.1 with eight of four; 16384 x 8192 149: 164 to 166 with four or eight of four
// units, 240 with sixteen; 4096 x 16384 75: 89 with eight, 101 with sixteen; 2048 x 28672 65: 89 with sixteen.  Up to 500 rows every shape takes the time of a
// launch.  The sum of squares in f64 costs 2 % of the short ones (f32 over four values, then f64: 1500 x 5120 11.4, and 4 of 134 million codes off).
template <Format F, typename T, bool ADD, int WPR, int VPL, bool WHOLE>
__device__ __forceinline__ void norm_held(const TensorArg<2>* residual, const TensorArg<2>& x, const TensorArg<1>& w, const PartitionArg<2>& out,
                                          const PartitionArg<2>& scales, const PartitionArg<2>* residual_out, NormMean m, TensorScale t, int64_t rows,
                                          int32_t units, double (*part)[WPR]) {
  constexpr int kRows = WPR < 4 ? 4 / WPR : 1;      // of a workgroup
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, slot = wave / WPR, sub = wave % WPR;
  const int64_t r = (int64_t)blockIdx.x * kRows + slot;
  const bool live = r < rows;
  const int32_t n = x.shape[1];
  Unit<T> a[VPL], b[ADD ? VPL : 1], g[VPL];
  float c[VPL][8];
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int32_t u = i * (WPR * 64) + sub * 64 + lane;
    if (!live || u >= units) continue;
    const int64_t j = (int64_t)u * 8;
    a[i].template load<WHOLE>((const T*)x.ptr + r * x.strides[0] + j, n - j);
    if constexpr (ADD) b[i].template load<WHOLE>((const T*)residual->ptr + r * residual->strides[0] + j, n - j);
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int32_t u = i * (WPR * 64) + sub * 64 + lane;
    if (live && u < units) g[i].template load<WHOLE>((const T*)w.ptr + (int64_t)u * 8, n - (int64_t)u * 8);
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c[i][e] = ADD ? (float)a[i].v[e] + (float)b[ADD ? i : 0].v[e] : (float)a[i].v[e];
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = __builtin_fma((double)c[i][e], (double)c[i][e], sum);
    ss += sum;
  }
  ss = wave_sum(ss);
  if constexpr (WPR > 1) {
    if (lane == 0) part[slot][sub] = ss;
    __syncthreads();
    ss = 0.0;
#pragma unroll
    for (int i = 0; i < WPR; ++i) ss += part[slot][i];
  }
  if (!live) return;
  const Scale s = norm_scale(__builtin_fma(ss, m.inv_n, m.eps));
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int32_t u = i * (WPR * 64) + sub * 64 + lane;
    if (u >= units) continue;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = s.times<F>(c[i][e], (float)g[i].v[e]);
    auto again = [&](int at) {   // (from registers: a load here is what a row's last wavefront would wait for)
      float cv = 0.0f, gv = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) cv = e == at ? c[i][e] : cv, gv = e == at ? (float)g[i].v[e] : gv;
      return s.in_f64(cv, gv);
    };
    if (F == kNvfp4 && s.r == __builtin_inff()) retake<F>(v, 0xff, kNormTie, again);   // a row of subnormals: f32 does not hold its r (infinities lie on a border of the mx formats)
    settle<F>(v, kNormSlack, kNormTie, again);
    if constexpr (ADD) {   // (may be residual or x itself: this lane has read what it writes)
      Unit<T> o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o.v[e] = (T)c[i][e];
      o.template store<WHOLE>((T*)residual_out->ptr + r * residual_out->strides[0] + (int64_t)u * 8, n - (int64_t)u * 8);
    }
    if (!WHOLE && (int64_t)u * 8 + 8 > n) {   // behind the row nothing but zeros, whatever the norm is
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (int64_t)u * 8 + e < n ? v[e] : 0.0f;
    }
    quantize_unit<F>(v, t, data_at<F>(out, r, u), scale_at<F>(scales, r, u));
  }
}

// ---- any strides -------------------------------------------------------------------------------------------------------
// Sum over the workgroup, in every thread.
__device__ __forceinline__ double workgroup_sum(double v) {
  __shared__ double part[kThreads / 64];
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return part[0] + part[1] + part[2] + part[3];
}

template <Format F, typename T, bool ADD>
__device__ __forceinline__ void norm_rows(const TensorArg<2>* residual, const TensorArg<2>& x, const TensorArg<1>& w, const PartitionArg<2>& out,
                                          const PartitionArg<2>& scales, const PartitionArg<2>* residual_out, NormMean m, TensorScale t, int64_t rows,
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
    float c[8];
    double ss = 0.0;
    for (int32_t u = threadIdx.x; u < units; u += kThreads) {
      load(u, c);
      double sum = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = __builtin_fma((double)c[e], (double)c[e], sum);
      ss += sum;
    }
    const Scale s = norm_scale(__builtin_fma(workgroup_sum(ss), m.inv_n, m.eps));
    for (int32_t u = threadIdx.x; u < units; u += kThreads) {
      load(u, c);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t j = (int64_t)u * 8 + e;
        if (j >= n) continue;
        if constexpr (ADD) *at<T>(*residual_out, r, j) = (T)c[e];   // (may be residual or x itself: this thread has read the element)
        c[e] = settled<F>(s.in_f64(c[e], (float)((const T*)w.ptr)[j * w.strides[0]]), kNormTie);
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
      if ((int64_t)u * 8 + e < n) *at<T>(out, r, (int64_t)u * 8 + e) = (T)v[e];
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
#define BLOCK_UNITS(FMT, F, TYPE, T)                                                                                                                \
  extern "C" __global__ void __launch_bounds__(kThreads) block_quantize_entry__##FMT##_##TYPE##_rows(                                               \
      TensorArg<2> x, PartitionArg<2> out, PartitionArg<2> scales, TensorScale t, uint32_t rows, uint32_t units, int64_t n) {                       \
    if (n == 8ll * units) quantize_units<F, T, false, true>(x, nullptr, out, scales, t, rows, units, n);                                            \
    else quantize_units<F, T, false, false>(x, nullptr, out, scales, t, rows, units, n);                                                                        \
  }                                                                                                                                                 \
  extern "C" __global__ void __launch_bounds__(kColThreads) block_quantize_entry__##FMT##_##TYPE##_columns(                                         \
      TensorArg<2> x, PartitionArg<2> out, PartitionArg<2> scales, TensorScale t, int64_t rows, int32_t units, uint32_t groups) {                   \
    __shared__ __attribute__((aligned(16))) ColumnStage<F> stage;                                                                                   \
    if (rows % 8 == 0) quantize_columns<F, T, true>(x, out, scales, t, rows, units, groups, stage);                                                 \
    else quantize_columns<F, T, false>(x, out, scales, t, rows, units, groups, stage);                                                              \
  }                                                                                                                                                 \
  extern "C" __global__ void __launch_bounds__(kThreads) block_dequantize_entry__##FMT##_##TYPE##_rows(                                             \
      TensorArg<2> x, TensorArg<2> scales, PartitionArg<2> out, float g, uint32_t rows, uint32_t units, int64_t n) {                                \
    if (n == 8ll * units) dequantize_units<F, T, true>(x, scales, out, g, rows, units, n);                                                          \
    else dequantize_units<F, T, false>(x, scales, out, g, rows, units, n);                                                                                      \
  }
#define BLOCK_UNITS_16(FMT, F, TYPE, T)                                                                                                             \
  BLOCK_UNITS(FMT, F, TYPE, T)                                                                                                                      \
  extern "C" __global__ void __launch_bounds__(kThreads) silu_mul_quantize_entry__##FMT##_##TYPE##_rows(                                            \
      TensorArg<2> gate, TensorArg<2> up, PartitionArg<2> out, PartitionArg<2> scales, TensorScale t, uint32_t rows, uint32_t units, int64_t n) {   \
    if (n == 8ll * units) quantize_units<F, T, true, true>(gate, &up, out, scales, t, rows, units, n);                                              \
    else quantize_units<F, T, true, false>(gate, &up, out, scales, t, rows, units, n);                                                                          \
  }
#define NORM_HELD(FMT, F, TYPE, T, WPR, VPL)                                                                                                        \
  extern "C" __global__ void __launch_bounds__(WPR < 4 ? 256 : WPR * 64) rms_norm_quantize_entry__##FMT##_##TYPE##_w##WPR##v##VPL(                  \
      TensorArg<2> x, TensorArg<1> w, PartitionArg<2> out, PartitionArg<2> scales, NormMean m, TensorScale t, int64_t rows, int32_t units) {         \
    __shared__ double part[WPR < 4 ? 4 / WPR : 1][WPR];                                                                                              \
    if (x.shape[1] == 8ll * units) norm_held<F, T, false, WPR, VPL, true>(nullptr, x, w, out, scales, nullptr, m, t, rows, units, part);          \
    else norm_held<F, T, false, WPR, VPL, false>(nullptr, x, w, out, scales, nullptr, m, t, rows, units, part);                                   \
  }                                                                                                                                                 \
  extern "C" __global__ void __launch_bounds__(WPR < 4 ? 256 : WPR * 64) add_rms_norm_quantize_entry__##FMT##_##TYPE##_w##WPR##v##VPL(              \
      TensorArg<2> residual, TensorArg<2> x, TensorArg<1> w, PartitionArg<2> out, PartitionArg<2> scales, PartitionArg<2> residual_out, NormMean m,  \
      TensorScale t, int64_t rows, int32_t units) {                                                                                                 \
    __shared__ double part[WPR < 4 ? 4 / WPR : 1][WPR];                                                                                              \
    if (x.shape[1] == 8ll * units) norm_held<F, T, true, WPR, VPL, true>(&residual, x, w, out, scales, &residual_out, m, t, rows, units, part);   \
    else norm_held<F, T, true, WPR, VPL, false>(&residual, x, w, out, scales, &residual_out, m, t, rows, units, part);                            \
  }
#define NORMS_HELD(FMT, F, TYPE, T)   \
  NORM_HELD(FMT, F, TYPE, T, 1, 1)    \
  NORM_HELD(FMT, F, TYPE, T, 1, 2)    \
  NORM_HELD(FMT, F, TYPE, T, 4, 2)    \
  NORM_HELD(FMT, F, TYPE, T, 4, 3)    \
  NORM_HELD(FMT, F, TYPE, T, 4, 4)    \
  NORM_HELD(FMT, F, TYPE, T, 8, 4)    \
  NORM_HELD(FMT, F, TYPE, T, 16, 4)
#define BLOCK_KERNELS_16(FMT, F, TYPE, T)                                                                                                           \
  BLOCK_KERNELS(FMT, F, TYPE, T)                                                                                                                    \
  extern "C" __global__ void __launch_bounds__(kThreads) silu_mul_quantize_entry__##FMT##_##TYPE##_any(                                             \
      TensorArg<2> gate, TensorArg<2> up, PartitionArg<2> out, PartitionArg<2> scales, TensorScale t, int64_t rows, int32_t units) {                \
    quantize_rows<F, T, true>(gate, &up, out, scales, t, rows, units);                                                                              \
  }                                                                                                                                                 \
  extern "C" __global__ void __launch_bounds__(kThreads) rms_norm_quantize_entry__##FMT##_##TYPE##_any(                                             \
      TensorArg<2> x, TensorArg<1> w, PartitionArg<2> out, PartitionArg<2> scales, NormMean m, TensorScale t, int64_t rows, int32_t units) {         \
    norm_rows<F, T, false>(nullptr, x, w, out, scales, nullptr, m, t, rows, units);                                                               \
  }                                                                                                                                                 \
  extern "C" __global__ void __launch_bounds__(kThreads) add_rms_norm_quantize_entry__##FMT##_##TYPE##_any(                                         \
      TensorArg<2> residual, TensorArg<2> x, TensorArg<1> w, PartitionArg<2> out, PartitionArg<2> scales, PartitionArg<2> residual_out, NormMean m,  \
      TensorScale t, int64_t rows, int32_t units) {                                                                                                 \
    norm_rows<F, T, true>(&residual, x, w, out, scales, &residual_out, m, t, rows, units);                                                        \
  }
#define BLOCK_FORMAT(FMT, F)               \
  BLOCK_KERNELS_16(FMT, F, f16, _Float16)  \
  BLOCK_KERNELS_16(FMT, F, bf16, __bf16)   \
  BLOCK_KERNELS(FMT, F, f32, float)        \
  BLOCK_UNITS_16(FMT, F, f16, _Float16)    \
  BLOCK_UNITS_16(FMT, F, bf16, __bf16)     \
  BLOCK_UNITS(FMT, F, f32, float)          \
  NORMS_HELD(FMT, F, f16, _Float16)        \
  NORMS_HELD(FMT, F, bf16, __bf16)
BLOCK_FORMAT(mxfp8, kMxfp8)
BLOCK_FORMAT(mxfp4, kMxfp4)
BLOCK_FORMAT(nvfp4, kNvfp4)
