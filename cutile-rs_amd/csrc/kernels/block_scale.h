// Block-scaled formats: rows of narrow floats in blocks along K that share a scale.
//   mxfp8   e4m3 values, an e8m0 scale (2^(byte - 127)) to 32 of them
//   mxfp4   e2m1 values (two a byte, low nibble first), an e8m0 scale to 32
//   nvfp4   e2m1 values, an e4m3 scale to 16, and one f32 scale g of the whole tensor
//
// What a block of values v with largest magnitude a is turned into:
//   mx      byte = clamp(floor(log2 a) - emax + 127, 0, 254), emax = 8 (e4m3) or 2 (e2m1), a = 0: byte 0;
//           elements round(v * 2^(127 - byte)), to nearest even, saturated to 448 or 6 (the conversion of the OCP MX
//           specification 1.0, section 6.3)
//   nvfp4   s = e4m3(min(a * (1 / (6 g)), 448)); elements e2m1(v * (1 / (s g))), 0 where s is 0, every operation in f32.  (With g = largest / (6 * 448),
//           as tensors are calibrated, many a / (6 g) lie on a border between two scales: in f32 throughout the bytes are those that any program that
//           takes these steps gets; 1 / (6 g) rounded once instead moves one scale in eighty of some such tensors to its neighbour.)
//   a block that holds a NaN or an infinity: scale NaN (0xff or 0x7f), elements 0 - the whole block stands for NaN
// The exponent of a is that of its f32 bits, so the mx scale is an integer subtraction and the scaling exact.  Magnitudes are
// compared as integers: they order like floats, with infinities and NaN on top, where a float maximum would drop a NaN.
#pragma once
#include <hip/hip_runtime.h>

#include "lane_exchange.h"

namespace cutile {
namespace blocks {

enum Format { kMxfp8, kMxfp4, kNvfp4 };
template <Format F>
struct Traits {
  static constexpr int kBlock = F == kNvfp4 ? 16 : 32;
  static constexpr bool kFp4 = F != kMxfp8;
  static constexpr int kUnitBytes = kFp4 ? 4 : 8;     // of a unit: 8 consecutive values, what a lane holds
  static constexpr int kLanes = kBlock / 8;           // lanes of a block
};

// The scale of the tensor as the kernels take it: g, and 1 / (6 g).
struct TensorScale {
  float g, inv6g;
};

struct BlockScale {
  float mul;        // elements = round(v * mul)
  uint32_t byte;    // the scale as stored
  bool lost;        // a NaN or an infinity in the block
};

__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// The largest of the block's magnitudes in each of its lanes.
template <Format F>
__device__ __forceinline__ uint32_t block_most(uint32_t m) {
  m = max(m, (uint32_t)lanes::dpp<lanes::kQuadXor1>((int32_t)m));
  if constexpr (Traits<F>::kLanes == 4) m = max(m, (uint32_t)lanes::dpp<lanes::kQuadXor2>((int32_t)m));
  return m;
}

template <Format F>
__device__ __forceinline__ BlockScale block_scale(uint32_t most, TensorScale t) {
  BlockScale s;
  s.lost = most >= 0x7f800000u;
  if constexpr (F == kNvfp4) {
    const float want = fminf(__builtin_bit_cast(float, most) * t.inv6g, 448.0f);
    const int packed = __builtin_amdgcn_cvt_pk_fp8_f32(want, want, 0, false);
    const float unit = __builtin_amdgcn_cvt_f32_fp8(packed, 0);
    s.mul = unit > 0.0f ? 1.0f / (unit * t.g) : 0.0f;
    s.byte = s.lost ? 0x7fu : (uint32_t)packed & 0xffu;
  } else {
    const int byte = max((int)(most >> 23) - (F == kMxfp8 ? 8 : 2), 0);
    s.mul = __builtin_bit_cast(float, (uint32_t)(254 - byte) << 23);
    s.byte = s.lost ? 0xffu : (uint32_t)byte;
  }
  return s;
}

// Eight scaled values as stored: two dwords of e4m3 or one of e2m1.  Both conversions round to nearest even; the one to e2m1
// saturates by itself, the one to e4m3 makes NaN of what is beyond 464.
template <Format F>
__device__ __forceinline__ void pack_unit(const float (&v)[8], const BlockScale& s, uint32_t (&out)[2]) {
  if constexpr (F == kMxfp8) {
    auto e = [&](int i) { return __builtin_amdgcn_fmed3f(v[i] * s.mul, -448.0f, 448.0f); };
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      int p = __builtin_amdgcn_cvt_pk_fp8_f32(e(4 * d), e(4 * d + 1), 0, false);
      p = __builtin_amdgcn_cvt_pk_fp8_f32(e(4 * d + 2), e(4 * d + 3), p, true);
      out[d] = s.lost ? 0u : (uint32_t)p;
    }
  } else {
    uint32_t p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0] * s.mul, v[1] * s.mul, 1.0f, 0);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[2] * s.mul, v[3] * s.mul, 1.0f, 1);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[4] * s.mul, v[5] * s.mul, 1.0f, 2);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[6] * s.mul, v[7] * s.mul, 1.0f, 3);
    out[0] = s.lost ? 0u : p;
  }
}

// A lane's unit, quantised with the other lanes of its block, to its place in a row: `data` and `scale` are where the unit's
// bytes and the block's scale byte go.  All lanes of a block call it together.
template <Format F>
__device__ __forceinline__ void quantize_unit(const float (&v)[8], TensorScale t, uint8_t* data, uint8_t* scale) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, magnitude(v[i]));
  const BlockScale s = block_scale<F>(block_most<F>(most), t);
  uint32_t out[2];
  pack_unit<F>(v, s, out);
  if constexpr (F == kMxfp8)
    *reinterpret_cast<uint2*>(data) = uint2{out[0], out[1]};
  else
    *reinterpret_cast<uint32_t*>(data) = out[0];
  if ((threadIdx.x & (Traits<F>::kLanes - 1)) == 0) *scale = (uint8_t)s.byte;
}

// The eight values of a unit: `lo`, `hi` its bytes (hi: mxfp8 only), `byte` its block's scale.
template <Format F>
__device__ __forceinline__ void unpack_unit(uint32_t lo, uint32_t hi, uint32_t byte, float g, float (&v)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  if constexpr (F == kMxfp8) {
    // byte 255 is NaN, 0 the subnormal 2^-127
    const float s = __builtin_bit_cast(float, byte == 0xffu ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23);
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const int w = (int)(d ? hi : lo);
      v[4 * d] = __builtin_amdgcn_cvt_f32_fp8(w, 0) * s;
      v[4 * d + 1] = __builtin_amdgcn_cvt_f32_fp8(w, 1) * s;
      v[4 * d + 2] = __builtin_amdgcn_cvt_f32_fp8(w, 2) * s;
      v[4 * d + 3] = __builtin_amdgcn_cvt_f32_fp8(w, 3) * s;
    }
  } else {
    const f32x2 e[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(lo, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(lo, 1.0f, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(lo, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(lo, 1.0f, 3)};
    // nvfp4: element times scale is exact in f32, so g is the one rounding
    const float s = F == kNvfp4 ? __builtin_amdgcn_cvt_f32_fp8((int)byte, 0)
                                : __builtin_bit_cast(float, byte == 0xffu ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = F == kNvfp4 ? e[i / 2][i % 2] * s * g : e[i / 2][i % 2] * s;
  }
}

}  // namespace blocks
}  // namespace cutile
