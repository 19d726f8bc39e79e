// Element conversions, activations and the 16-bit form of act' of the per-pixel heads.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/volume_integration_b200.h"

namespace vi {
namespace heads {

template <typename T>
__device__ __forceinline__ float to_f(T v) { return (float)v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v) { return (T)v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLog2e = 1.4426950408889634f;

// act(z) and act'(z) in float32.  A NaN stays a NaN.  EXACT: to a few float32 steps,
// beside float32 outputs; else to 1e-6 of the value, beside 16-bit ones.
//
// sigmoid: with e = exp(-z), s = 1 / (1 + e) and 1 - s = e s, without cancellation
// for large z; e is kept finite, so e s tends to 1 and not to inf * 0.
// gelu: Phi(-x) = exp(-x^2 / 2) r(t) for x >= 0, t = 1 / (1 + 0.265 x), r a polynomial of
// degree 7 without constant term fitted here to Mills' ratio / sqrt(2 pi) by iteratively
// reweighted least squares: 6.3e-7 of the value over [0, 14], where float32 ends.
// One exponential serves Phi and the density.
template <int ACT, bool EXACT>
__device__ __forceinline__ void activate(float z, float& y, float& d) {
  if constexpr (ACT == VI_ACT_RELU) {
    y = z <= 0.0f ? 0.0f : z;
    d = z > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (ACT == VI_ACT_SILU || ACT == VI_ACT_SIGMOID) {
    float e, s;
    if constexpr (EXACT) {
      e = expf(fminf(-z, 87.0f));
      s = 1.0f / (1.0f + e);
    } else {
      e = exp2_fast(fminf(-z * kLog2e, 126.0f));
      s = __fdividef(1.0f, 1.0f + e);
    }
    if (z != z) s = z;
    const float c = e * s;
    if constexpr (ACT == VI_ACT_SILU) {
      y = z * s;
      d = s * fmaf(z, c, 1.0f);
    } else {
      y = s;
      d = s * c;
    }
  } else if constexpr (ACT == VI_ACT_GELU) {
    if constexpr (EXACT) {
      const float cdf = normcdff(z);
      y = z * cdf;
      d = cdf + z * 0.3989422804f * expf(-0.5f * z * z);
    } else {
      const float x = fabsf(z), t = __fdividef(1.0f, fmaf(0.265f, x, 1.0f));
      float r = -0.0677848929f;
      r = fmaf(r, t, 0.195265483f);
      r = fmaf(r, t, -0.0663519581f);
      r = fmaf(r, t, 0.142485184f);
      r = fmaf(r, t, 0.0829498892f);
      r = fmaf(r, t, 0.107836094f);
      r = fmaf(r, t, 0.105599892f);
      const float g = exp2_fast(z * z * (-0.5f * kLog2e)), q = g * (r * t);
      const float cdf = z < 0.0f ? q : 1.0f - q;
      y = z * cdf;
      d = fmaf(z * 0.3989422804f, g, cdf);
    }
  } else {
    y = z;
    d = 1.0f;
  }
}

// act' lies in (-0.2, 1.2).  Beside 16-bit outputs it is kept in 16 bits, with a sign, 4
// bits of exponent and 11 of mantissa: half a step is 2^-12 of the value (down to
// 2^-14, 2^-26 absolute below), a half of float16's and an eighth of bfloat16's, so
// the product dy * act' is off by its own rounding and little else.
// The float scaled by 2^-112 has its exponent in the low 4 bits of the field.
__device__ __forceinline__ uint16_t pack_slope(float d) {
  const uint32_t f = __float_as_uint(d);
  uint32_t u = __float_as_uint(__fmul_rn(__uint_as_float(f & 0x7fffffffu), 0x1p-112f));
  u = (u + 0x7ffu + ((u >> 12) & 1u)) >> 12;
  // a NaN (and nothing else) is beyond the 15 bits: keep it as the largest code
  return (uint16_t)((u > 0x7fffu ? 0x7fffu : u) | ((f >> 16) & 0x8000u));
}
__device__ __forceinline__ float unpack_slope(uint16_t v) {
  const float m = (v & 0x7fffu) == 0x7fffu ? NAN : __fmul_rn(__uint_as_float((uint32_t)(v & 0x7fffu) << 12), 0x1p112f);
  return v & 0x8000u ? -m : m;
}

// x = p0 + p1 + p2 with bfloat16 parts: 24 bits in all.  p0 is cut, not rounded, so that
// it cannot overflow; infinities and NaNs are p0 alone.
__device__ __forceinline__ void split3(float x, __nv_bfloat16 p[3]) {
  const uint32_t hi = __float_as_uint(x) & 0xffff0000u;
  float h = __uint_as_float(hi);
  if (!(fabsf(x) <= 3.402823466e38f)) {
    p[0] = x != x ? __ushort_as_bfloat16((unsigned short)0x7fff) : __ushort_as_bfloat16((unsigned short)(hi >> 16));
    p[1] = p[2] = __ushort_as_bfloat16((unsigned short)0);
    return;
  }
  p[0] = __ushort_as_bfloat16((unsigned short)(hi >> 16));
  const float r1 = x - h;
  p[1] = __float2bfloat16_rn(r1);
  p[2] = __float2bfloat16_rn(r1 - __bfloat162float(p[1]));
}

}  // namespace heads
}  // namespace vi
