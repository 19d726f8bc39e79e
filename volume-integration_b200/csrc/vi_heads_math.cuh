// Element conversions, activations and the 16-bit form of act' of the per-pixel heads.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

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
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float2 pair(float v) { return make_float2(v, v); }

constexpr float kLog2e = 1.4426950408889634f;

// act(z) and, where SLOPE, act'(z) of two values in float32.  A NaN stays a NaN.  EXACT: to a
// few float32 steps, beside float32 outputs; else to 6e-6 of the value, beside 16-bit ones.
// act' of a NaN is a NaN too, but relu's, which is 0 there (z > 0 is false).
//
// sigmoid: with e = exp(-z), s = 1 / (1 + e) and 1 - s = e s, without cancellation
// for large z.  The slope's e is kept finite, so that e s is 0 and not inf * 0 where s is 0; the
// value does not depend on whether the slope is wanted.
// gelu: with x = -|z| and Q = Phi(x), z Phi(z) = max(z, 0) + x Q, and act' is h = Q + x phi(x) for
// z < 0, 1 - h else.  log2 Phi is smooth on [-13.1, 0]; Q is exp2 of a polynomial of degree 8
// fitted to it here by minimax (a linear program over 4000 points, weighted by what the result can tell apart): 6e-6 of
// the value in float32 down to -3, 2e-8 absolute of x Q down to -5, 6e-3 of the value beyond.  Below -13.1, where
// Q < 2^-126 is 0, x stays there.  14 instructions a pair instead of 22 with the reciprocal form: they, not
// memory, bounded 64-channel frames.
// Sums and products of pairs are one instruction each.
template <int ACT, bool EXACT, bool SLOPE>
__device__ __forceinline__ void activate(float2 z, float2& y, float2& d) {
  if constexpr (ACT == VI_ACT_RELU) {
    y = make_float2(z.x <= 0.0f ? 0.0f : z.x, z.y <= 0.0f ? 0.0f : z.y);
    d = make_float2(z.x > 0.0f ? 1.0f : 0.0f, z.y > 0.0f ? 1.0f : 0.0f);
  } else if constexpr (ACT == VI_ACT_SILU || ACT == VI_ACT_SIGMOID) {
    float2 e, s;
    if constexpr (EXACT) {
      e = make_float2(expf(-z.x), expf(-z.y));
      s = make_float2(1.0f / (1.0f + e.x), 1.0f / (1.0f + e.y));
    } else {
      const float2 t = __fmul2_rn(z, pair(-kLog2e));
      e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
      const float2 q = __fadd2_rn(e, pair(1.0f));
      s = make_float2(rcp_fast(q.x), rcp_fast(q.y));
    }
    const float2 c = __fmul2_rn(make_float2(min_nan(e.x, 0x1p126f), min_nan(e.y, 0x1p126f)), s);
    if constexpr (ACT == VI_ACT_SILU) {
      y = __fmul2_rn(z, s);
      d = __fmul2_rn(s, __ffma2_rn(z, c, pair(1.0f)));
    } else {
      y = s;
      d = __fmul2_rn(s, c);
    }
  } else if constexpr (ACT == VI_ACT_GELU) {
    if constexpr (EXACT) {
      const float2 cdf = make_float2(normcdff(z.x), normcdff(z.y));
      y = __fmul2_rn(z, cdf);
      const float2 g = make_float2(expf(-0.5f * z.x * z.x), expf(-0.5f * z.y * z.y));
      d = __ffma2_rn(__fmul2_rn(z, pair(0.3989422804f)), g, cdf);
    } else {
      const float2 x = make_float2(max_nan(-fabsf(z.x), -13.1f), max_nan(-fabsf(z.y), -13.1f));
      float2 r = __ffma2_rn(x, pair(4.1239154e-08f), pair(2.531927e-06f));
      r = __ffma2_rn(r, x, pair(6.5017906e-05f));
      r = __ffma2_rn(r, x, pair(0.00093099725f));
      r = __ffma2_rn(r, x, pair(0.008470713f));
      r = __ffma2_rn(r, x, pair(0.05386456f));
      r = __ffma2_rn(r, x, pair(-0.45854974f));
      r = __ffma2_rn(r, x, pair(1.1512262f));
      r = __ffma2_rn(r, x, pair(-0.99999654f));
      const float2 q = make_float2(exp2_fast(r.x), exp2_fast(r.y));
      y = __ffma2_rn(x, q, make_float2(max_nan(z.x, 0.0f), max_nan(z.y, 0.0f)));
      if constexpr (SLOPE) {
        const float2 a = __fmul2_rn(__fmul2_rn(x, pair(-0.5f * kLog2e)), x);
        const float2 g = make_float2(exp2_fast(a.x), exp2_fast(a.y));
        const float2 h = __ffma2_rn(__fmul2_rn(x, pair(0.3989422804f)), g, q);
        const float2 k = __ffma2_rn(h, pair(-1.0f), pair(1.0f));
        d = make_float2(z.x > 0.0f ? k.x : h.x, z.y > 0.0f ? k.y : h.y);
      }
    }
  } else {
    y = z;
    d = pair(1.0f);
  }
}

// act' lies in (-0.2, 1.2) and is kept in 16 bits beside 16-bit types, more precisely
// than they hold values, so that the product dy * act' is off by its own rounding
// and little else.
// Beside bfloat16 as float16 of act' * 2^15 (half a step 2^-11 of the value, an eighth of bfloat16's, down to 2^-29;
// 2^-40 absolute below: a saturated unit keeps its gradient to sigmoid(27), where float16 alone gave 0 from 18 on).  A code
// with 6 bits of exponent and 9 of mantissa reached 2^-62, but packing it cost the forward of 65536 x 512 -> 512 with
// silu 10 us of 97.
// Beside float16 with a sign, 4 bits of exponent and 11 of mantissa (2^-12, half of float16's, down to 2^-14; 2^-26
// absolute below).  The float scaled by 2^-112 has its exponent in the low 4 bits of the field; a
// NaN, like all above the range, becomes the largest code, which no act' has.
template <typename T>
struct Slope;
template <>
struct Slope<__nv_bfloat16> {
  // two products by an immediate: a pair's constant would hold two registers through the epilogue (2M x 64 -> 64 with gelu,
  // which does not even keep act': 216 us, 221)
  static __device__ __forceinline__ uint32_t pack(float2 d) {
    const __half2 h = __float22half2_rn(make_float2(d.x * 0x1p15f, d.y * 0x1p15f));
    return *(const uint32_t*)&h;
  }
  static __device__ __forceinline__ float unpack(uint16_t v) { return __half2float(__ushort_as_half(v)) * 0x1p-15f; }
};
template <>
struct Slope<__half> {
  static constexpr uint32_t kNan = 0x7fff;
  static __device__ __forceinline__ uint32_t pack(float2 d) {
    const float2 s = __fmul2_rn(d, pair(0x1p-112f));
    const uint32_t a = __float_as_uint(s.x), b = __float_as_uint(s.y);
    const uint32_t m = min(((a & 0x7fffffffu) + 0x800u) >> 12, kNan), n = min(((b & 0x7fffffffu) + 0x800u) >> 12, kNan);
    return m | (n << 16) | ((a >> 16) & 0x8000u) | (b & 0x80000000u);
  }
  static __device__ __forceinline__ float unpack(uint16_t v) {
    const uint32_t a = v & 0x7fffu;
    const float m = a == kNan ? NAN : __uint_as_float(a << 12) * 0x1p112f;
    return v & 0x8000u ? -m : m;
  }
};

// A relu result that may serve as its act': a positive value that float16 rounds to 0 becomes -0 (equal to it, but told
// from the 0 of z <= 0), so that its gradient passes.  bfloat16's smallest step is below float32's normal range.
template <typename T>
__device__ __forceinline__ float2 relu_signed_zero(float2 y) {
  if constexpr (std::is_same<T, __half>::value)
    return make_float2(y.x > 0.0f && y.x <= 0x1p-25f ? -0.0f : y.x, y.y > 0.0f && y.y <= 0x1p-25f ? -0.0f : y.y);
  return y;
}

// act' as kept: the code above (float32 beside float32), or for relu anything that is positive where it
// is 1, so that the result itself serves (float16's -0 is, a NaN is not).
template <typename T>
__device__ __forceinline__ float kept_slope(uint16_t v, bool relu) {
  constexpr bool kIsHalf = std::is_same<T, __half>::value;
  constexpr uint32_t kInf = kIsHalf ? 0x7c00u : 0x7f80u;
  return relu ? ((uint32_t)v - 1u < kInf || (kIsHalf && v == 0x8000u) ? 1.0f : 0.0f) : Slope<T>::unpack(v);
}
__device__ __forceinline__ float kept_slope(float v, bool relu) { return relu ? (v > 0.0f ? 1.0f : 0.0f) : v; }

// Two float32 values rounded to T, packed.
__device__ __forceinline__ uint32_t pack2(float2 v, __half) {
  const __half2 h = __float22half2_rn(v);
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t pack2(float2 v, __nv_bfloat16) {
  const __nv_bfloat162 h = __float22bfloat162_rn(v);
  return *(const uint32_t*)&h;
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
