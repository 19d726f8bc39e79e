// The rounding of rows to 8-bit integers (vi_quant.cu has the mathematics).
#pragma once
#include "vi_heads_math.cuh"

namespace vi {
namespace heads {
namespace {

// For a scale whose reciprocal is no float: the quotient of two floats is never so near a half without being one that 53
// bits would not tell.
__device__ __noinline__ int quotient(float x, float s) {
  const double q = rint((double)x / (double)s);
  return (int)fmin(fmax(q, -127.0), 127.0);
}

struct Scale {
  float s, inv;
  bool exact;  // x inv does not decide: the row is not finite, of zeros, or its scale has no float reciprocal
  __device__ __forceinline__ Scale() {}
  // of the largest magnitude's bits
  __device__ __forceinline__ explicit Scale(uint32_t top) {
    const float x = __uint_as_float(top);
    // Division by a constant as P. Markstein published it (IBM J. Res. Dev. 34, 1990): with r the rounded reciprocal and q within one
    // last place of x / 127, the rest x - 127 q is exact in one fused operation and q + r rest is the rounded quotient.  r is
    // off by 2^-28 of itself and x r is rounded once more, so q is within one last place.  The bounds keep every step among
    // normal numbers, the rest (down to 2^-24 of x) too.
    if (top >= 0x10000000u && top < 0x7f000000u) {
      constexpr float r = 1.0f / 127.0f;
      const float q = x * r;
      s = fmaf(fmaf(-127.0f, q, x), r, q);
      inv = rcp_fast(s);
      exact = false;
    } else {
      s = top >= 0x7f800000u ? NAN : __fdiv_rn(x, 127.0f);
      inv = 0.0f;
      exact = true;
    }
  }
};
// N values of a lane divided and rounded.  x inv is within 127 * 2^-22 of the quotient, so it decides but within that of a
// half.  There the rest x - q s does, which is exact: it is a multiple of half a last place of s and at most s / 2 or so.  (A
// bfloat16 row has its largest value's half in one of 400 places, whose quotient is 63.5: halves are not rare.)
template <int N>
__device__ __forceinline__ void quantize(const float (&x)[N], const Scale& s, int (&q)[N]) {
  float far = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float f = fmaf(x[i], s.inv, 12582912.0f);  // 1.5 * 2^23: the whole number is in the low bits
    far = fmaxf(far, fabsf(fmaf(x[i], s.inv, 12582912.0f - f)));
    q[i] = __float_as_int(f);
  }
  if (s.exact) {
#pragma unroll
    for (int i = 0; i < N; i++) q[i] = s.s > 0.0f ? quotient(x[i], s.s) : 0;
  } else if (far > 0.49996f) {
    const float half = 0.5f * s.s;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float e = fmaf(12582912.0f - __int_as_float(q[i]), s.s, x[i]);
      if (fabsf(e) > half || (fabsf(e) == half && (q[i] & 1))) q[i] += e > 0.0f ? 1 : -1;
    }
  }
}
__device__ __forceinline__ uint32_t bytes4(int a, int b, int c, int d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

}  // namespace
}  // namespace heads
}  // namespace vi
