// Rows of 8-bit integers with a scale each.
//
// Mathematics.  s = f32(max_k |x_k| / 127), q_k = x_k / s rounded to the nearest whole number, ties to even: |q| <= 127.
// The rounding is that of the exact quotient: x times the rounded 1 / s decides it, but near halves, where a division in
// 64 bits does.  A row of zeros has s = 0 and q = 0; one that holds an infinity or a NaN has s = NaN and q = 0, so
// that what is made of it is NaN.
//
// Memory bounds it: one pass over x, held in registers between the maximum and the rounding.
#include <algorithm>

#include "vi_heads.h"
#include "vi_heads_math.cuh"
#include "vi_internal.h"

namespace vi {
namespace heads {
namespace {

constexpr int kThreads = 256;

// Near a half, or for a scale whose reciprocal is no float: the quotient of two floats is never so near a half without being
// one that 53 bits would not tell.
__device__ __noinline__ int quotient(float x, float s) {
  const double q = rint((double)x / (double)s);
  return (int)fmin(fmax(q, -127.0), 127.0);
}
struct Scale {
  float s, inv;
  bool slow;
  // of the largest magnitude's bits
  __device__ __forceinline__ explicit Scale(uint32_t top) {
    s = __fdiv_rn(__uint_as_float(top), 127.0f);
    if (top >= 0x7f800000u) s = NAN;
    slow = s > 0.0f && s < 0x1p-100f;
    inv = s >= 0x1p-100f ? __fdiv_rn(1.0f, s) : 0.0f;
  }
  __device__ __forceinline__ int of(float x) const {
    if (!(s > 0.0f)) return 0;  // zeros; not finite
    const float t = x * inv, r = rintf(t);
    if (slow || fabsf(t - r) > 0.4999f) return quotient(x, s);
    return (int)r;
  }
};

// A block a row at a time, any strides and lengths.
template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const __grid_constant__ QuantArgs a) {
  __shared__ uint32_t sh[kThreads / 32];
  for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
    const T* x = (const T*)a.x.p + m * a.x.rs;
    uint32_t top = 0;
    for (int k = threadIdx.x; k < a.K; k += kThreads) top = max(top, __float_as_uint(to_f(x[k * a.x.cs])) & 0x7fffffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; i++) top = max(top, sh[i]);
    const Scale s(top);
    for (int k = threadIdx.x; k < a.K; k += kThreads) a.q[m * a.ld + k] = (int8_t)s.of(to_f(x[k * a.x.cs]));
    if (threadIdx.x == 0) a.scale[m] = s.s;
  }
}

__global__ void __launch_bounds__(kThreads) pack8_kernel(View src, int64_t rows, int64_t k, int8_t* dst, int64_t ld) {
  const int8_t* p = (const int8_t*)src.p;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows * k; i += (int64_t)gridDim.x * kThreads)
    dst[i / k * ld + i % k] = p[i / k * src.rs + i % k * src.cs];
}

}  // namespace

cudaError_t launch_quantize(int dtype, const QuantArgs& a, int sms, cudaStream_t s) {
  const unsigned blocks = (unsigned)std::min<int64_t>(a.M, (int64_t)sms * 8);
  if (dtype == VI_F32) quantize_kernel<float><<<blocks, kThreads, 0, s>>>(a);
  else if (dtype == VI_F16) quantize_kernel<__half><<<blocks, kThreads, 0, s>>>(a);
  else quantize_kernel<__nv_bfloat16><<<blocks, kThreads, 0, s>>>(a);
  return cudaPeekAtLastError();
}
cudaError_t launch_pack8(const View& src, int64_t rows, int64_t k, int8_t* dst, int64_t ld, cudaStream_t s) {
  const unsigned blocks = (unsigned)std::min<int64_t>((rows * k + kThreads - 1) / kThreads, 148 * 16);
  pack8_kernel<<<blocks, kThreads, 0, s>>>(src, rows, k, dst, ld);
  return cudaPeekAtLastError();
}

}  // namespace heads
}  // namespace vi
