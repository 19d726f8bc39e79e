// The heads' products when they are small: on the FP32 cores, straight from the caller's matrices in
// any strides, several products in one launch.
//
// A step on a few rows is bound by its launches (3 us each on the host, as much again before a kernel does
// work), not by arithmetic: the tensor-core path takes five to seven of them for a backward
// (lay out, two products, their pieces' sums), this one takes one.  A block makes a 32 x 32 tile
// of a product, 2 x 2 outputs a thread, with the next 64 of k on their way in registers.
// Elements are float32 once loaded, so dy * act' is not rounded here.
#include <algorithm>

#include "vi_heads.h"
#include "vi_heads_math.cuh"
#include "vi_internal.h"

namespace vi {
namespace heads {
namespace {

constexpr int kT = 32;      // tile
constexpr int kDepth = 64;  // of k in shared memory: a block waits for memory once per this many
constexpr int kThreads = 256;
constexpr int kEach = kT * kDepth / kThreads;  // elements a thread loads of either operand

template <typename T>
__device__ __forceinline__ float slope_at(const void* p, int64_t i, bool relu) {
  if constexpr (sizeof(T) == 4) return kept_slope(((const float*)p)[i], relu);
  else return kept_slope<T>(((const uint16_t*)p)[i], relu);
}

// Element `i` of a thread's share of 32 rows x 64 k: neighbouring threads along the contiguous axis.
__device__ __forceinline__ void place(bool k_fast, int i, int& row, int& k) {
  const int e = threadIdx.x + i * kThreads;
  row = k_fast ? e / kDepth : e % kT;
  k = k_fast ? e % kDepth : e / kT;
}

template <typename T>
__device__ __forceinline__ void fetch_a(const SmallJob& q, bool k_fast, int m0, int k0, float (&v)[kEach]) {
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    int r, k;
    place(k_fast, i, r, k);
    r += m0, k += k0;
    v[i] = 0.0f;
    if (r < q.M && k < q.K) {
      v[i] = to_f(((const T*)q.a.p)[r * q.a.rs + k * q.a.cs]);
      if (q.slope.p) v[i] *= slope_at<T>(q.slope.p, r * q.slope.rs + k * q.slope.cs, q.relu);
    }
  }
}
template <typename T>
__device__ __forceinline__ void fetch_b(const SmallJob& q, bool k_fast, int n0, int k0, float (&v)[kEach]) {
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    int r, k;
    place(k_fast, i, r, k);
    r += n0, k += k0;
    v[i] = 0.0f;
    if (r < q.N && k < q.K && !(q.skip && q.skip[k] == 0.0f)) v[i] = to_f(((const T*)q.b.p)[r * q.b.rs + k * q.b.cs]);
  }
}

__device__ __forceinline__ void activate1(int act, bool exact, float z, float& y, float& d) {
  const float2 v = pair(z);
  float2 a = v, s = pair(1.0f);
  switch (act) {
    case VI_ACT_RELU: activate<VI_ACT_RELU, true, true>(v, a, s); break;
    case VI_ACT_SILU: exact ? activate<VI_ACT_SILU, true, true>(v, a, s) : activate<VI_ACT_SILU, false, true>(v, a, s); break;
    case VI_ACT_GELU: exact ? activate<VI_ACT_GELU, true, true>(v, a, s) : activate<VI_ACT_GELU, false, true>(v, a, s); break;
    case VI_ACT_SIGMOID:
      exact ? activate<VI_ACT_SIGMOID, true, true>(v, a, s) : activate<VI_ACT_SIGMOID, false, true>(v, a, s);
      break;
    default: break;
  }
  y = a.x;
  d = s.x;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) small_kernel(const __grid_constant__ SmallJobs jobs) {
  __shared__ float sa[kDepth][kT + 2], sb[kDepth][kT + 2];  // [k][row]
  const bool second = (int)blockIdx.x >= jobs.tiles0;
  const SmallJob& q = jobs.j[second];
  const int tile = blockIdx.x - (second ? jobs.tiles0 : 0), nt = (q.N + kT - 1) / kT;
  const int m0 = tile / nt * kT, n0 = tile % nt * kT;
  const bool fa = q.a.cs == 1, fb = q.b.cs == 1;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[2][2] = {}, rows[2] = {};
  float va[kEach], vb[kEach];
  fetch_a<T>(q, fa, m0, 0, va);
  fetch_b<T>(q, fb, n0, 0, vb);
  for (int k0 = 0; k0 < q.K; k0 += kDepth) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      int r, k;
      place(fa, i, r, k);
      sa[k][r] = va[i];
      place(fb, i, r, k);
      sb[k][r] = vb[i];
    }
    __syncthreads();
    if (k0 + kDepth < q.K) {
      fetch_a<T>(q, fa, m0, k0 + kDepth, va);
      fetch_b<T>(q, fb, n0, k0 + kDepth, vb);
    }
#pragma unroll 8
    for (int k = 0; k < kDepth; k++) {
      const float2 a = *(const float2*)&sa[k][2 * ty], b = *(const float2*)&sb[k][2 * tx];
      acc[0][0] = fmaf(a.x, b.x, acc[0][0]);
      acc[0][1] = fmaf(a.x, b.y, acc[0][1]);
      acc[1][0] = fmaf(a.y, b.x, acc[1][0]);
      acc[1][1] = fmaf(a.y, b.y, acc[1][1]);
      rows[0] += a.x;
      rows[1] += a.y;
    }
  }
  const float alpha = q.alpha ? *q.alpha : 1.0f;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int m = m0 + 2 * ty + i;
    if (m >= q.M) continue;
    if (q.sums && n0 == 0 && tx == 0) ((T*)q.sums)[m] = from_f<T>(rows[i] * alpha);
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int n = n0 + 2 * tx + j;
      if (n >= q.N || !q.out.p) continue;
      float z = acc[i][j];
      if (q.bias) z += to_f(((const T*)q.bias)[n]);
      if (q.coef) {  // the logits' gradient
        const float c = q.coef[m];
        const bool hit = q.target[m] == n;
        z = exp2_fast(fmaf(z - q.lse[m], kLog2e, -q.lse[q.M + m])) - (hit ? 1.0f : 0.0f);
        z = c == 0.0f ? 0.0f : z * c;
      } else {
        float d;
        activate1(q.act, sizeof(T) == 4, z * alpha, z, d);
        if (q.act == VI_ACT_RELU) z = relu_signed_zero<T>(pair(z)).x;
        if (q.dact) {
          const int64_t at = m * q.out.rs + n * q.out.cs;
          if constexpr (sizeof(T) == 4) ((float*)q.dact)[at] = d;
          else ((uint16_t*)q.dact)[at] = (uint16_t)Slope<T>::pack(pair(d));
        }
        if (q.res.p) z += to_f(((const T*)q.res.p)[m * q.res.rs + n * q.res.cs]);
      }
      ((T*)q.out.p)[m * q.out.rs + n * q.out.cs] = from_f<T>(z);
    }
  }
}

}  // namespace

bool small_product(int64_t M, int64_t N, int64_t K, int64_t longest) {
  return std::max({M, N, K}) <= 65536 && M * N * K <= kSmallWork && longest <= kSmallSum;
}

cudaError_t launch_small(int dtype, const SmallJob& a, const SmallJob* b, cudaStream_t s) {
  SmallJobs jobs{};
  jobs.j[0] = a;
  auto tiles = [](const SmallJob& q) { return ((q.M + kT - 1) / kT) * ((q.N + kT - 1) / kT); };
  jobs.tiles0 = tiles(a);
  int total = jobs.tiles0;
  if (b) jobs.j[1] = *b, total += tiles(*b);
  if (dtype == VI_F32) small_kernel<float><<<total, kThreads, 0, s>>>(jobs);
  else if (dtype == VI_F16) small_kernel<__half><<<total, kThreads, 0, s>>>(jobs);
  else small_kernel<__nv_bfloat16><<<total, kThreads, 0, s>>>(jobs);
  return cudaPeekAtLastError();
}

}  // namespace heads
}  // namespace vi
