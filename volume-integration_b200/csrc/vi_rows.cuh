// Pieces that the kernels over rows of features share: a lane's vectors of a row, or of neighbouring pixels.
#pragma once
#include "vi_heads.h"
#include "vi_heads_math.cuh"

namespace vi {
namespace heads {
namespace {

template <typename T, int N>
struct __align__(N * sizeof(T) >= 16 ? 16 : N * sizeof(T)) Chunk {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Chunk<T, N> chunk_zero() {
  Chunk<T, N> c;
#pragma unroll
  for (int i = 0; i < N; i++) c.v[i] = from_f<T>(0.0f);
  return c;
}

// The lane's NV chunks of a row: columns (v * lanes + lane) * VEC on.
template <typename T, int VEC, int NV>
__device__ __forceinline__ void load_row(Chunk<T, VEC> (&c)[NV], const View& m, int64_t row, int K, int lanes, int lane) {
  const T* p = (const T*)m.p + row * m.rs;
#pragma unroll
  for (int v = 0; v < NV; v++) {
    const int at = (v * lanes + lane) * VEC;
    if constexpr (VEC > 1) c[v] = at < K ? *(const Chunk<T, VEC>*)(p + at) : chunk_zero<T, VEC>();
    else c[v].v[0] = at < K ? p[at * m.cs] : from_f<T>(0.0f);
  }
}
// VP neighbouring pixels of a channel; those behind the last are 0.
template <typename T, int VP>
__device__ __forceinline__ Chunk<T, VP> load_pixels(const View& m, int64_t row, int64_t c, int64_t M) {
  const T* p = (const T*)m.p + row * m.rs + c * m.cs;
  Chunk<T, VP> r = chunk_zero<T, VP>();
  if (row + VP <= M) {
    r = *(const Chunk<T, VP>*)p;
  } else {
#pragma unroll
    for (int j = 0; j < VP; j++)
      if (row + j < M) r.v[j] = p[j * m.rs];
  }
  return r;
}
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int pow2_at_least(int64_t n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

// Whether n neighbouring elements along the contiguous axis may be moved at once.
template <typename T>
bool moves(const View& v, int n, bool along_rows) {
  return (along_rows ? v.rs : v.cs) == 1 && (along_rows ? v.cs : v.rs) % n == 0 && (uintptr_t)v.p % (n * sizeof(T)) == 0;
}

}  // namespace
}  // namespace heads
}  // namespace vi
