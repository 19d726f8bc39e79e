// Layer norm of rows, forward and backward.
//
// Mathematics.  For a row x of K features: mu = mean x, v = mean (x - mu)^2, r = 1 / sqrt(v + eps),
//   h = (x - mu) r,  y = h w + b.
// Backward, g = dy w:  dx = r (g - mean g - h mean(g h));  dw = sum_m dy h;  db = sum_m dy.
// All sums are float32.  The mean's own rounding is taken out again: with d = x - mu the mean of d is subtracted
// from d, so rows far from zero lose nothing (mean 1000, spread 1: 6e-5 of h otherwise).
//
// Memory bounds it: a row is read once, kept in registers, and its statistics are made of what the registers
// hold.  Rows of contiguous features belong to 1 to 32 lanes or to a block (vectors of 16 bytes, or single elements
// where strides or sizes do not allow them); images, where pixels are contiguous, to blocks whose lanes hold
// neighbouring pixels and whose warps share the channels.  Rows that no block can hold are read again for each step.
// The weights' gradients are summed in registers over a persistent block's rows, then over blocks in order.
// Sums of pairs and products of pairs are one instruction each.  2073600 x 64 in bfloat16: images 105 us forward (81 at the copy
// rate) and 250 backward (122), rows 120 and 189; 32768 x 4096 in float16: 128 (82) and 207 (123), where the latency of
// a block's sums is the bound.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "vi_heads.h"
#include "vi_heads_math.cuh"
#include "vi_internal.h"
#include "vi_rows.cuh"

namespace vi {
namespace heads {
namespace {

// Sum of S values over the lanes of a row: G lanes of a warp, or a block.  Every lane gets it, always added in the same
// order.  Of a block's up to 16 warps those that are not there left zeros (clear_sums).
template <int S, bool BLOCK>
__device__ __forceinline__ void row_sum(float (&s)[S], int lanes, float (*sh)[S][16], int& turn) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    if (!BLOCK && o >= lanes) continue;
#pragma unroll
    for (int i = 0; i < S; i++) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
  }
  if constexpr (BLOCK) {  // two buffers in turn: a barrier each sum
    if (threadIdx.x % 32 == 0) {
#pragma unroll
      for (int i = 0; i < S; i++) sh[turn][i][threadIdx.x / 32] = s[i];
    }
    __syncthreads();
    const bool few = blockDim.x <= 256;
#pragma unroll
    for (int i = 0; i < S; i++) {
      const float4 p = *(const float4*)&sh[turn][i][0], q = *(const float4*)&sh[turn][i][4];
      s[i] = ((p.x + p.y) + (p.z + p.w)) + ((q.x + q.y) + (q.z + q.w));
      if (!few) {
        const float4 u = *(const float4*)&sh[turn][i][8], v = *(const float4*)&sh[turn][i][12];
        s[i] += ((u.x + u.y) + (u.z + u.w)) + ((v.x + v.y) + (v.z + v.w));
      }
    }
    turn ^= 1;
  }
}
template <int N>
__device__ __forceinline__ void clear_sums(float* sh) {
  for (int i = threadIdx.x; i < N; i += blockDim.x) sh[i] = 0.0f;
  __syncthreads();
}

template <typename T, int VEC, int NV>
__device__ __forceinline__ void load_weights(Chunk<T, VEC> (&c)[NV], const void* w, float none, int K, int lanes, int lane) {
#pragma unroll
  for (int v = 0; v < NV; v++) {
    const int at = (v * lanes + lane) * VEC;
    if (w && at < K) c[v] = *(const Chunk<T, VEC>*)((const T*)w + at);
    else {
#pragma unroll
      for (int i = 0; i < VEC; i++) c[v].v[i] = from_f<T>(none);
    }
  }
}
template <typename T, int VEC, int NV>
__device__ __forceinline__ void store_row(const Chunk<T, VEC> (&c)[NV], const View& m, int64_t row, int K, int lanes, int lane) {
  T* p = (T*)m.p + row * m.rs;
#pragma unroll
  for (int v = 0; v < NV; v++) {
    const int at = (v * lanes + lane) * VEC;
    if (at < K) {
      if constexpr (VEC > 1) *(Chunk<T, VEC>*)(p + at) = c[v];
      else p[at * m.cs] = c[v].v[0];
    }
  }
}

constexpr int kRowThreads = 256;  // of a block whose rows belong to lanes
constexpr int kBlockMost = 512;   // of a block that a row belongs to

// A lane's elements of a row as pairs, which one instruction adds or multiplies.
template <typename T, int VEC, int NV>
__device__ __forceinline__ void pairs_of(const Chunk<T, VEC> (&c)[NV], float2 (&p)[(VEC * NV + 1) / 2]) {
#pragma unroll
  for (int i = 0; i < VEC * NV; i += 2)
    p[i / 2] = make_float2(to_f(c[i / VEC].v[i % VEC]), i + 1 < VEC * NV ? to_f(c[(i + 1) / VEC].v[(i + 1) % VEC]) : 0.0f);
}
template <typename T, int VEC, int NV>
__device__ __forceinline__ void chunks_of(const float2 (&p)[(VEC * NV + 1) / 2], Chunk<T, VEC> (&c)[NV]) {
#pragma unroll
  for (int i = 0; i < VEC * NV; i += 2) {
    if constexpr (sizeof(T) == 2 && VEC > 1) {
      ((uint32_t*)c[i / VEC].v)[i % VEC / 2] = pack2(p[i / 2], T());
    } else {
      c[i / VEC].v[i % VEC] = from_f<T>(p[i / 2].x);
      if (i + 1 < VEC * NV) c[(i + 1) / VEC].v[(i + 1) % VEC] = from_f<T>(p[i / 2].y);
    }
  }
}
// Whether element i of the lane lies in the row (whole vectors do or do not).
template <int VEC>
__device__ __forceinline__ bool in_row(int i, int lanes, int lane, int K) {
  return (i / VEC * lanes + lane) * VEC < K;
}
template <int N>
__device__ __forceinline__ float total(const float2 (&p)[N]) {
  float2 s[2] = {pair(0.0f), pair(0.0f)};
#pragma unroll
  for (int i = 0; i < N; i++) s[i & 1] = __fadd2_rn(s[i & 1], p[i]);
  s[0] = __fadd2_rn(s[0], s[1]);
  return s[0].x + s[0].y;
}

// R rows at a time for each group of lanes, so that short rows have loads in flight too.
template <typename T, int VEC, int NV, int R, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? kBlockMost : kRowThreads)
    norm_rows_forward(const __grid_constant__ NormArgs a, int lanes) {
  __shared__ __align__(16) float sh1[2][R][16], sh2[2][2 * R][16];
  constexpr int E = VEC * NV, P = (E + 1) / 2;
  if constexpr (BLOCK) clear_sums<32 * R>(&sh1[0][0][0]), clear_sums<64 * R>(&sh2[0][0][0]);
  const bool whole = a.K == lanes * E;  // of the lanes' elements none lies behind the row
  int turn1 = 0, turn2 = 0;
  const int lane = BLOCK ? threadIdx.x : threadIdx.x % lanes, group = BLOCK ? 0 : threadIdx.x / lanes;
  const int groups = BLOCK ? 1 : kRowThreads / lanes;
  const float inv = 1.0f / (float)a.K;
  float2 w[P], b[P];
  {
    Chunk<T, VEC> c[NV];
    load_weights(c, a.w, 1.0f, a.K, lanes, lane);
    pairs_of(c, w);
    load_weights(c, a.b, 0.0f, a.K, lanes, lane);
    pairs_of(c, b);
  }
  for (int64_t m0 = (int64_t)blockIdx.x * groups * R; m0 < a.M; m0 += (int64_t)gridDim.x * groups * R) {
    float2 x[R][P];
    {
      Chunk<T, VEC> c[R][NV];
#pragma unroll
      for (int r = 0; r < R; r++) load_row(c[r], a.x, min(m0 + r * groups + group, a.M - 1), a.K, lanes, lane);
#pragma unroll
      for (int r = 0; r < R; r++) pairs_of(c[r], x[r]);
    }
    float mean[R], q[2 * R];
#pragma unroll
    for (int r = 0; r < R; r++) mean[r] = total(x[r]);
    row_sum<R, BLOCK>(mean, lanes, sh1, turn1);
#pragma unroll
    for (int r = 0; r < R; r++) {
      mean[r] *= inv;
      float2 s1 = pair(0.0f), s2 = pair(0.0f);
#pragma unroll
      for (int i = 0; i < P; i++) {
        x[r][i] = __fadd2_rn(x[r][i], pair(-mean[r]));
        if (E % 2 && 2 * i + 1 >= E) x[r][i].y = 0.0f;
        if (!whole) {
          if (!in_row<VEC>(2 * i, lanes, lane, a.K)) x[r][i].x = 0.0f;
          if (2 * i + 1 < E && !in_row<VEC>(2 * i + 1, lanes, lane, a.K)) x[r][i].y = 0.0f;
        }
        s1 = __fadd2_rn(s1, x[r][i]);
        s2 = __ffma2_rn(x[r][i], x[r][i], s2);
      }
      q[2 * r] = s1.x + s1.y;
      q[2 * r + 1] = s2.x + s2.y;
    }
    row_sum<2 * R, BLOCK>(q, lanes, sh2, turn2);
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int64_t m = m0 + r * groups + group;
      const float shift = q[2 * r] * inv;
      const float rstd = 1.0f / sqrtf(fmaxf(fmaf(-shift, shift, q[2 * r + 1] * inv), 0.0f) + a.eps);
      if (m < a.M) {
#pragma unroll
        for (int i = 0; i < P; i++) x[r][i] = __ffma2_rn(__fmul2_rn(__fadd2_rn(x[r][i], pair(-shift)), pair(rstd)), w[i], b[i]);
        Chunk<T, VEC> y[NV];
        chunks_of(x[r], y);
        store_row(y, a.y, m, a.K, lanes, lane);
        if (a.stats && lane == 0) a.stats[m] = mean[r], a.stats[a.M + m] = shift, a.stats[2 * a.M + m] = rstd;
      }
    }
  }
}

// h and g are made twice of what memory gave, so that the registers leave room for two blocks of 256 threads on an SM (65536 x
// 512 with the weights' gradients: 52 us; with them held and the next rows on their way, one block, 97; three, spilling, 79).
template <typename T, int VEC, int NV, int R, bool BLOCK, int MOST>
__global__ void __launch_bounds__(BLOCK ? MOST : kRowThreads, BLOCK ? 512 / MOST : VEC * NV > 8 ? 2 : 3)
    norm_rows_backward(const __grid_constant__ NormArgs a, int lanes) {
  __shared__ __align__(16) float sh[2][2 * R][16];
  __shared__ float cols[BLOCK ? 1 : kRowThreads / 32][BLOCK ? 1 : 32 * VEC * NV];
  constexpr int E = VEC * NV, P = (E + 1) / 2;
  if constexpr (BLOCK) clear_sums<64 * R>(&sh[0][0][0]);
  int turn = 0;
  const int lane = BLOCK ? threadIdx.x : threadIdx.x % lanes, group = BLOCK ? 0 : threadIdx.x / lanes;
  const int groups = BLOCK ? 1 : kRowThreads / lanes;
  const float inv = 1.0f / (float)a.K;
  Chunk<T, VEC> w[NV];
  load_weights(w, a.w, 1.0f, a.K, lanes, lane);
  float2 dw[P], db[P];
#pragma unroll
  for (int i = 0; i < P; i++) dw[i] = db[i] = pair(0.0f);
  for (int64_t m0 = (int64_t)blockIdx.x * groups * R; m0 < a.M; m0 += (int64_t)gridDim.x * groups * R) {
    // of a row that is not there, and behind a row's end, all is 0 and adds nothing
    Chunk<T, VEC> x[R][NV], dy[R][NV];
    float mean[R], shift[R], rstd[R], q[2 * R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int64_t m = m0 + r * groups + group;
      const int K = m < a.M ? a.K : 0;
      load_row(x[r], a.x, m, K, lanes, lane);
      load_row(dy[r], a.dy, m, K, lanes, lane);
      mean[r] = shift[r] = rstd[r] = 0.0f;
      if (K) mean[r] = -a.stats[m], shift[r] = -a.stats[a.M + m], rstd[r] = a.stats[2 * a.M + m];
    }
    float2 wp[P];
    pairs_of(w, wp);
#pragma unroll
    for (int r = 0; r < R; r++) {
      float2 h[P], g[P], s1 = pair(0.0f), s2 = pair(0.0f);
      pairs_of(x[r], h);
      pairs_of(dy[r], g);
#pragma unroll
      for (int i = 0; i < P; i++) {
        h[i] = __fmul2_rn(__fadd2_rn(__fadd2_rn(h[i], pair(mean[r])), pair(shift[r])), pair(rstd[r]));
        dw[i] = __ffma2_rn(g[i], h[i], dw[i]);
        db[i] = __fadd2_rn(db[i], g[i]);
        g[i] = __fmul2_rn(g[i], wp[i]);
        s1 = __fadd2_rn(s1, g[i]);
        s2 = __ffma2_rn(g[i], h[i], s2);
      }
      q[2 * r] = s1.x + s1.y;
      q[2 * r + 1] = s2.x + s2.y;
    }
    if (!a.y.p) continue;
    row_sum<2 * R, BLOCK>(q, lanes, sh, turn);
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int64_t m = m0 + r * groups + group;
      if (m < a.M) {
        const float mg = -q[2 * r] * inv, mgh = -q[2 * r + 1] * inv;
        float2 h[P], g[P];
#pragma unroll
        for (int v = 0; v < NV; v++) {  // not to be kept from above
          uint32_t* t = (uint32_t*)x[r][v].v;
          if constexpr (sizeof(x[r][v]) >= 4) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(x[r][v]) / 4; i++) asm volatile("" : "+r"(t[i]));
          }
        }
        pairs_of(x[r], h);
        pairs_of(dy[r], g);
#pragma unroll
        for (int i = 0; i < P; i++) {
          h[i] = __fmul2_rn(__fadd2_rn(__fadd2_rn(h[i], pair(mean[r])), pair(shift[r])), pair(rstd[r]));
          g[i] = __fmul2_rn(__ffma2_rn(h[i], pair(mgh), __ffma2_rn(g[i], wp[i], pair(mg))), pair(rstd[r]));
        }
        Chunk<T, VEC> y[NV];
        chunks_of(g, y);
        store_row(y, a.y, m, a.K, lanes, lane);
      }
    }
  }
  if (!a.part) return;
  float* out = a.part + (int64_t)blockIdx.x * 2 * a.K;
#pragma unroll
  for (int which = 0; which < 2; which++) {
#pragma unroll
    for (int i = 0; i < E; i++) {
      const float2 v = which ? db[i / 2] : dw[i / 2];
      float s = i % 2 ? v.y : v.x;
      const int at = (i / VEC * lanes + lane) * VEC + i % VEC;
      if constexpr (BLOCK) {
        if (at < a.K) out[which * a.K + at] = s;
      } else {
        for (int o = lanes; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (threadIdx.x % 32 < lanes) cols[threadIdx.x / 32][at] = s;
      }
    }
    if constexpr (!BLOCK) {
      __syncthreads();
      for (int c = threadIdx.x; c < a.K; c += kRowThreads) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kRowThreads / 32; i++) s += cols[i][c];
        out[which * a.K + c] = s;
      }
      __syncthreads();
    }
  }
}

// Rows of any length: a block a row, which it reads again for each step.
template <typename T, bool BACKWARD>
__global__ void __launch_bounds__(512) norm_long_kernel(const __grid_constant__ NormArgs a) {
  __shared__ __align__(16) float sh1[2][1][16], sh2[2][2][16];
  clear_sums<32>(&sh1[0][0][0]);
  clear_sums<64>(&sh2[0][0][0]);
  int turn1 = 0, turn2 = 0;
  const float inv = 1.0f / (float)a.K;
  const T *w = (const T*)a.w, *b = (const T*)a.b;
  for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
    const T* x = (const T*)a.x.p + m * a.x.rs;
    const T* dy = (const T*)a.dy.p + m * a.dy.rs;
    T* y = (T*)a.y.p + m * a.y.rs;
    float q[2] = {0.0f, 0.0f};
    if constexpr (BACKWARD) {
      const float mean = a.stats[m], shift = a.stats[a.M + m], rstd = a.stats[2 * a.M + m];
      for (int k = threadIdx.x; k < a.K; k += 512) {
        const float h = (to_f(x[k * a.x.cs]) - mean - shift) * rstd, g = to_f(dy[k * a.dy.cs]) * (w ? to_f(w[k]) : 1.0f);
        q[0] += g;
        q[1] = fmaf(g, h, q[1]);
      }
      row_sum<2, true>(q, 512, sh2, turn2);
      for (int k = threadIdx.x; k < a.K; k += 512) {
        const float h = (to_f(x[k * a.x.cs]) - mean - shift) * rstd;
        y[k * a.y.cs] = from_f<T>(rstd * (fmaf(to_f(dy[k * a.dy.cs]), w ? to_f(w[k]) : 1.0f, -q[0] * inv) - h * (q[1] * inv)));
      }
    } else {
      float s[1] = {0.0f};
      for (int k = threadIdx.x; k < a.K; k += 512) s[0] += to_f(x[k * a.x.cs]);
      row_sum<1, true>(s, 512, sh1, turn1);
      const float mean = s[0] * inv;
      for (int k = threadIdx.x; k < a.K; k += 512) {
        const float d = to_f(x[k * a.x.cs]) - mean;
        q[0] += d;
        q[1] = fmaf(d, d, q[1]);
      }
      row_sum<2, true>(q, 512, sh2, turn2);
      const float shift = q[0] * inv, rstd = 1.0f / sqrtf(fmaxf(fmaf(-shift, shift, q[1] * inv), 0.0f) + a.eps);
      for (int k = threadIdx.x; k < a.K; k += 512)
        y[k * a.y.cs] = from_f<T>(fmaf((to_f(x[k * a.x.cs]) - mean - shift) * rstd, w ? to_f(w[k]) : 1.0f, b ? to_f(b[k]) : 0.0f));
      if (a.stats && threadIdx.x == 0) a.stats[m] = mean, a.stats[a.M + m] = shift, a.stats[2 * a.M + m] = rstd;
    }
  }
}

// The weights' gradients alone, of rows that no block holds: lanes along columns (or along rows, for images), a block
// 32 columns of a piece of the rows.
template <typename T>
__global__ void __launch_bounds__(256) norm_columns_kernel(const __grid_constant__ NormArgs a, int64_t rows, bool image) {
  __shared__ float sh[2][8][32];
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  const int64_t m0 = (int64_t)blockIdx.y * rows, m1 = min(a.M, m0 + rows);
  float* out = a.part + (int64_t)blockIdx.y * 2 * a.K;
  const T *x = (const T*)a.x.p, *dy = (const T*)a.dy.p;
  const auto add = [&](int64_t m, int64_t k, float& dw, float& db) {
    const float d = to_f(dy[m * a.dy.rs + k * a.dy.cs]);
    dw = fmaf(d, (to_f(x[m * a.x.rs + k * a.x.cs]) - a.stats[m] - a.stats[a.M + m]) * a.stats[2 * a.M + m], dw);
    db += d;
  };
  if (image) {  // a warp a column
    for (int c = ty; c < 32; c += 8) {
      const int64_t k = (int64_t)blockIdx.x * 32 + c;
      if (k >= a.K) break;
      float dw = 0.0f, db = 0.0f;
      for (int64_t m = m0 + tx; m < m1; m += 32) add(m, k, dw, db);
      for (int o = 16; o; o >>= 1) {
        dw += __shfl_xor_sync(0xffffffffu, dw, o);
        db += __shfl_xor_sync(0xffffffffu, db, o);
      }
      if (tx == 0) out[k] = dw, out[a.K + k] = db;
    }
    return;
  }
  const int64_t k = (int64_t)blockIdx.x * 32 + tx;
  float dw = 0.0f, db = 0.0f;
  if (k < a.K)
    for (int64_t m = m0 + ty; m < m1; m += 8) add(m, k, dw, db);
  sh[0][ty][tx] = dw, sh[1][ty][tx] = db;
  __syncthreads();
  if (ty < 2 && k < a.K) {
    float s = 0.0f;
    for (int i = 0; i < 8; i++) s += sh[ty][i][tx];
    out[ty * a.K + k] = s;
  }
}

// ---- images: pixels contiguous ----
// A lane holds VP neighbouring pixels, a warp every `warps`-th channel of them, up to R; `warps` warps make a tile of
// 32 VP pixels.  VP = 1: any strides.
template <typename T, int VP>
__device__ __forceinline__ void store_pixels(const Chunk<T, VP>& r, const View& m, int64_t row, int64_t c, int64_t M) {
  T* p = (T*)m.p + row * m.rs + c * m.cs;
  if (row + VP <= M) {
    *(Chunk<T, VP>*)p = r;
  } else {
#pragma unroll
    for (int j = 0; j < VP; j++)
      if (row + j < M) p[j * m.rs] = r.v[j];
  }
}
// Sum of a lane's VP values over the warps of its tile, in order; sh holds a block's lanes' values.
template <int VP>
__device__ __forceinline__ void tile_sum(float (&s)[VP], float* sh, int first, int warps, int lane) {
#pragma unroll
  for (int j = 0; j < VP; j++) s[j] = 0.0f;
  for (int i = 0; i < warps; i++) {
#pragma unroll
    for (int j = 0; j < VP; j++) s[j] += sh[((first + i) * VP + j) * 32 + lane];
  }
}
template <int VP>
__device__ __forceinline__ void tile_put(const float (&s)[VP], float* sh, int warp, int lane) {
#pragma unroll
  for (int j = 0; j < VP; j++) sh[(warp * VP + j) * 32 + lane] = s[j];
}

// One pixel or two as a value that one instruction adds or multiplies.
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float2 add(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float mul(float a, float b) { return a * b; }
__device__ __forceinline__ float2 mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float fma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float2 fma(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
// VP pixels of one channel as they lie in memory: a pair of 16-bit ones in a word (M is even then).
template <typename T, int VP>
struct Pixels;
template <typename T>
struct Pixels<T, 1> {
  using V = float;
  T t;
  __device__ __forceinline__ void load(const char* p) { t = *(const T*)p; }
  __device__ __forceinline__ V get() const { return to_f(t); }
  static __device__ __forceinline__ void store(V v, char* p) { *(T*)p = from_f<T>(v); }
  static __device__ __forceinline__ V all(float f) { return f; }
  static __device__ __forceinline__ float sum(V v) { return v; }
};
template <typename T>
struct Pixels<T, 2> {
  using V = float2;
  uint32_t w;
  __device__ __forceinline__ void load(const char* p) { w = *(const uint32_t*)p; }
  __device__ __forceinline__ V get() const {
    const T* t = (const T*)&w;
    return make_float2(to_f(t[0]), to_f(t[1]));
  }
  static __device__ __forceinline__ void store(V v, char* p) { *(uint32_t*)p = pack2(v, T()); }
  static __device__ __forceinline__ V all(float f) { return pair(f); }
  static __device__ __forceinline__ float sum(V v) { return v.x + v.y; }
};
// f(i, p) for each of the lane's channels, p the bytes of its pixels there; WHOLE: it has R of them.
template <typename T, int R, bool WHOLE, typename F>
__device__ __forceinline__ void each_channel(const View& m, int64_t row, int tw, int warps, int K, F f) {
  char* p = (char*)m.p + (row * m.rs + tw * m.cs) * (int64_t)sizeof(T);
  const int64_t step = warps * m.cs * (int64_t)sizeof(T);
#pragma unroll
  for (int i = 0; i < R; i++, p += step)
    if (WHOLE || tw + i * warps < K) f(i, p);
}
// Sum of a lane's value over the warps of its tile, in order, through sh (one value a thread of the block).
template <typename V>
__device__ __forceinline__ V tile_total(V v, V* sh, int warps) {
  if (warps == 1) return v;
  sh[threadIdx.x] = v;
  __syncthreads();
  const int first = threadIdx.x / 32 / warps * warps * 32 + threadIdx.x % 32;
  v = sh[first];
  for (int i = 1; i < warps; i++) v = add(v, sh[first + i * 32]);
  return v;
}

// The channels' weights, doubled, in shared memory: (w, w, b, b).
template <typename T>
__device__ __forceinline__ void stage_weights(float4* to, const NormArgs& a) {
  for (int c = threadIdx.x; c < a.K; c += blockDim.x) {
    const float w = a.w ? to_f(((const T*)a.w)[c]) : 1.0f, b = a.b ? to_f(((const T*)a.b)[c]) : 0.0f;
    to[c] = make_float4(w, w, b, b);
  }
  __syncthreads();
}
__device__ __forceinline__ float low(float4 q, float) { return q.x; }
__device__ __forceinline__ float2 low(float4 q, float2) { return make_float2(q.x, q.y); }
__device__ __forceinline__ float high(float4 q, float) { return q.z; }
__device__ __forceinline__ float2 high(float4 q, float2) { return make_float2(q.z, q.w); }

// A lane holds every warps-th channel of its pixels, up to R, as they lie in memory.  With one warp a tile (up to 64 channels)
// nothing is exchanged, and a warp has 8 KB on the way at a time.  Channels are reached by one pointer that steps: products of
// strides and a test a channel made 37 instructions an element (317 us at 2073600 x 64 in bfloat16, 105 so).
template <typename T, int VP, int R, bool WHOLE, int THREADS>
__global__ void __launch_bounds__(THREADS, R > 32 ? 2 : 3) norm_image_forward(const __grid_constant__ NormArgs a, int warps) {
  using X = Pixels<T, VP>;
  using V = typename X::V;
  extern __shared__ float4 weights[];
  V* const sh = (V*)(weights + a.K);  // three exchanges
  stage_weights<T>(weights, a);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, tw = warp % warps, per = THREADS / 32 / warps;
  const V inv = X::all(1.0f / (float)a.K);
  const int64_t tiles = (a.M + 32 * VP - 1) / (32 * VP);
  for (int64_t t0 = (int64_t)blockIdx.x * per; t0 < tiles; t0 += (int64_t)gridDim.x * per) {
    const int64_t m = ((t0 + warp / warps) * 32 + lane) * VP;
    const bool on = m < a.M;
    X x[R];
    V s = X::all(0.0f);
    if (on) {
      each_channel<T, R, WHOLE>(a.x, m, tw, warps, a.K, [&](int i, const char* p) { x[i].load(p); });
#pragma unroll
      for (int i = 0; i < R; i++)
        if (WHOLE || tw + i * warps < a.K) s = add(s, x[i].get());
    }
    const V mean = mul(tile_total(s, sh, warps), inv), less = mul(mean, X::all(-1.0f));
    V s1 = X::all(0.0f), s2 = s1;
    if (on) {
#pragma unroll
      for (int i = 0; i < R; i++)
        if (WHOLE || tw + i * warps < a.K) {
          const V d = add(x[i].get(), less);
          s1 = add(s1, d);
          s2 = fma(d, d, s2);
        }
    }
    const V shift = mul(tile_total(s1, sh + THREADS, warps), inv), sq = mul(tile_total(s2, sh + 2 * THREADS, warps), inv);
    if (!on) continue;
    V var = fma(mul(shift, X::all(-1.0f)), shift, sq), rstd;
#pragma unroll
    for (int j = 0; j < VP; j++) {
      ((float*)&rstd)[j] = 1.0f / sqrtf(fmaxf(((float*)&var)[j], 0.0f) + a.eps);
      if (a.stats && tw == 0) {
        a.stats[m + j] = ((const float*)&mean)[j];
        a.stats[a.M + m + j] = ((const float*)&shift)[j];
        a.stats[2 * a.M + m + j] = ((const float*)&rstd)[j];
      }
    }
    const V under = mul(shift, X::all(-1.0f));
    each_channel<T, R, WHOLE>(a.y, m, tw, warps, a.K, [&](int i, char* p) {
      const float4 q = weights[tw + i * warps];
      X::store(fma(mul(add(add(x[i].get(), less), under), rstd), low(q, V()), high(q, V())), p);
    });
  }
}

template <typename T, int VP, int R, bool WHOLE, int THREADS>
__global__ void __launch_bounds__(THREADS, 512 / THREADS) norm_image_backward(const __grid_constant__ NormArgs a, int warps) {
  using X = Pixels<T, VP>;
  using V = typename X::V;
  extern __shared__ float4 weights[];
  V* const sh = (V*)(weights + a.K);  // two exchanges, twice
  stage_weights<T>(weights, a);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, tw = warp % warps, per = THREADS / 32 / warps;
  const V inv = X::all(-1.0f / (float)a.K);
  V dw[R], db[R];
#pragma unroll
  for (int i = 0; i < R; i++) dw[i] = db[i] = X::all(0.0f);
  const int64_t tiles = (a.M + 32 * VP - 1) / (32 * VP);
  int turn = 0;
  for (int64_t t0 = (int64_t)blockIdx.x * per; t0 < tiles; t0 += (int64_t)gridDim.x * per) {
    const int64_t m = ((t0 + warp / warps) * 32 + lane) * VP;
    const bool on = m < a.M;
    X x[R], dy[R];
    V less = X::all(0.0f), under = less, rstd = less, q1 = less, q2 = less;
    if (on) {
      each_channel<T, R, WHOLE>(a.x, m, tw, warps, a.K, [&](int i, const char* p) { x[i].load(p); });
      each_channel<T, R, WHOLE>(a.dy, m, tw, warps, a.K, [&](int i, const char* p) { dy[i].load(p); });
#pragma unroll
      for (int j = 0; j < VP; j++) {
        ((float*)&less)[j] = -a.stats[m + j];
        ((float*)&under)[j] = -a.stats[a.M + m + j];
        ((float*)&rstd)[j] = a.stats[2 * a.M + m + j];
      }
#pragma unroll
      for (int i = 0; i < R; i++) {
        const int c = tw + i * warps;
        if (WHOLE || c < a.K) {
          const V h = mul(add(add(x[i].get(), less), under), rstd), d = dy[i].get(), g = mul(d, low(weights[c], V()));
          q1 = add(q1, g);
          q2 = fma(g, h, q2);
          dw[i] = fma(d, h, dw[i]);
          db[i] = add(db[i], d);
        }
      }
    }
    if (!a.y.p) continue;
    V* const s = sh + turn * 2 * THREADS;
    turn ^= 1;
    q1 = mul(tile_total(q1, s, warps), inv);
    q2 = mul(tile_total(q2, s + THREADS, warps), inv);
    if (!on) continue;
    each_channel<T, R, WHOLE>(a.y, m, tw, warps, a.K, [&](int i, char* p) {
      const V h = mul(add(add(x[i].get(), less), under), rstd), g = mul(dy[i].get(), low(weights[tw + i * warps], V()));
      X::store(mul(fma(h, q2, add(g, q1)), rstd), p);
    });
  }
  if (!a.part) return;
  float* out = a.part + ((int64_t)blockIdx.x * per + warp / warps) * 2 * a.K;
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int c = tw + i * warps;
    float s = X::sum(dw[i]), t = X::sum(db[i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    if (lane == 0 && c < a.K) out[c] = s, out[a.K + c] = t;
  }
}

// More channels than the warps hold: each step reads them again.
template <typename T, int VP, int R>
__global__ void __launch_bounds__(512) norm_image_long_forward(const __grid_constant__ NormArgs a, int warps) {
  extern __shared__ float sh[];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, tw = warp % warps, first = warp - tw, per = blockDim.x / 32 / warps;
  const int size = blockDim.x * VP;  // floats of one exchange
  const float inv = 1.0f / (float)a.K;
  const T *w = (const T*)a.w, *b = (const T*)a.b;
  const int64_t tiles = (a.M + 32 * VP - 1) / (32 * VP);
  for (int64_t t0 = (int64_t)blockIdx.x * per; t0 < tiles; t0 += (int64_t)gridDim.x * per) {
    const int64_t m = ((t0 + warp / warps) * 32 + lane) * VP;
    Chunk<T, VP> x[R];
    const auto load = [&](int k0) {
#pragma unroll
      for (int i = 0; i < R; i++)
        if (k0 + tw + i * warps < a.K) x[i] = load_pixels<T, VP>(a.x, m, k0 + tw + i * warps, a.M);
    };
    const auto channels = [&](auto f) {
      if (m >= a.M) return;
      for (int k0 = 0; k0 < a.K; k0 += R * warps) {
        load(k0);
#pragma unroll
        for (int i = 0; i < R; i++)
          if (k0 + tw + i * warps < a.K) f(x[i], k0 + tw + i * warps);
      }
    };
    float mean[VP] = {}, d1[VP] = {}, d2[VP] = {}, rstd[VP];
    channels([&](const Chunk<T, VP>& v, int) {
#pragma unroll
      for (int j = 0; j < VP; j++) mean[j] += to_f(v.v[j]);
    });
    if (warps > 1) {
      tile_put(mean, sh, warp, lane);
      __syncthreads();
      tile_sum(mean, sh, first, warps, lane);
    }
#pragma unroll
    for (int j = 0; j < VP; j++) mean[j] *= inv;
    channels([&](const Chunk<T, VP>& v, int) {
#pragma unroll
      for (int j = 0; j < VP; j++) {
        const float d = to_f(v.v[j]) - mean[j];
        d1[j] += d;
        d2[j] = fmaf(d, d, d2[j]);
      }
    });
    if (warps > 1) {
      tile_put(d1, sh + size, warp, lane);
      tile_put(d2, sh + 2 * size, warp, lane);
      __syncthreads();
      tile_sum(d1, sh + size, first, warps, lane);
      tile_sum(d2, sh + 2 * size, first, warps, lane);
    }
#pragma unroll
    for (int j = 0; j < VP; j++) {
      d1[j] *= inv;
      rstd[j] = 1.0f / sqrtf(fmaxf(fmaf(-d1[j], d1[j], d2[j] * inv), 0.0f) + a.eps);
      if (a.stats && tw == 0 && m + j < a.M)
        a.stats[m + j] = mean[j], a.stats[a.M + m + j] = d1[j], a.stats[2 * a.M + m + j] = rstd[j];
    }
    channels([&](const Chunk<T, VP>& v, int c) {
      const float wc = w ? to_f(w[c]) : 1.0f, bc = b ? to_f(b[c]) : 0.0f;
      Chunk<T, VP> y;
#pragma unroll
      for (int j = 0; j < VP; j++) y.v[j] = from_f<T>(fmaf((to_f(v.v[j]) - mean[j] - d1[j]) * rstd[j], wc, bc));
      store_pixels<T, VP>(y, a.y, m, c, a.M);
    });
  }
}

template <typename T, int VP, int R>
__global__ void __launch_bounds__(512) norm_image_long_backward(const __grid_constant__ NormArgs a, int warps) {
  extern __shared__ float sh[];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, tw = warp % warps, first = warp - tw, per = blockDim.x / 32 / warps;
  const int size = blockDim.x * VP;
  const float inv = 1.0f / (float)a.K;
  const T* w = (const T*)a.w;
  const int64_t tiles = (a.M + 32 * VP - 1) / (32 * VP);
  int turn = 0;
  for (int64_t t0 = (int64_t)blockIdx.x * per; t0 < tiles; t0 += (int64_t)gridDim.x * per) {
    const int64_t m = ((t0 + warp / warps) * 32 + lane) * VP;
    Chunk<T, VP> x[R], dy[R];
    const auto load = [&](int k0) {
#pragma unroll
      for (int i = 0; i < R; i++) {
        const int c = k0 + tw + i * warps;
        if (c < a.K) x[i] = load_pixels<T, VP>(a.x, m, c, a.M), dy[i] = load_pixels<T, VP>(a.dy, m, c, a.M);
      }
    };
    const auto channels = [&](auto f) {
      if (m >= a.M) return;
      for (int k0 = 0; k0 < a.K; k0 += R * warps) {
        load(k0);
#pragma unroll
        for (int i = 0; i < R; i++)
          if (k0 + tw + i * warps < a.K) f(i, k0 + tw + i * warps);
      }
    };
    float mean[VP], shift[VP], rstd[VP], q1[VP] = {}, q2[VP] = {};
#pragma unroll
    for (int j = 0; j < VP; j++) {  // h of a pixel that is not there: 0
      const bool in = m + j < a.M;
      mean[j] = in ? a.stats[m + j] : 0.0f;
      shift[j] = in ? a.stats[a.M + m + j] : 0.0f;
      rstd[j] = in ? a.stats[2 * a.M + m + j] : 0.0f;
    }
    channels([&](int i, int c) {
      const float wc = w ? to_f(w[c]) : 1.0f;
#pragma unroll
      for (int j = 0; j < VP; j++) {
        const float h = (to_f(x[i].v[j]) - mean[j] - shift[j]) * rstd[j], d = to_f(dy[i].v[j]), g = d * wc;
        q1[j] += g;
        q2[j] = fmaf(g, h, q2[j]);
      }
    });
    if (!a.y.p) continue;
    if (warps > 1) {  // two exchanges in turn: one barrier a tile
      float* s = sh + turn * 2 * size;
      tile_put(q1, s, warp, lane);
      tile_put(q2, s + size, warp, lane);
      __syncthreads();
      tile_sum(q1, s, first, warps, lane);
      tile_sum(q2, s + size, first, warps, lane);
      turn ^= 1;
    }
    channels([&](int i, int c) {
      const float wc = w ? to_f(w[c]) : 1.0f;
      Chunk<T, VP> y;
#pragma unroll
      for (int j = 0; j < VP; j++) {
        const float h = (to_f(x[i].v[j]) - mean[j] - shift[j]) * rstd[j];
        y.v[j] = from_f<T>(rstd[j] * (fmaf(to_f(dy[i].v[j]), wc, -q1[j] * inv) - h * (q2[j] * inv)));
      }
      store_pixels<T, VP>(y, a.y, m, c, a.M);
    });
  }
}

// ---- host ----
// One call: what is launched, in how many blocks; `pieces` partial sums of the weights' gradients.
struct Call {
  const NormArgs& a;
  int sms;
  cudaStream_t s;
  bool dry;
  int pieces = 0, launches = 0;
  cudaError_t rc = cudaSuccess;

  // `units` pieces of work, one a block at a time; `per` partial sums a block.
  template <auto kernel>
  void run(int threads, size_t smem, int64_t units, int lanes, int per) {
    static std::atomic<int> known[33];  // blocks per SM by warps a block (shared memory differs little)
    int n = known[threads / 32].load(std::memory_order_relaxed);
    if (n <= 0) {
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) == cudaSuccess && n > 0)
        known[threads / 32].store(n, std::memory_order_relaxed);
      else
        cudaGetLastError(), n = 1;
    }
    const int64_t blocks = std::min<int64_t>(units, (int64_t)sms * n);
    pieces = (int)blocks * per;
    if (dry || (!a.y.p && !a.part)) return;
    kernel<<<(unsigned)blocks, threads, smem, s>>>(a, lanes);
    rc = cudaPeekAtLastError();
    launches++;
  }
  template <typename T>
  void run_long(bool backward, bool image) {
    const unsigned blocks = (unsigned)std::min<int64_t>(a.M, (int64_t)sms * 4);
    if (!dry && a.y.p) {
      if (backward) norm_long_kernel<T, true><<<blocks, 512, 0, s>>>(a);
      else norm_long_kernel<T, false><<<blocks, 512, 0, s>>>(a);
      rc = cudaPeekAtLastError();
      launches++;
    }
    if (backward) columns<T>(image);
  }
  template <typename T>
  void columns(bool image) {
    const int64_t strips = ceil_div(a.K, 32);
    const int64_t rows = std::max<int64_t>(64, ceil_div(a.M, std::max<int64_t>(1, sms * 8 / strips)));
    pieces = (int)ceil_div(a.M, rows);
    if (dry || !a.part || rc != cudaSuccess) return;
    norm_columns_kernel<T><<<dim3((unsigned)strips, (unsigned)pieces), 256, 0, s>>>(a, rows, image);
    rc = cudaPeekAtLastError();
    launches++;
  }
};

// Rows of `units` vectors or elements by lanes, or by a block: false where this shape does not hold them.
template <typename T, int VEC, int NV, int R, bool BACKWARD>
bool rows_lanes(Call& c, int64_t units) {
  if (units > 32 * NV) return false;
  const int lanes = NV > 1 ? 32 : pow2_at_least(units);
  const int64_t work = ceil_div(c.a.M, (int64_t)kRowThreads / lanes * R);
  if constexpr (BACKWARD) c.run<norm_rows_backward<T, VEC, NV, R, false, 1>>(kRowThreads, 0, work, lanes, 1);
  else c.run<norm_rows_forward<T, VEC, NV, R, false>>(kRowThreads, 0, work, lanes, 1);
  return true;
}
template <typename T, int VEC, int NV, bool BACKWARD>
bool rows_block(Call& c, int64_t units) {
  if (units > (int64_t)kBlockMost * NV) return false;
  const int threads = (int)ceil_div(ceil_div(units, NV), 32) * 32;
  if constexpr (BACKWARD) {
    if (threads <= 256) c.run<norm_rows_backward<T, VEC, NV, 1, true, 256>>(threads, 0, c.a.M, threads, 1);
    else c.run<norm_rows_backward<T, VEC, NV, 1, true, kBlockMost>>(threads, 0, c.a.M, threads, 1);
  } else c.run<norm_rows_forward<T, VEC, NV, 1, true>>(threads, 0, c.a.M, threads, 1);
  return true;
}
template <typename T, int VP, int R, bool BACKWARD, int THREADS = 256>
void image_tiles(Call& c) {
  const int warps = pow2_at_least(ceil_div(c.a.K, R)), per = THREADS / 32 / warps;
  const int64_t work = ceil_div(ceil_div(c.a.M, 32 * VP), per);
  const size_t smem = (size_t)c.a.K * 16 + (size_t)THREADS * VP * 4 * (BACKWARD ? 4 : 3);
  const auto run = [&](auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
    if constexpr (BACKWARD) c.run<norm_image_backward<T, VP, R, WHOLE, THREADS>>(THREADS, smem, work, warps, per);
    else c.run<norm_image_forward<T, VP, R, WHOLE, THREADS>>(THREADS, smem, work, warps, per);
  };
  if (c.a.K == R * warps) run(std::true_type());
  else run(std::false_type());
}
template <typename T, int VP, int R, bool BACKWARD>
void image_long(Call& c) {
  const int64_t work = ceil_div(c.a.M, 32 * VP);
  const size_t smem = (size_t)512 * VP * 4 * (BACKWARD ? 4 : 3);
  if constexpr (BACKWARD) c.run<norm_image_long_backward<T, VP, R>>(512, smem, work, 16, 1);
  else c.run<norm_image_long_forward<T, VP, R>>(512, smem, work, 16, 1);
}

template <typename T>
void norm_call(Call& c, bool backward) {
  const NormArgs& a = c.a;
  constexpr int VEC = 16 / (int)sizeof(T);
  // An image of many channels and so few pixels that its tiles leave most SMs idle goes by rows, a block each, element by
  // element (36 pixels x 7216 channels: 890 us by tiles).
  const bool image = a.x.rs == 1 && a.x.cs != 1 && a.M > 1 && (a.K <= (backward ? 256 : 512) || a.M > 8192);
  const auto wide = [&](int n, bool along_rows) {
    for (const View* v : {&a.x, &a.dy, &a.y})
      if (v->p && !moves<T>(*v, n, along_rows)) return false;
    return along_rows || (a.K % n == 0 && (uintptr_t)a.w % (n * sizeof(T)) == 0 && (uintptr_t)a.b % (n * sizeof(T)) == 0);
  };
  if (image) {
    constexpr int VP = 4 / (int)sizeof(T);
    const bool pairs = a.M % VP == 0 && wide(VP, true);  // else any strides
    if (!backward) {
      if (a.K <= 512) {
        if (a.K <= 16) pairs ? image_tiles<T, VP, 16, false>(c) : image_tiles<T, 1, 16, false>(c);
        else if (a.K <= 32) pairs ? image_tiles<T, VP, 32, false>(c) : image_tiles<T, 1, 32, false>(c);
        else pairs ? image_tiles<T, VP, 64, false>(c) : image_tiles<T, 1, 64, false>(c);
      } else {
        pairs ? image_long<T, VP, 32, false>(c) : image_long<T, 1, 32, false>(c);
      }
    } else if (a.K <= 128) {
      pairs ? image_tiles<T, VP, 16, true>(c) : image_tiles<T, 1, 16, true>(c);
    } else if (a.K <= 256) {
      pairs ? image_tiles<T, VP, 16, true, 512>(c) : image_tiles<T, 1, 16, true, 512>(c);
    } else {
      if (a.y.p) pairs ? image_long<T, VP, 16, true>(c) : image_long<T, 1, 16, true>(c);
      c.columns<T>(true);
    }
    return;
  }
  const int64_t n = a.K / VEC;
  if (wide(VEC, false)) {
    if (!backward) {
      if (rows_lanes<T, VEC, 1, 4, false>(c, n) || rows_lanes<T, VEC, 2, 2, false>(c, n) || rows_lanes<T, VEC, 4, 1, false>(c, n) ||
          (n > 256 && rows_block<T, VEC, 4, false>(c, n)) ||  // fewer warps to add up (32768 x 4096: 146 us with 2, 128)
          rows_block<T, VEC, 2, false>(c, n) || rows_block<T, VEC, 4, false>(c, n))
        return;
    } else {  // sums of 16 columns a lane at most, in registers
      if (rows_lanes<T, VEC, 1, 2, true>(c, n) || rows_lanes<T, VEC, 2, 1, true>(c, n)) return;
      if constexpr (sizeof(T) == 4) {
        if (rows_lanes<T, VEC, 4, 1, true>(c, n) || rows_block<T, VEC, 4, true>(c, n)) return;
      } else {
        if (rows_block<T, VEC, 2, true>(c, n)) return;
      }
    }
  } else if (!backward) {
    if (rows_lanes<T, 1, 1, 4, false>(c, a.K) || rows_lanes<T, 1, 4, 1, false>(c, a.K) || rows_lanes<T, 1, 16, 1, false>(c, a.K) ||
        rows_block<T, 1, 8, false>(c, a.K) || rows_block<T, 1, 16, false>(c, a.K))
      return;
  } else {
    if (rows_lanes<T, 1, 1, 2, true>(c, a.K) || rows_lanes<T, 1, 4, 1, true>(c, a.K) || rows_lanes<T, 1, 16, 1, true>(c, a.K) ||
        rows_block<T, 1, 8, true>(c, a.K) || rows_block<T, 1, 16, true>(c, a.K))
      return;
  }
  c.run_long<T>(backward, image);
}

}  // namespace

int norm_pieces(int dtype, const NormArgs& a, int sms) {
  Call c{a, sms, nullptr, true};
  if (dtype == VI_F32) norm_call<float>(c, true);
  else if (dtype == VI_F16) norm_call<__half>(c, true);
  else norm_call<__nv_bfloat16>(c, true);
  return c.pieces;
}

cudaError_t launch_norm(int dtype, const NormArgs& a, bool backward, int sms, cudaStream_t s, int* launches) {
  Call c{a, sms, s, false};
  if (dtype == VI_F32) norm_call<float>(c, backward);
  else if (dtype == VI_F16) norm_call<__half>(c, backward);
  else norm_call<__nv_bfloat16>(c, backward);
  *launches += c.launches;
  return c.rc;
}

}  // namespace heads
}  // namespace vi
