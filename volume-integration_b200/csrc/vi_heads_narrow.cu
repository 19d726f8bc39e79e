// linear_act on images of few channels (K <= 8), the first layer behind the renderer's
// feature image: out^T = act(W x + b), x [K][pixels], out [N][pixels].
//
// With so few products per element memory is the bound (K = 4, N = 64, float32: 8 FMA and 4
// bytes an output), so the FP32 cores do it, 4 pixels a thread, straight from the
// image and back to it, 16 bytes a lane (8 beside 16-bit types).  The sum runs over k in order and
// the bias is added last.  The backward keeps no act': it computes z again (K FMA beside the
// N-fold traffic that storing it would cost), and in one pass over dy forms
//   s = dy act'(z), dx[k] += s w[n][k] in registers, dW[n][k] += s x[k], db[n] += s,
// the latter two summed over a warp for every n, kept per warp in shared memory, and written as one
// piece per block.
#include <algorithm>

#include "vi_heads.h"
#include "vi_heads_math.cuh"
#include "vi_internal.h"

namespace vi {
namespace heads {
namespace {

constexpr int kVec = 4;           // pixels a thread
constexpr int kThreads = 128;
constexpr int kTile = kVec * kThreads;  // pixels a block and step

template <typename T>
struct Quad {
  using type = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
};

// Four neighbouring pixels, `left` of them existing.
template <typename T>
__device__ __forceinline__ void load4(const T* p, int left, bool vec, float v[4]) {
  if (vec && left >= 4) {
    const typename Quad<T>::type q = *(const typename Quad<T>::type*)p;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = to_f(((const T*)&q)[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = i < left ? to_f(p[i]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int left, bool vec, const float v[4]) {
  if (vec && left >= 4) {
    typename Quad<T>::type q;
#pragma unroll
    for (int i = 0; i < 4; i++) ((T*)&q)[i] = from_f<T>(v[i]);
    *(typename Quad<T>::type*)p = q;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < left) p[i] = from_f<T>(v[i]);
  }
}

// Weights [n][KT] and bias [n] of rows [n0, n0 + n) in shared memory, float32, zeros beyond K.
template <typename T, int KT>
__device__ __forceinline__ void load_weights(const NarrowArgs& a, int n0, int n, float* sw, float* sb) {
  for (int i = threadIdx.x; i < n * KT; i += kThreads) {
    const int r = i / KT, k = i % KT;
    sw[i] = k < a.K ? to_f(((const T*)a.w.p)[(int64_t)(n0 + r) * a.w.rs + (int64_t)k * a.w.cs]) : 0.0f;
  }
  for (int i = threadIdx.x; i < n; i += kThreads) sb[i] = a.bias ? to_f(((const T*)a.bias)[n0 + i]) : 0.0f;
}

template <int KT>
__device__ __forceinline__ void dot4(const float (&x)[KT][4], const float* w, float bias, float2& lo, float2& hi) {
  lo = hi = pair(0.0f);
#pragma unroll
  for (int k = 0; k < KT; k++) {
    lo = __ffma2_rn(make_float2(x[k][0], x[k][1]), pair(w[k]), lo);
    hi = __ffma2_rn(make_float2(x[k][2], x[k][3]), pair(w[k]), hi);
  }
  lo = __fadd2_rn(lo, pair(bias));
  hi = __fadd2_rn(hi, pair(bias));
}

// blockIdx.x strides over pixels, blockIdx.y takes a.span channels.
template <typename T, int KT, int ACT>
__global__ void __launch_bounds__(kThreads) narrow_forward_kernel(const __grid_constant__ NarrowArgs a) {
  extern __shared__ float sh[];
  const int n0 = blockIdx.y * a.span, n = min(a.span, a.N - n0);
  float *sw = sh, *sb = sh + a.span * KT;
  load_weights<T, KT>(a, n0, n, sw, sb);
  __syncthreads();
  for (int64_t m = (int64_t)blockIdx.x * kTile + threadIdx.x * kVec; m < a.M; m += (int64_t)gridDim.x * kTile) {
    const int left = (int)min((int64_t)4, a.M - m);
    float x[KT][4];
#pragma unroll
    for (int k = 0; k < KT; k++) {
      if (k < a.K) {
        load4((const T*)a.x.p + m + k * a.x.cs, left, a.vec, x[k]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[k][i] = 0.0f;
      }
    }
    T* y = (T*)a.y.p + m + n0 * a.y.cs;
    const T* r = a.res.p ? (const T*)a.res.p + m + n0 * a.res.cs : nullptr;
#pragma unroll 4
    for (int j = 0; j < n; j++) {
      float2 z[2], v[2], d;
      dot4<KT>(x, sw + j * KT, sb[j], z[0], z[1]);
      activate<ACT, sizeof(T) == 4, false>(z[0], v[0], d);
      activate<ACT, sizeof(T) == 4, false>(z[1], v[1], d);
      if (r) {
        float q[4];
        load4(r + j * a.res.cs, left, a.vec, q);
        v[0] = __fadd2_rn(v[0], make_float2(q[0], q[1]));
        v[1] = __fadd2_rn(v[1], make_float2(q[2], q[3]));
      }
      const float o[4] = {v[0].x, v[0].y, v[1].x, v[1].y};
      store4(y + j * a.y.cs, left, a.vec, o);
    }
  }
}

// Sums of V (a power of two) values over a warp.  In each of the first steps a lane hands half of
// its values to its partner and keeps the other half, so they cost V + log2(32 / V) - 1
// exchanges instead of 5 V.  The sum of value `index` is returned to its 32 / V lanes.
template <int V>
__device__ __forceinline__ float warp_sums(float (&t)[V], int lane, int& index) {
  index = 0;
  int o = 16;
#pragma unroll
  for (int h = V / 2; h; h /= 2, o /= 2) {
    const bool up = lane & o;
    if (up) index += h;
#pragma unroll
    for (int i = 0; i < h; i++) {
      const float give = up ? t[i] : t[i + h], keep = up ? t[i + h] : t[i];
      t[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  float s = t[0];
#pragma unroll
  for (; o; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// The backward: every block runs through all channels of its pixels.
template <typename T, int KT, int ACT>
__global__ void __launch_bounds__(kThreads) narrow_backward_kernel(const __grid_constant__ NarrowArgs a) {
  extern __shared__ float sh[];
  constexpr int kSums = KT + 1;
  float *sw = sh, *sb = sw + a.N * KT, *acc = sb + a.N;  // acc: [warps][N][KT + 1]
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  load_weights<T, KT>(a, 0, a.N, sw, sb);
  for (int i = threadIdx.x; i < kThreads / 32 * a.N * kSums; i += kThreads) acc[i] = 0.0f;
  __syncthreads();
  float* mine = acc + warp * a.N * kSums;
  constexpr int kQuads = KT <= 4 ? 2 : 1;  // groups of 4 pixels a thread, so that a warp's sum serves 256 pixels
  constexpr int kStep = kTile * kQuads;
  // whole warps stay in the loop: its sums are warps' sums
  for (int64_t base = (int64_t)blockIdx.x * kStep + warp * 32 * kVec * kQuads; base < a.M; base += (int64_t)gridDim.x * kStep) {
    float x[kQuads][KT][4], dx[kQuads][KT][4];
    int64_t m[kQuads];
    int left[kQuads];
#pragma unroll
    for (int q = 0; q < kQuads; q++) {
      m[q] = base + (q * 32 + lane) * kVec;
      left[q] = (int)max((int64_t)0, min((int64_t)4, a.M - m[q]));
#pragma unroll
      for (int k = 0; k < KT; k++) {
        if (k < a.K) {
          load4((const T*)a.x.p + m[q] + k * a.x.cs, left[q], a.vec, x[q][k]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++) x[q][k][i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) dx[q][k][i] = 0.0f;
      }
    }
    const T* dy = (const T*)a.y.p;
    constexpr int kAhead = 4;  // channels whose gradients are in flight at a time
    for (int j0 = 0; j0 < a.N; j0 += kAhead) {
      float g[kAhead][kQuads][4];
#pragma unroll
      for (int u = 0; u < kAhead; u++)
#pragma unroll
        for (int q = 0; q < kQuads; q++)
          if (j0 + u < a.N) load4(dy + (j0 + u) * a.y.cs + m[q], left[q], a.vec, g[u][q]);
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const int j = j0 + u;
        if (j >= a.N) break;
        const float* w = sw + j * KT;
        constexpr int kSlots = KT <= 4 ? 8 : 16;
        float t[kSlots] = {};
#pragma unroll
        for (int q = 0; q < kQuads; q++) {
          float2 z[2], v, d[2];
          if (ACT == VI_ACT_NONE) {
            d[0] = d[1] = pair(1.0f);
          } else {
            dot4<KT>(x[q], w, sb[j], z[0], z[1]);
            activate<ACT, sizeof(T) == 4, true>(z[0], v, d[0]);
            activate<ACT, sizeof(T) == 4, true>(z[1], v, d[1]);
          }
          // pixels beyond the image add nothing, whatever act' is there
          const float s[4] = {left[q] > 0 ? g[u][q][0] * d[0].x : 0.0f, left[q] > 1 ? g[u][q][1] * d[0].y : 0.0f,
            left[q] > 2 ? g[u][q][2] * d[1].x : 0.0f, left[q] > 3 ? g[u][q][3] * d[1].y : 0.0f};
#pragma unroll
          for (int k = 0; k < KT; k++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
              dx[q][k][i] = fmaf(s[i], w[k], dx[q][k][i]);
              t[k] = fmaf(s[i], x[q][k][i], t[k]);
            }
          }
          t[KT] += (s[0] + s[1]) + (s[2] + s[3]);
        }
        if (a.part) {
          int index;
          const float sum = warp_sums<kSlots>(t, lane, index);
          if (lane % (32 / kSlots) == 0 && index < kSums) mine[j * kSums + index] += sum;
        }
      }
    }
    if (a.dx.p) {
#pragma unroll
      for (int q = 0; q < kQuads; q++)
#pragma unroll
        for (int k = 0; k < KT; k++)
          if (k < a.K && left[q] > 0) store4((T*)a.dx.p + m[q] + k * a.dx.cs, left[q], a.vec, dx[q][k]);
    }
  }
  if (!a.part) return;
  __syncthreads();
  for (int i = threadIdx.x; i < a.N * kSums; i += kThreads) {
    float t = 0.0f;
    for (int w = 0; w < kThreads / 32; w++) t += acc[w * a.N * kSums + i];
    a.part[(int64_t)blockIdx.x * a.N * kSums + i] = t;
  }
}

template <typename T, int KT, int ACT>
cudaError_t run(const NarrowArgs& args, bool backward, int blocks, int sms, cudaStream_t s) {
  NarrowArgs a = args;
  if (backward) {
    const size_t smem = ((size_t)a.N * (KT + 1) + (size_t)kThreads / 32 * a.N * (KT + 1)) * 4;
    narrow_backward_kernel<T, KT, ACT><<<blocks, kThreads, smem, s>>>(a);
  } else {
    // few pixels: channels are spread over blocks too
    const int64_t tiles = (a.M + kTile - 1) / kTile;
    const int64_t ways = std::max<int64_t>(1, std::min<int64_t>((sms * 4 + tiles - 1) / tiles, (a.N + 7) / 8));
    a.span = std::min<int>((int)((a.N + ways - 1) / ways), 1024);
    const dim3 grid((unsigned)std::min<int64_t>(tiles, (int64_t)sms * 16), (unsigned)((a.N + a.span - 1) / a.span));
    narrow_forward_kernel<T, KT, ACT><<<grid, kThreads, (size_t)a.span * (KT + 1) * 4, s>>>(a);
  }
  return cudaPeekAtLastError();
}
template <typename T, int KT>
cudaError_t run_act(const NarrowArgs& a, bool backward, int blocks, int sms, cudaStream_t s) {
  switch (a.act) {
    case VI_ACT_RELU: return run<T, KT, VI_ACT_RELU>(a, backward, blocks, sms, s);
    case VI_ACT_SILU: return run<T, KT, VI_ACT_SILU>(a, backward, blocks, sms, s);
    case VI_ACT_GELU: return run<T, KT, VI_ACT_GELU>(a, backward, blocks, sms, s);
    case VI_ACT_SIGMOID: return run<T, KT, VI_ACT_SIGMOID>(a, backward, blocks, sms, s);
    default: return run<T, KT, VI_ACT_NONE>(a, backward, blocks, sms, s);
  }
}

bool image(const View& v) { return !v.p || (v.rs == 1 && v.cs > 1); }

}  // namespace

// The limit on N is the backward's, whose warps keep the sums of every channel in shared memory
// (46 KB at N = 256, K = 8); a forward without gradients follows it, so that it gives the same bits.
bool narrow_forward(int64_t N, int64_t K, const View& x, const View& y, const View& res) {
  return K <= kNarrowK && N <= kNarrowN && image(x) && image(y) && image(res);
}
bool narrow_backward(int64_t N, int64_t K, const View& x, const View& dy, const View& dx) {
  return K <= kNarrowK && N <= kNarrowN && image(x) && image(dy) && image(dx);
}
int narrow_sums(int64_t K) { return K <= 4 ? 5 : 9; }
int narrow_blocks(int64_t M, int sms) {
  return (int)std::max<int64_t>(1, std::min<int64_t>((M + kTile - 1) / kTile, (int64_t)sms * 3));
}

cudaError_t launch_narrow(int dtype, const NarrowArgs& args, bool backward, int blocks, int sms, cudaStream_t s) {
  NarrowArgs a = args;
  // vector accesses need every column of every matrix on a boundary of four elements
  const uintptr_t es = dtype == VI_F32 ? 4 : 2;
  a.vec = true;
  for (const View& v : {a.x, a.y, a.res, a.dx})
    if (v.p && ((uintptr_t)v.p % (4 * es) || v.cs % 4)) a.vec = false;
  if (dtype == VI_F32) return a.K <= 4 ? run_act<float, 4>(a, backward, blocks, sms, s) : run_act<float, 8>(a, backward, blocks, sms, s);
  if (dtype == VI_F16)
    return a.K <= 4 ? run_act<__half, 4>(a, backward, blocks, sms, s) : run_act<__half, 8>(a, backward, blocks, sms, s);
  return a.K <= 4 ? run_act<__nv_bfloat16, 4>(a, backward, blocks, sms, s)
                  : run_act<__nv_bfloat16, 8>(a, backward, blocks, sms, s);
}

}  // namespace heads
}  // namespace vi
