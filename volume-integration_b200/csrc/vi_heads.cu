// Per-pixel heads: dense layers and the label loss on rendered feature images.
//
// Mathematics.  The products are one z = x W^T + b with an epilogue:
//   linear_act            y = act(z) + r
//                         s = dy * act'(z); dx = s W; dW = s^T x; db = sum_m s
//   linear_cross_entropy  l_m = log sum_v exp z_mv - z_m,t
//                         G = g_m (softmax(z) - onehot(t)); dx = G W; dW = G^T x; db = sum_m G
// Beside them, with kernels of their own: layer_norm (vi_norm.cu), linear_act in 8-bit integers (vi_quant.cu,
// vi_heads_int8.cu) and sample_labels (vi_sample.cu).
// Sums, the softmax's maximum and sum, and biases' gradients are float32; sums over
// rows are split into pieces that are added in a fixed order, so results do not
// depend on scheduling.
#include <algorithm>
#include <atomic>
#include <cstdio>
#include <type_traits>
#include <utility>

#include "vi_heads.h"
#include "vi_heads_math.cuh"
#include "vi_internal.h"

namespace vi {
namespace heads {
namespace {

// One operand laid out for the tensor cores: 16-bit planes, rows of `inner`
// elements `ld` apart, a multiple of 8; 0 in rows whose coef is 0.
struct PackJob {
  View src;
  const float* coef;  // [rows] or null
  int64_t rows, k;
  void* dst;
  int64_t ld, plane;
  int k_major;
};
struct PackJobs {
  PackJob j[2];
};

// The 16-bit element type the tensor cores read for T.
template <typename T>
using Cell16 = typename std::conditional<std::is_same<T, __half>::value, __half, __nv_bfloat16>::type;

// Eight elements `step` apart, n of them existing; 16 bytes at a time where they lie so.
template <typename T>
__device__ __forceinline__ void load8(const T* s, int64_t step, int n, float v[8]) {
  if (step == 1 && n >= 8 && ((uintptr_t)s & 15) == 0) {
    uint4 w[sizeof(T) / 2];
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; j++) w[j] = ((const uint4*)s)[j];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = to_f(((const T*)w)[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = j < n ? to_f(s[j * step]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void load8_slope(const void* p, int64_t at, int64_t step, int n, bool relu, float v[8]) {
  if constexpr (sizeof(T) == 4) {
    load8((const float*)p + at, step, n, v);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = kept_slope(v[j], relu);
  } else {
    const uint16_t* s = (const uint16_t*)p + at;
    uint4 w;
    uint16_t* q = (uint16_t*)&w;
    if (step == 1 && n >= 8 && ((uintptr_t)s & 15) == 0) {
      w = *(const uint4*)s;
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) q[j] = j < n ? s[j * step] : 0;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = kept_slope<T>(q[j], relu);
  }
}
// Eight values as the tensor cores' elements, in one plane or three.
template <typename T>
__device__ __forceinline__ void store8(const float v[8], Cell16<T>* d, int64_t plane) {
  if constexpr (sizeof(T) == 4) {
    uint4 w[3];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      __nv_bfloat16 p[3];
      split3(v[j], p);
#pragma unroll
      for (int pl = 0; pl < 3; pl++) ((__nv_bfloat16*)&w[pl])[j] = p[pl];
    }
#pragma unroll
    for (int pl = 0; pl < 3; pl++) *(uint4*)(d + pl * plane) = w[pl];
  } else {
    uint4 w;
#pragma unroll
    for (int j = 0; j < 8; j++) ((Cell16<T>*)&w)[j] = from_f<Cell16<T>>(v[j]);
    *(uint4*)d = w;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ PackJobs jobs) {
  const PackJob& q = jobs.j[blockIdx.y];
  const int64_t inner = q.k_major ? q.k : q.rows, outer = q.k_major ? q.rows : q.k;
  const uint32_t chunks = (uint32_t)((inner + 7) / 8);
  const int64_t total = outer * chunks;
  const int64_t si = q.k_major ? q.src.cs : q.src.rs, so = q.k_major ? q.src.rs : q.src.cs;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t o = i < INT32_MAX ? (uint32_t)i / chunks : i / chunks, c = (i - o * chunks) * 8;
    const int n = (int)min((int64_t)8, inner - c);
    float v[8];
    load8((const T*)q.src.p + o * so + c * si, si, n, v);
    if (q.coef) {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (j < n && q.coef[q.k_major ? o : c + j] == 0.0f) v[j] = 0.0f;
    }
    store8<T>(v, (Cell16<T>*)q.dst + o * q.ld + c, q.plane);
  }
}

// s = src * slope (slope absent: src), laid out
// for the tensor cores (dst null: not wanted) and its columns' sums over a piece of the
// rows, part[piece][N] (null: not wanted): one pass over both.  Memory bounds it.
struct Strip {
  View src;
  View slope;
  int64_t M, N, rows;  // rows of a piece
  void* dst;
  int64_t ld, plane;
  float* part;
  bool padded;  // rows of src may be read up to their stride
  bool relu;    // slope is positive where act' is 1
};

template <typename T>
__device__ __forceinline__ void strip8(const Strip& q, int64_t m, int64_t n, int64_t step_src, int64_t step_slope, int count,
                                       float v[8]) {
  load8((const T*)q.src.p + m * q.src.rs + n * q.src.cs, step_src, count, v);
  if (q.slope.p) {
    float w[8];
    load8_slope<T>(q.slope.p, m * q.slope.rs + n * q.slope.cs, step_slope, count, q.relu, w);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] *= w[j];
  }
}

// Columns contiguous (or any strides): a thread takes 8 columns of every (256 / per)-th row.
template <typename T>
__global__ void __launch_bounds__(256) strip_rows_kernel(const __grid_constant__ Strip q, int per) {
  __shared__ float sh[256 * 8];
  const int tx = threadIdx.x % per, ty = threadIdx.x / per, step = 256 / per;
  const int64_t n = ((int64_t)blockIdx.x * per + tx) * 8, m0 = (int64_t)blockIdx.y * q.rows, m1 = min(q.M, m0 + q.rows);
  const int count = (int)min((int64_t)8, q.N - n);
  float sum[8] = {};
  const T* src = (const T*)q.src.p + n;
  const typename std::conditional<sizeof(T) == 4, float, uint16_t>::type* slope = nullptr;
  if (q.slope.p) slope = (decltype(slope))q.slope.p + n;
  constexpr int kPer = 16 / (int)sizeof(T), kVec = (int)sizeof(T) / 2;  // elements a load, loads of 8 elements
  const bool vec = (count == 8 || (count > 0 && q.padded)) && q.src.cs == 1 && q.src.rs % kPer == 0 && ((uintptr_t)src & 15) == 0 &&
                   (!slope || (q.slope.cs == 1 && q.slope.rs % kPer == 0 && ((uintptr_t)slope & 15) == 0));
  if (vec) {  // several rows' loads in flight before the first is used
    constexpr int kRows = 4;
    for (int64_t m = m0 + ty; m < m1; m += kRows * step) {
      uint4 a[kRows][kVec], b[kRows][kVec];
#pragma unroll
      for (int i = 0; i < kRows; i++) {
        const int64_t row = m + i * step;
        if (row < m1) {
#pragma unroll
          for (int j = 0; j < kVec; j++) {
            a[i][j] = __ldg((const uint4*)(src + row * q.src.rs) + j);
            if (slope) b[i][j] = __ldg((const uint4*)(slope + row * q.slope.rs) + j);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; i++) {
        const int64_t row = m + i * step;
        if (row < m1) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; j++) {
            v[j] = to_f(((const T*)a[i])[j]);
            if (slope) {
              if constexpr (sizeof(T) == 4) v[j] *= kept_slope(((const float*)b[i])[j], q.relu);
              else v[j] *= kept_slope<T>(((const uint16_t*)b[i])[j], q.relu);
            }
          }
          if (q.dst) store8<T>(v, (Cell16<T>*)q.dst + row * q.ld + n, q.plane);
#pragma unroll
          for (int j = 0; j < 8; j++) sum[j] += v[j];
        }
      }
    }
  } else if (count > 0) {
    for (int64_t m = m0 + ty; m < m1; m += step) {
      float v[8];
      strip8<T>(q, m, n, q.src.cs, q.slope.cs, count, v);
      if (q.dst) store8<T>(v, (Cell16<T>*)q.dst + m * q.ld + n, q.plane);
#pragma unroll
      for (int j = 0; j < 8; j++) sum[j] += v[j];
    }
  }
  if (!q.part) return;
#pragma unroll
  for (int j = 0; j < 8; j++) sh[(ty * per + tx) * 8 + j] = sum[j];
  __syncthreads();
  for (int i = threadIdx.x; i < per * 8; i += 256) {
    float a = 0.0f;
    for (int y = 0; y < step; y++) a += sh[y * per * 8 + i];
    const int64_t col = (int64_t)blockIdx.x * per * 8 + i;
    if (col < q.N) q.part[(int64_t)blockIdx.y * q.N + col] = a;
  }
}

// Rows contiguous (an image): a block takes a piece of one column after another.
template <typename T>
__global__ void __launch_bounds__(256) strip_image_kernel(const __grid_constant__ Strip q) {
  __shared__ float sh[8];
  const int64_t m0 = (int64_t)blockIdx.x * q.rows, m1 = min(q.M, m0 + q.rows);
  for (int64_t n = blockIdx.y; n < q.N; n += gridDim.y) {
    float sum = 0.0f;
#pragma unroll 2
    for (int64_t m = m0 + threadIdx.x * 8; m < m1; m += 2048) {
      const int count = (int)min((int64_t)8, m1 - m);
      float v[8];
      strip8<T>(q, m, n, q.src.rs, q.slope.rs, count, v);
      if (q.dst) store8<T>(v, (Cell16<T>*)q.dst + n * q.ld + m, q.plane);
#pragma unroll
      for (int j = 0; j < 8; j++) sum += v[j];
    }
    if (!q.part) continue;
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < 8; i++) sum += sh[i];
      q.part[(int64_t)blockIdx.x * q.N + n] = sum;
    }
  }
}

// act' of no activation, 1, as kept: for a caller that asks for it (the backward does not read it).
template <typename T>
__global__ void __launch_bounds__(256) ones_kernel(View d, int64_t M, int64_t N) {
  const bool by_col = d.cs == 1;
  const int64_t run = by_col ? N : M, total = M * N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t hi = i / run, at = hi * (by_col ? d.rs : d.cs) + (i - hi * run);
    if constexpr (sizeof(T) == 4) ((float*)d.p)[at] = 1.0f;
    else ((uint16_t*)d.p)[at] = (uint16_t)Slope<T>::pack(pair(1.0f));
  }
}

// out(r, c) = alpha * sum of the pieces' elements (r, c), added in a fixed order.  Up to two jobs a launch.
struct SumJob {
  const float* part;
  int pieces;
  int64_t piece;     // elements from one piece to the next
  int64_t prs, pcs;  // strides of an element in its piece
  int64_t rows, cols;
  const float* alpha;
  View out;
};
struct SumJobs {
  SumJob j[2];
};

// SPLIT threads share an element's pieces: 1 for few pieces, 32 (a block is 8 elements, a sector of
// every piece) for many.
template <typename T, int SPLIT>
__global__ void __launch_bounds__(256) sum_kernel(const __grid_constant__ SumJobs jobs) {
  __shared__ float sh[SPLIT][256 / SPLIT + 1];
  const SumJob& q = jobs.j[blockIdx.y];
  const int64_t total = q.rows * q.cols;
  const bool by_col = q.out.cs == 1;
  const uint32_t run = (uint32_t)(by_col ? q.cols : q.rows);
  const float alpha = q.alpha ? *q.alpha : 1.0f;
  const int lane = threadIdx.x % (256 / SPLIT), w = threadIdx.x / (256 / SPLIT);
  for (int64_t base = (int64_t)blockIdx.x * (256 / SPLIT); base < total; base += (int64_t)gridDim.x * (256 / SPLIT)) {
    const int64_t i = base + lane;
    const int64_t hi = i < INT32_MAX ? (uint32_t)i / run : i / run, lo = i - hi * run;
    const int64_t r = by_col ? hi : lo, c = by_col ? lo : hi;
    float sum = 0.0f;
    if (i < total) {
      const float* p = q.part + r * q.prs + c * q.pcs;
#pragma unroll 4
      for (int k = w; k < q.pieces; k += SPLIT) sum += p[k * q.piece];
    }
    if (SPLIT > 1) {
      sh[w][lane] = sum;
      __syncthreads();
      if (w == 0)
        for (int k = 1; k < SPLIT; k++) sum += sh[k][lane];
      __syncthreads();
    }
    if (w == 0 && i < total) ((T*)q.out.p)[r * q.out.rs + c * q.out.cs] = from_f<T>(sum * alpha);
  }
}

// Rows' losses from the parts' maxima and sums; per block the sum of its rows' losses and their count (total not null: the one block's sum or mean itself).
__global__ void __launch_bounds__(256) loss_kernel(const float* pmax, const float* psum, int parts,
                                                   int64_t M, int64_t V, const int64_t* target,
                                                   int64_t ignore, float* rows, float* lse, float* bsum,
                                                   float* bcount, float* total, int mean) {
  __shared__ float sh[2][8];
  float loss = 0.0f, live = 0.0f;
  for (int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x; m < M; m += (int64_t)gridDim.x * 256) {
    float top = -INFINITY, sum = 0.0f;
    for (int i = 0; i < parts; i++) top = fmaxf(top, pmax[(int64_t)i * M + m]);
    for (int i = 0; i < parts; i++) {
      const float p = pmax[(int64_t)i * M + m];
      sum += psum[(int64_t)i * M + m] * (p == top ? 1.0f : exp2f((p - top) * kLog2e));
    }
    const float l = log2f(sum);
    const int64_t t = target[m];
    const bool ignored = t == ignore, bad = !ignored && (t < 0 || t >= V);
    lse[m] = top;
    lse[M + m] = bad ? NAN : l;
    const float row = ignored ? 0.0f : bad ? NAN : fmaf(l, 0.6931471806f, top - lse[2 * M + m]);
    loss += row;
    live += ignored ? 0.0f : 1.0f;
    if (rows) rows[m] = row;
  }
  for (int o = 16; o; o >>= 1) {
    loss += __shfl_xor_sync(0xffffffffu, loss, o);
    live += __shfl_xor_sync(0xffffffffu, live, o);
  }
  if (threadIdx.x % 32 == 0) sh[0][threadIdx.x / 32] = loss, sh[1][threadIdx.x / 32] = live;
  __syncthreads();
  if (threadIdx.x == 0 && (bsum || total)) {
    for (int i = 1; i < 8; i++) loss += sh[0][i], live += sh[1][i];
    if (total) {  // the only block
      total[0] = mean ? loss / live : loss;
    } else {
      bsum[blockIdx.x] = loss;
      bcount[blockIdx.x] = live;
    }
  }
}

// loss[0] = the blocks' sums (mean: over their count), in a fixed order, in double.
__global__ void __launch_bounds__(256) reduce_loss_kernel(const float* bsum, const float* bcount, int64_t blocks,
                                                          int mean, float* loss) {
  __shared__ double sh[2][256];
  double a = 0.0, c = 0.0;
  for (int64_t i = threadIdx.x; i < blocks; i += 256) a += bsum[i], c += bcount[i];
  sh[0][threadIdx.x] = a;
  sh[1][threadIdx.x] = c;
  for (int o = 128; o; o >>= 1) {
    __syncthreads();
    if (threadIdx.x < o) {
      sh[0][threadIdx.x] += sh[0][threadIdx.x + o];
      sh[1][threadIdx.x] += sh[1][threadIdx.x + o];
    }
  }
  if (threadIdx.x == 0) loss[0] = (float)(mean ? sh[0][0] / sh[1][0] : sh[0][0]);
}

// Per-row factors of the logits' gradient.  Their common size goes to the
// products' end instead (alpha): G is kept in 16 bits, and float16 would lose
// probabilities divided by a pixel count.  lift (a power of two) moves float16's G
// up further, so that a probability keeps float16's full precision down to 4e-9.  Rows with gradients of their
// own share one scale, the largest's, because dweight sums over them: beside float16 a row of 2^-20 of the largest
// |dloss| keeps G to 2^-19 of its own scale (its dx is rounded to 2^-12), and one below 2^-26 loses its small probabilities.
// First per block: the largest finite |dloss| and the number of rows not ignored.
__global__ void __launch_bounds__(256) coef_parts_kernel(const int64_t* target, int64_t ignore, int64_t M,
                                                         const float* dloss, float* bmax, uint32_t* bcount) {
  __shared__ float shm[8];
  __shared__ uint32_t shc[8];
  float top = 0.0f;
  uint32_t live = 0;
  for (int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x; m < M; m += (int64_t)gridDim.x * 256) {
    const bool on = target[m] != ignore;
    live += on;
    if (dloss && on && isfinite(dloss[m])) top = fmaxf(top, fabsf(dloss[m]));
  }
  for (int o = 16; o; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    live += __shfl_xor_sync(0xffffffffu, live, o);
  }
  if (threadIdx.x % 32 == 0) shm[threadIdx.x / 32] = top, shc[threadIdx.x / 32] = live;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; i++) top = fmaxf(top, shm[i]), live += shc[i];
    bmax[blockIdx.x] = top;
    bcount[blockIdx.x] = live;
  }
}

// Then the factors themselves; every block adds the (at most 256) parts up again (bmax null: there is one block).
__global__ void __launch_bounds__(256) coef_kernel(const int64_t* target, int64_t ignore, int64_t M, int reduction,
                                                   const float* dloss, const float* bmax, const uint32_t* bcount,
                                                   int parts, float lift, float* coef, float* alpha) {
  __shared__ float shm[8];
  __shared__ uint32_t shc[8];
  float top = 0.0f;
  uint32_t live = 0;
  if (bmax) {
    if (threadIdx.x < parts) top = bmax[threadIdx.x], live = bcount[threadIdx.x];
  } else {  // one block: it finds them itself
    for (int64_t m = threadIdx.x; m < M; m += 256) {
      const bool on = target[m] != ignore;
      live += on;
      if (reduction == VI_REDUCE_NONE && on && isfinite(dloss[m])) top = fmaxf(top, fabsf(dloss[m]));
    }
  }
  for (int o = 16; o; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    live += __shfl_xor_sync(0xffffffffu, live, o);
  }
  if (threadIdx.x % 32 == 0) shm[threadIdx.x / 32] = top, shc[threadIdx.x / 32] = live;
  __syncthreads();
  top = 0.0f;
  live = 0;
  for (int i = 0; i < 8; i++) top = fmaxf(top, shm[i]), live += shc[i];
  int ex = 0;
  frexpf(top, &ex);
  ex = min(max(ex, -100), 100);  // a power of two at or above every finite |g|: the division is exact
  // a common size that is not finite stays in the rows that it belongs to: at the products' end it would
  // meet the zeros of the ignored ones
  const float common = reduction == VI_REDUCE_NONE  ? ldexpf(1.0f, ex)
                       : reduction == VI_REDUCE_SUM ? *dloss
                       : live                       ? *dloss / (float)live
                                                    : 0.0f;
  const bool finite = isfinite(common);
  if (blockIdx.x == 0 && threadIdx.x == 0) *alpha = (finite ? common : 1.0f) / lift;
  for (int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x; m < M; m += (int64_t)gridDim.x * 256) {
    const float g = reduction == VI_REDUCE_NONE ? ldexpf(dloss[m], -ex) : finite ? 1.0f : common;
    coef[m] = target[m] != ignore ? g * lift : 0.0f;
  }
}

// ---------------------------------------------------------------------------
// Host side.  One function per operator carves the scratch and launches; with
// `dry` it only carves, which is how the _scratch_bytes queries count.
// ---------------------------------------------------------------------------
int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64) {
    if ((n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n > 0 ? n : 148;
}

// Bytes of the logits' gradient that exist at a time, if 256 columns fit.
constexpr int64_t kPieceBytes = 640ll << 20;

struct Run {
  char* base;
  cudaStream_t s;
  bool dry;
  int sms = sm_count();
  size_t cur = 0, peak = 0;
  int launches = 0;
  void* take(size_t bytes) {
    cur = align_up(cur);
    char* p = base + cur;
    cur += bytes;
    peak = std::max(peak, cur);
    return p;
  }
  // what was taken since `mark` may be taken again (by work that the stream runs later)
  void release(size_t mark) { cur = mark; }
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t elem(int dtype) { return dtype == VI_F32 ? 4 : 2; }
View view(const vi_matrix* m) { return m ? View{m->data, m->row_stride, m->col_stride} : View{nullptr, 0, 0}; }
// A [rows, cols] scratch matrix in the memory order of `like`.
View scratch_like(void* p, const View& like, int64_t rows, int64_t cols) {
  return like.rs == 1 && like.cs != 1 ? View{p, 1, rows} : View{p, cols, 1};
}
View transposed(View v) { return View{v.p, v.cs, v.rs}; }
Operand transposed(Operand o) {
  std::swap(o.rows, o.k);
  o.k_major = !o.k_major;
  return o;
}

#define VI_DISPATCH(dtype, ...)                                    \
  do {                                                             \
    if ((dtype) == VI_F32) {                                       \
      using T = float;                                             \
      __VA_ARGS__;                                                 \
    } else if ((dtype) == VI_F16) {                                \
      using T = __half;                                            \
      __VA_ARGS__;                                                 \
    } else {                                                       \
      using T = __nv_bfloat16;                                     \
      __VA_ARGS__;                                                 \
    }                                                              \
  } while (0)

// Whether the tensor cores' copies can read the matrix where it lies: 16-bit elements,
// one axis contiguous, the other's stride and the address multiples of 16 bytes.
bool direct(int dtype, const View& v, int64_t rows, int64_t k) {
  if (dtype == VI_F32 || (uintptr_t)v.p % 16) return false;
  if (v.cs == 1) return v.rs % 8 == 0 && v.rs >= k && v.rs < (1ll << 38);
  return v.rs == 1 && v.cs % 8 == 0 && v.cs >= rows && v.cs < (1ll << 38);
}

// Operands of one call; those that have to be laid out first are collected and done by one launch.
struct Packer {
  Run& r;
  int dtype;
  PackJobs jobs{};
  int n = 0;
  int64_t chunks = 0;
  Operand add(const View& v, int64_t rows, int64_t k, const float* coef = nullptr) {
    const bool k_major = v.cs == 1 || v.rs != 1;
    if (!coef && direct(dtype, v, rows, k)) return Operand{v.p, rows, k, k_major ? v.rs : v.cs, 0, k_major};
    const int64_t inner = k_major ? k : rows, outer = k_major ? rows : k;
    const int64_t ld = ceil_div(inner, 8) * 8, plane = ld * outer;
    void* dst = r.take((size_t)plane * 2 * (dtype == VI_F32 ? 3 : 1));
    jobs.j[n++] = PackJob{v, coef, rows, k, dst, ld, plane, k_major};
    chunks = std::max(chunks, outer * (ld / 8));
    if (n == 2) run();
    return Operand{dst, rows, k, ld, plane, k_major};
  }
  void run() {
    if (n && !r.dry) {
      const dim3 grid((unsigned)std::min<int64_t>(ceil_div(chunks, 256), 148 * 16), n);
      VI_DISPATCH(dtype, (pack_kernel<T><<<grid, 256, 0, r.s>>>(jobs)));
      r.launches++;
    }
    n = 0;
    chunks = 0;
  }
};

// Tiles of a width, and how many of them run at a time.
int64_t tiles_of(int epi, int64_t M, int64_t N, int bn) { return ceil_div(M, pair_tile(epi, bn) ? 256 : 128) * ceil_div(N, bn); }
int64_t tile_slots(int epi, int bn, int sms) { return std::max(1, pair_tile(epi, bn) ? sms / 2 : sms); }

// Tile width: the one whose waves of tiles take the least tensor-core time; narrow tiles
// read their operands more often.
int tile_width(int dtype, int epi, int64_t M, int64_t N, int64_t kblocks, int sms) {
  if (long_chain_kernel(dtype, epi, kblocks)) return 128;
  int best = 64;
  double cost = 1e300;
  for (int bn : {256, 128, 64}) {
    if (bn == 256 && (dtype == VI_F32 || (pair_tile(epi, bn) && M <= 128))) continue;
    const double c = (double)ceil_div(tiles_of(epi, M, N, bn), tile_slots(epi, bn, sms)) * (bn == 256 ? 240 : bn == 128 ? 150 : 90);
    if (c < cost) cost = c, best = bn;
  }
  return best;
}

// A result in image order (rows contiguous) of enough channels to fill most of a tile's 128
// rows is asked for transposed, out^T = B A^T: a thread of the epilogue then has a
// channel's pixels next to each other, and the bias in one register.  With fewer
// channels (64 of 128 rows used: 399 us against 263 at 2M x 64 x 64) it is not.
int gemm(Run& r, int dtype, int epi, const Operand& A, const Operand& B, const Epilogue& e) {
  if (r.dry) return VI_OK;
  if ((epi == kEpiAct || epi == kEpiStore) && e.out.rs == 1 && e.out.cs != 1 && 4 * B.rows >= 3 * 128 * ceil_div(B.rows, 128)) {
    Epilogue f = e;
    f.out = transposed(e.out);
    f.res = transposed(e.res);
    f.bias_rows = e.bias != nullptr;
    Plan p{};
    p.splits = 1;
    p.kps = (int)ceil_div(A.k, 64);
    p.bn = tile_width(dtype, epi, B.rows, A.rows, p.kps, r.sms);
    return launch_gemm(dtype, epi, B, A, p, f, r.sms, r.s);
  }
  Plan p{};
  p.splits = 1;
  p.kps = (int)ceil_div(A.k, 64);
  p.bn = tile_width(dtype, epi, A.rows, B.rows, p.kps, r.sms);
  return launch_gemm(dtype, epi, A, B, p, e, r.sms, r.s);
}

// Pieces of a long sum over k: enough that the tiles fill the SMs, or fill their last wave where
// that gains more than the pieces' float32 results cost to write and read (16384 x 512 over
// 18944: 1.73 waves of tiles in one piece, 3.46 in two; 240 us -> 217).  Precision asks for no pieces: the product makes
// a long one of chains (float32 dx of 16384 x 4096 <- 1024 in pieces of 768 terms: 1077 us, in chains 636).
Plan split_plan(int dtype, const Operand& A, const Operand& B, int sms) {
  Plan p{};
  p.bn = B.rows <= 64 ? 64 : B.rows <= 128 || A.rows <= 128 || dtype == VI_F32 ? 128 : 256;
  const int64_t tiles = tiles_of(kEpiPartial, A.rows, B.rows, p.bn), slots = tile_slots(kEpiPartial, p.bn, sms), kb = ceil_div(A.k, 64);
  int64_t want = 1;
  if (tiles < slots) {
    want = std::max<int64_t>(1, std::min<int64_t>(slots / tiles, kb / 4));  // at least four blocks of k each
  } else {
    const double product = 2.0 * A.rows * B.rows * A.k * (dtype == VI_F32 ? 6 : 1) / 1.3e15, copy = 8.0 * A.rows * B.rows / 5e12;
    double best = 1e300;
    for (int64_t s = 1; s <= 4 && kb / s >= 32; s++) {
      const double waves = (double)(ceil_div(tiles * s, slots) * slots) / (double)(tiles * s);
      const double t = product * waves + (s > 1 ? copy * s : 0.0);
      if (t < best) best = t, want = s;
    }
  }
  p.kps = (int)ceil_div(kb, want);
  p.splits = (int)ceil_div(kb, p.kps);
  return p;
}

// Sums of pieces that wait for their launch; their part buffers stay taken until then.  A job is added just
// before the kernel that writes its pieces is launched: adding the next one may launch the sums so far.
struct Summer {
  Run& r;
  int dtype;
  SumJobs jobs{};
  int n = 0;
  bool shared = false;
  int64_t total = 0;
  void add(const SumJob& j) {
    // many pieces of few elements: threads share an element
    const bool share = j.pieces > 8 && j.rows * j.cols < 65536;
    if (n == 2 || (n && shared != share)) run();
    shared = share;
    jobs.j[n++] = j;
    total = std::max(total, j.rows * j.cols);
  }
  void run() {
    if (n && !r.dry) {
      if (shared) {
        const dim3 grid((unsigned)std::min<int64_t>(ceil_div(total, 8), 148 * 16), n);
        VI_DISPATCH(dtype, (sum_kernel<T, 32><<<grid, 256, 0, r.s>>>(jobs)));
      } else {
        const dim3 grid((unsigned)std::min<int64_t>(ceil_div(total, 256), 148 * 16), n);
        VI_DISPATCH(dtype, (sum_kernel<T, 1><<<grid, 256, 0, r.s>>>(jobs)));
      }
      r.launches++;
    }
    n = 0;
    total = 0;
  }
};

// out = alpha * A B^T; a long sum with few tiles in pieces, in float32, added in order (by `sums`).
int gemm_out(Run& r, Summer& sums, const Operand& A, const Operand& B, const float* alpha, const View& out) {
  const Plan p = split_plan(sums.dtype, A, B, r.sms);
  Epilogue e{};
  if (p.splits == 1) {
    e.out = out;
    e.alpha = alpha;
    return gemm(r, sums.dtype, kEpiStore, A, B, e);
  }
  e.part = (float*)r.take((size_t)p.splits * A.rows * B.rows * 4);
  sums.add(SumJob{e.part, p.splits, A.rows * B.rows, B.rows, 1, A.rows, B.rows, alpha, out});
  return r.dry ? VI_OK : launch_gemm(sums.dtype, kEpiPartial, A, B, p, e, r.sms, r.s);
}

// One pass over src * slope: laid out in dst (null: no), its columns' sums in `sums` (db null: no).
void strip(Run& r, Summer& sums, int dtype, Strip q, const float* alpha, void* db) {
  const bool image = q.src.rs == 1 && q.src.cs != 1;
  int per = 256;  // threads along a row: long runs of it, so that DRAM pages are read whole
  while (per > 1 && (per / 2) * 8 >= q.N) per /= 2;
  const int64_t blocks = image ? std::min<int64_t>(q.N, 1024) : ceil_div(q.N, per * 8);
  // enough pieces of the rows to fill the SMs, each long enough to be worth its sum
  const int64_t least = image ? 8192 : 256 / per * 8;
  const int64_t pieces = std::max<int64_t>(1, std::min<int64_t>(ceil_div(r.sms * 8, blocks), q.M / least));
  q.rows = ceil_div(ceil_div(q.M, pieces), 8) * 8;
  const int64_t count = ceil_div(q.M, q.rows);
  q.part = nullptr;
  if (db) {
    q.part = (float*)r.take((size_t)count * q.N * 4);
    sums.add(SumJob{q.part, (int)count, q.N, 0, 1, 1, q.N, alpha, View{db, 0, 1}});
  }
  if (r.dry) return;
  if (image) {
    const dim3 grid((unsigned)count, (unsigned)blocks);
    VI_DISPATCH(dtype, (strip_image_kernel<T><<<grid, 256, 0, r.s>>>(q)));
  } else {
    const dim3 grid((unsigned)blocks, (unsigned)count);
    VI_DISPATCH(dtype, (strip_rows_kernel<T><<<grid, 256, 0, r.s>>>(q, per)));
  }
  r.launches++;
}

int small(Run& r, int dtype, const SmallJob& a, const SmallJob* b) {
  if (r.dry) return VI_OK;
  const cudaError_t rc = launch_small(dtype, a, b, r.s);
  r.launches++;
  return rc == cudaSuccess ? VI_OK : set_error(VI_ERR_CUDA, cudaGetErrorString(rc));
}

// Gradients of the weights over no rows at all.
void zero_gradients(Run& r, int dtype, int64_t N, int64_t K, const vi_matrix* dw, void* db) {
  Summer sums{r, dtype};
  if (dw && dw->data) sums.add(SumJob{nullptr, 0, 0, 0, 0, N, K, nullptr, view(dw)});
  if (db) sums.add(SumJob{nullptr, 0, 0, 0, 0, 1, N, nullptr, View{db, 0, 1}});
  sums.run();
}

// ---- argument checks ----
int bad(const char* msg) { return set_error(VI_ERR_INVALID_ARGUMENT, msg); }

constexpr int64_t kMaxSize = 1ll << 30;  // tile coordinates are 32-bit

bool dense(const vi_matrix* m) {  // one stride 1, the other at least the extent
  if (m->rows <= 0 || m->cols <= 0) return true;
  return (m->col_stride == 1 && (m->row_stride >= m->cols || m->rows == 1)) ||
         (m->row_stride == 1 && (m->col_stride >= m->rows || m->cols == 1));
}
bool given(const vi_matrix* m) { return m && (m->data || m->rows == 0); }

int check_operands(int dtype, const vi_matrix* x, const vi_matrix* w) {
  if (dtype < VI_F32 || dtype > VI_BF16) return bad("heads: unknown element type");
  if (!x || !w) return bad("heads: x and weight are required");
  if (x->rows < 0 || x->cols < 1 || w->rows < 1) return bad("heads: x needs at least one column and weight one row");
  if (w->cols != x->cols) return bad("heads: weight and x differ in their number of columns");
  if (x->rows > kMaxSize || w->rows > kMaxSize || x->cols > kMaxSize) return bad("heads: sizes are limited to 2^30");
  if ((!x->data && x->rows) || !w->data) return bad("heads: x and weight need data");
  if (x->row_stride < 0 || x->col_stride < 0 || w->row_stride < 0 || w->col_stride < 0)
    return bad("heads: strides must not be negative");
  if ((uintptr_t)x->data % elem(dtype) || (uintptr_t)w->data % elem(dtype)) return bad("heads: data must lie on whole elements");
  return VI_OK;
}
int check_vector(int dtype, const void* p) {
  return (uintptr_t)p % elem(dtype) ? bad("heads: data must lie on whole elements") : VI_OK;
}
int check_shape(int dtype, const vi_matrix* m, int64_t rows, int64_t cols, bool need_dense, const char* msg) {
  if (!m || !m->data) return VI_OK;
  if (m->rows != rows || m->cols != cols || m->row_stride < 0 || m->col_stride < 0) return bad(msg);
  if (int rc = check_vector(dtype, m->data)) return rc;
  if (need_dense && !dense(m)) return bad(msg);
  return VI_OK;
}

int finish(Run& r, const char* where) {
  note_launches(r.launches);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    char msg[256];
    snprintf(msg, sizeof msg, "%s: %s", where, cudaGetErrorString(e));
    return set_error(VI_ERR_CUDA, msg);
  }
  return VI_OK;
}

// A dry run's base is not null, so that what it carves passes for given, as in the real run.
char* dry_base() { return (char*)256; }

template <class F>
uint64_t count_bytes(F&& f) {
  Run r{dry_base(), nullptr, true};
  return f(r) == VI_OK ? align_up(r.peak) + 256 : 0;
}
template <class F>
int execute(F&& f, void* scratch, uint64_t bytes, void* stream, const char* where) {
  Run d{scratch ? (char*)scratch : dry_base(), nullptr, true};  // exactly what the real run will take
  int rc = f(d);
  if (rc) return rc;
  if (d.peak > bytes || (d.peak && (!scratch || (uintptr_t)scratch % 256)))
    return bad("heads: scratch is too small or not 256-byte aligned");
  Run r{(char*)scratch, (cudaStream_t)stream, false};
  rc = f(r);
  return rc ? rc : finish(r, where);
}

// ---- linear_act ----
int act_forward(Run& r, int dtype, int act, const vi_matrix* x, const vi_matrix* w, const void* bias,
                const vi_matrix* res, const vi_matrix* y, const vi_matrix* dact) {
  if (int rc = check_operands(dtype, x, w)) return rc;
  if (act < VI_ACT_NONE || act > VI_ACT_SIGMOID) return bad("linear_act: unknown activation");
  if (int rc = check_vector(dtype, bias)) return rc;
  const int64_t M = x->rows, K = x->cols, N = w->rows;
  if (!given(y) || y->rows != M) return bad("linear_act: y is required, [M, N]");
  if (int rc = check_shape(dtype, res, M, N, false, "linear_act: residual must be [M, N]")) return rc;
  if (int rc = check_shape(dtype, y, M, N, true, "linear_act: y must be a dense [M, N]")) return rc;
  if (int rc = check_shape(dtype, dact, M, N, true, "linear_act: dact must be a dense [M, N]")) return rc;
  if (dact && dact->data && (dact->row_stride != y->row_stride || dact->col_stride != y->col_stride))
    return bad("linear_act: dact must have y's strides");
  if (M == 0) return VI_OK;
  Epilogue e{};
  e.act = act;
  e.bias = bias;
  e.res = view(res);
  e.out = view(y);
  e.dact = dact && act != VI_ACT_NONE ? dact->data : nullptr;
  if (act == VI_ACT_NONE && dact && dact->data && !r.dry) {
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(M * N, 256), 148 * 16);
    VI_DISPATCH(dtype, (ones_kernel<T><<<blocks, 256, 0, r.s>>>(view(dact), M, N)));
    r.launches++;
  }
  if (!e.dact && narrow_forward(N, K, view(x), e.out, e.res)) {
    if (r.dry) return VI_OK;
    const cudaError_t rc = launch_narrow(dtype, NarrowArgs{M, (int)N, (int)K, act, view(x), view(w), bias, e.out, e.res},
                                         false, 0, r.sms, r.s);
    r.launches++;
    return rc == cudaSuccess ? VI_OK : set_error(VI_ERR_CUDA, cudaGetErrorString(rc));
  }
  // a small product whose operands would have to be laid out first (with longer sums that launch is worth it:
  // 37 x 203 -> 131: 16 us, 20 here)
  if (K <= 128 && small_product(M, N, K, K) && !(direct(dtype, view(x), M, K) && direct(dtype, view(w), N, K))) {
    SmallJob q{view(x), {}, view(w), nullptr, (int)M, (int)N, (int)K, e.out};
    q.bias = bias;
    q.act = act;
    q.res = e.res;
    q.dact = e.dact;
    return small(r, dtype, q, nullptr);
  }
  Packer pk{r, dtype};
  const Operand A = pk.add(view(x), M, K), B = pk.add(view(w), N, K);
  pk.run();
  return gemm(r, dtype, kEpiAct, A, B, e);
}

int act_backward(Run& r, int dtype, int act, const vi_matrix* dy, const vi_matrix* dact, const vi_matrix* x,
                 const vi_matrix* w, const void* bias, const vi_matrix* dx, const vi_matrix* dw, void* db) {
  if (int rc = check_operands(dtype, x, w)) return rc;
  if (act < VI_ACT_NONE || act > VI_ACT_SIGMOID) return bad("linear_act backward: unknown activation");
  if (int rc = check_vector(dtype, bias)) return rc;
  if (int rc = check_vector(dtype, db)) return rc;
  const int64_t M = x->rows, K = x->cols, N = w->rows;
  if (!given(dy) || dy->rows != M) return bad("linear_act backward: dy is required, [M, N]");
  if (int rc = check_shape(dtype, dy, M, N, false, "linear_act backward: dy must be [M, N]")) return rc;
  if (int rc = check_shape(dtype, dact, M, N, true, "linear_act backward: dact must be a dense [M, N]")) return rc;
  if (int rc = check_shape(dtype, dx, M, K, true, "linear_act backward: dx must be a dense [M, K]")) return rc;
  if (int rc = check_shape(dtype, dw, N, K, true, "linear_act backward: dweight must be a dense [N, K]")) return rc;
  const size_t es = elem(dtype);
  if (M == 0) {
    zero_gradients(r, dtype, N, K, dw, db);
    return VI_OK;
  }
  View slope = act == VI_ACT_NONE ? View{nullptr, 0, 0} : view(dact);
  const bool need_dx = dx && dx->data, need_dw = dw && dw->data;
  Summer sums{r, dtype};
  if (!slope.p && narrow_backward(N, K, view(x), view(dy), view(dx))) {
    const int blocks = narrow_blocks(M, r.sms), per = narrow_sums(K);
    NarrowArgs a{M, (int)N, (int)K, act, view(x), view(w), bias, view(dy), View{nullptr, 0, 0}, view(dx)};
    if (need_dw || db) a.part = (float*)r.take((size_t)blocks * N * per * 4);
    if (!r.dry) {
      const cudaError_t rc = launch_narrow(dtype, a, true, blocks, r.sms, r.s);
      r.launches++;
      if (rc != cudaSuccess) return set_error(VI_ERR_CUDA, cudaGetErrorString(rc));
    }
    if (need_dw) sums.add(SumJob{a.part, blocks, N * per, per, 1, N, K, nullptr, view(dw)});
    if (db) sums.add(SumJob{a.part + per - 1, blocks, N * per, 0, per, 1, N, nullptr, View{db, 0, 1}});
    sums.run();
    return VI_OK;
  }
  if ((slope.p || act == VI_ACT_NONE) && small_product(M, N, K, std::max(M, N))) {
    SmallJob jx{view(dy), slope, transposed(view(w)), nullptr, (int)M, (int)K, (int)N, view(dx)};
    SmallJob jw{transposed(view(dy)), transposed(slope), transposed(view(x)), nullptr, (int)N, need_dw ? (int)K : 1, (int)M, view(dw)};
    jw.sums = db;
    jx.relu = jw.relu = act == VI_ACT_RELU;
    const bool second = need_dw || db;
    return need_dx ? small(r, dtype, jx, second ? &jw : nullptr) : second ? small(r, dtype, jw, nullptr) : VI_OK;
  }
  Packer pk{r, dtype};
  Operand S{}, W{}, X{};
  const bool again = !slope.p && act != VI_ACT_NONE;  // act' was not kept
  if (need_dx || again) W = pk.add(view(w), N, K);
  if (need_dw || again) X = pk.add(view(x), M, K);
  pk.run();
  if (again) {
    Epilogue e{};
    e.act = act;
    e.bias = bias;
    e.out = scratch_like(r.take((size_t)M * N * es), view(dy), M, N);
    slope = scratch_like(r.take((size_t)M * N * es), view(dy), M, N);
    e.dact = slope.p;
    if (int rc = gemm(r, dtype, kEpiAct, X, W, e)) return rc;
  }
  // s = dy * act', where dy itself does not serve; the bias's gradient in the same pass
  const View d = view(dy);
  const bool in_place = !slope.p && direct(dtype, d, M, N);
  Strip q{d, slope, M, N};
  q.relu = act == VI_ACT_RELU;
  if (need_dx || need_dw) {
    const bool k_major = d.cs == 1 || d.rs != 1;
    if (in_place) {
      S = Operand{d.p, M, N, k_major ? d.rs : d.cs, 0, k_major};
    } else {
      q.ld = ceil_div(k_major ? N : M, 8) * 8;
      q.plane = q.ld * (k_major ? M : N);
      q.dst = r.take((size_t)q.plane * 2 * (dtype == VI_F32 ? 3 : 1));
      S = Operand{q.dst, M, N, q.ld, q.plane, k_major};
    }
  }
  if (q.dst || db) strip(r, sums, dtype, q, nullptr, db);
  if (need_dx)
    if (int rc = gemm_out(r, sums, S, transposed(W), nullptr, view(dx))) return rc;
  if (need_dw)
    if (int rc = gemm_out(r, sums, transposed(S), transposed(X), nullptr, view(dw))) return rc;
  sums.run();
  return VI_OK;
}

// ---- linear_cross_entropy ----
int ce_forward(Run& r, int dtype, const vi_matrix* x, const vi_matrix* w, const void* bias, const int64_t* target,
               int64_t ignore, int reduction, float* loss, float* lse) {
  if (int rc = check_operands(dtype, x, w)) return rc;
  if (reduction < VI_REDUCE_NONE || reduction > VI_REDUCE_SUM) return bad("linear_ce: unknown reduction");
  if (int rc = check_vector(dtype, bias)) return rc;
  const int64_t M = x->rows, K = x->cols, V = w->rows;
  if (!r.dry && M && (!target || !loss || !lse)) return bad("linear_ce: target, loss and lse are required");
  const int64_t blocks = M <= 1024 ? std::min<int64_t>(M, 1) : ceil_div(M, 256);  // few rows: one block ends the sum too
  Plan p{};
  p.splits = 1;
  p.kps = (int)ceil_div(K, 64);
  // a small vocabulary in narrow tiles, two blocks per SM (640000 x 64 x 150: 88 us in one 256-wide tile, 81)
  p.bn = V <= 64 && !long_chain_kernel(dtype, kEpiLse, p.kps) ? 64 : V <= 256 ? 128 : tile_width(dtype, kEpiLse, M, V, p.kps, r.sms);
  // column tiles in runs, so that a block keeps a row's maximum and sum in registers over several of them
  const int64_t nt = ceil_div(V, p.bn), mt = std::max<int64_t>(1, ceil_div(M, 128));
  p.span = (int)ceil_div(nt, std::min(nt, ceil_div(4 * r.sms, mt)));
  p.spans = (int)ceil_div(nt, p.span);
  const int parts = lse_parts(p.bn) * p.spans;
  float* pmax = (float*)r.take((size_t)parts * M * 4);
  float* psum = (float*)r.take((size_t)parts * M * 4);
  float* bsum = (float*)r.take((size_t)blocks * 4);
  float* bcount = (float*)r.take((size_t)blocks * 4);
  Operand A{}, B{};
  if (M) {
    Packer pk{r, dtype};
    A = pk.add(view(x), M, K);
    B = pk.add(view(w), V, K);
    pk.run();
  }
  if (r.dry) return VI_OK;
  if (M) {
    Epilogue e{};
    e.bias = bias;
    e.pmax = pmax;
    e.psum = psum;
    e.ztarget = lse + 2 * M;
    e.target = target;
    if (int rc = launch_gemm(dtype, kEpiLse, A, B, p, e, r.sms, r.s)) return rc;
    const bool none = reduction == VI_REDUCE_NONE;
    loss_kernel<<<(unsigned)blocks, 256, 0, r.s>>>(pmax, psum, parts, M, V, target, ignore,
                                                   none ? loss : nullptr, lse, none || blocks == 1 ? nullptr : bsum, bcount,
                                                   !none && blocks == 1 ? loss : nullptr, reduction == VI_REDUCE_MEAN);
    r.launches++;
  }
  if (reduction != VI_REDUCE_NONE && blocks != 1) {
    if (!loss) return bad("linear_ce: loss is required");
    reduce_loss_kernel<<<1, 256, 0, r.s>>>(bsum, bcount, blocks, reduction == VI_REDUCE_MEAN, loss);
    r.launches++;
  }
  return VI_OK;
}

int ce_backward(Run& r, int dtype, const vi_matrix* x, const vi_matrix* w, const void* bias, const int64_t* target,
                int64_t ignore, int reduction, const float* lse, const float* dloss, const vi_matrix* dx,
                const vi_matrix* dw, void* db) {
  if (int rc = check_operands(dtype, x, w)) return rc;
  if (reduction < VI_REDUCE_NONE || reduction > VI_REDUCE_SUM) return bad("linear_ce backward: unknown reduction");
  if (int rc = check_vector(dtype, bias)) return rc;
  if (int rc = check_vector(dtype, db)) return rc;
  const int64_t M = x->rows, K = x->cols, V = w->rows;
  if (int rc = check_shape(dtype, dx, M, K, true, "linear_ce backward: dx must be a dense [M, K]")) return rc;
  if (int rc = check_shape(dtype, dw, V, K, true, "linear_ce backward: dweight must be a dense [V, K]")) return rc;
  if (!r.dry && M && (!target || !lse || !dloss)) return bad("linear_ce backward: target, lse and dloss are required");
  const size_t es = elem(dtype);
  if (M == 0) {
    zero_gradients(r, dtype, V, K, dw, db);
    return VI_OK;
  }
  const bool need_dx = dx && dx->data, need_dw = dw && dw->data;
  const int planes = dtype == VI_F32 ? 3 : 1;
  float* coef = (float*)r.take((size_t)M * 4);
  float* alpha = (float*)r.take(4);
  const int parts = M <= 4096 ? 1 : (int)std::min<int64_t>(ceil_div(M, 1024), 256);
  float* bmax = (float*)r.take((size_t)parts * 4);
  uint32_t* bcount = (uint32_t*)r.take((size_t)parts * 4);
  if (!r.dry) {
    if (parts > 1) {
      coef_parts_kernel<<<parts, 256, 0, r.s>>>(target, ignore, M, reduction == VI_REDUCE_NONE ? dloss : nullptr, bmax, bcount);
      r.launches++;
    }
    coef_kernel<<<parts, 256, 0, r.s>>>(target, ignore, M, reduction, dloss, parts > 1 ? bmax : nullptr, bcount, parts,
                                        dtype == VI_F16 ? 16384.0f : 1.0f, coef, alpha);
    r.launches++;
  }
  if (small_product(M, V, K, std::max({M, V, K}))) {
    const View G{r.take((size_t)M * V * es), V, 1};
    SmallJob g{view(x), {}, view(w), nullptr, (int)M, (int)V, (int)K, G};
    g.bias = bias;
    g.coef = coef;
    g.lse = lse;
    g.target = target;
    if (int rc = small(r, dtype, g, nullptr)) return rc;
    SmallJob jx{G, {}, transposed(view(w)), nullptr, (int)M, (int)K, (int)V, view(dx), alpha};
    SmallJob jw{transposed(G), {}, transposed(view(x)), coef, (int)V, need_dw ? (int)K : 1, (int)M, view(dw), alpha, db};
    const bool second = need_dw || db;
    return need_dx ? small(r, dtype, jx, second ? &jw : nullptr) : second ? small(r, dtype, jw, nullptr) : VI_OK;
  }
  // x without the rows of ignored targets: their zero gradient times a NaN or an
  // infinity would else reach the weights' gradient
  Packer pk{r, dtype};
  const Operand X = pk.add(view(x), M, K, need_dw ? coef : nullptr), W = pk.add(view(w), V, K);
  pk.run();

  // G in pieces of the vocabulary
  int64_t piece = std::max<int64_t>(256, kPieceBytes / (M * 2 * planes) / 256 * 256);
  if (piece < V && dtype != VI_F32 && K > 128) {  // whole waves of dweight's 256 x 256 tiles
    const int64_t nt = ceil_div(K, 256), slots = tile_slots(kEpiStore, 256, r.sms), waves = piece / 256 * nt / slots;
    // more features than the slots take side by side: a wave is less than one piece of 256 columns
    if (waves) piece = std::max<int64_t>(256, waves * slots / nt * 256);
  }
  piece = std::min(piece, V);
  const int64_t ld = ceil_div(piece, 8) * 8;
  void* grad = r.take((size_t)planes * M * ld * 2);
  const bool several = piece < V;
  float* acc = nullptr;  // dx over the pieces so far
  Plan px{};
  if (need_dx && several) {
    px = split_plan(dtype, Operand{nullptr, M, piece}, Operand{nullptr, K, piece}, r.sms);
    acc = (float*)r.take((size_t)px.splits * M * K * 4);
  }
  const size_t mark = r.cur;
  for (int64_t c = 0; c < V; c += piece) {
    const int64_t n = std::min(piece, V - c);
    r.release(mark);
    Summer sums{r, dtype};
    Operand Wc = W;
    Wc.rows = n;
    Wc.p = (const char*)W.p + c * (W.k_major ? W.ld : 1) * 2;
    Epilogue e{};
    e.bias = bias ? (const char*)bias + c * elem(dtype) : nullptr;
    e.target = target;
    e.lse = lse;
    e.coef = coef;
    e.col0 = c;
    e.grad = grad;
    e.grad_ld = ld;
    e.grad_plane = M * ld;
    if (db && dtype != VI_F32) {  // the columns' sums on the way
      const int64_t blocks = ceil_div(M, 32);
      e.column_part = (float*)r.take((size_t)blocks * n * 4);
      sums.add(SumJob{e.column_part, (int)blocks, n, 0, 1, 1, n, alpha, View{(char*)db + c * elem(dtype), 0, 1}});
    }
    if (int rc = gemm(r, dtype, kEpiGrad, X, Wc, e)) return rc;
    const Operand G{grad, M, n, ld, M * ld, true};
    if (need_dx) {
      if (several) {
        Epilogue d{};
        d.part = acc;
        d.add = c > 0;
        Plan p = px;  // the last piece may be shorter: fewer blocks of k, some of px's splits empty
        p.kps = (int)ceil_div(ceil_div(n, 64), px.splits);
        p.splits = (int)ceil_div(ceil_div(n, 64), p.kps);
        if (!r.dry)
          if (int rc = launch_gemm(dtype, kEpiPartial, G, transposed(Wc), p, d, r.sms, r.s)) return rc;
      } else if (int rc = gemm_out(r, sums, G, transposed(Wc), alpha, view(dx))) {
        return rc;
      }
    }
    if (need_dw) {
      View out = view(dw);
      out.p = (char*)out.p + c * out.rs * elem(dtype);
      if (int rc = gemm_out(r, sums, transposed(G), transposed(X), alpha, out)) return rc;
    }
    if (db && dtype == VI_F32) {
      Strip q{View{grad, ld, 1}, View{nullptr, 0, 0}, M * planes, n};  // the planes' rows one after another
      q.padded = true;
      strip(r, sums, VI_BF16, q, alpha, (char*)db + c * elem(dtype));
    }
    sums.run();
    if (r.dry && c + piece < V) {  // the last piece alone may be smaller: one more round counts it
      c = (V - 1) / piece * piece - piece;
    }
  }
  if (need_dx && several) {
    Summer sums{r, dtype};
    sums.add(SumJob{acc, px.splits, M * K, K, 1, M, K, alpha, view(dx)});
    sums.run();
  }
  return VI_OK;
}

// ---- layer_norm ----
int check_norm(int dtype, const vi_matrix* x, const void* w, const void* b, double eps) {
  if (dtype < VI_F32 || dtype > VI_BF16) return bad("layer_norm: unknown element type");
  if (!x || x->rows < 0 || x->cols < 1) return bad("layer_norm: x needs at least one column");
  if (x->rows > kMaxSize || x->cols > kMaxSize) return bad("layer_norm: sizes are limited to 2^30");
  if (!x->data && x->rows) return bad("layer_norm: x needs data");
  if (x->row_stride < 0 || x->col_stride < 0) return bad("layer_norm: strides must not be negative");
  if (!(eps >= 0.0) || eps > 3e38) return bad("layer_norm: eps must be a number of at least 0");
  if (int rc = check_vector(dtype, x->data)) return rc;
  if (int rc = check_vector(dtype, w)) return rc;
  return check_vector(dtype, b);
}

int norm_forward(Run& r, int dtype, const vi_matrix* x, const void* w, const void* b, float eps, const vi_matrix* y, float* stats) {
  if (int rc = check_norm(dtype, x, w, b, eps)) return rc;
  if (!given(y) || y->rows != x->rows) return bad("layer_norm: y is required, [M, K]");
  if (int rc = check_shape(dtype, y, x->rows, x->cols, true, "layer_norm: y must be a dense [M, K]")) return rc;
  if ((uintptr_t)stats % 4) return bad("layer_norm: data must lie on whole elements");
  if (x->rows == 0 || r.dry) return VI_OK;
  NormArgs a{x->rows, (int)x->cols, view(x), {}, view(y), w, b, eps, stats, nullptr};
  const cudaError_t rc = launch_norm(dtype, a, false, r.sms, r.s, &r.launches);
  return rc == cudaSuccess ? VI_OK : set_error(VI_ERR_CUDA, cudaGetErrorString(rc));
}

int norm_backward(Run& r, int dtype, const vi_matrix* dy, const vi_matrix* x, const void* w, const float* stats, const vi_matrix* dx,
                  void* dw, void* db) {
  if (int rc = check_norm(dtype, x, w, nullptr, 0.0)) return rc;
  if (int rc = check_vector(dtype, dw)) return rc;
  if (int rc = check_vector(dtype, db)) return rc;
  const int64_t M = x->rows, K = x->cols;
  if (!given(dy) || dy->rows != M) return bad("layer_norm backward: dy is required, [M, K]");
  if (int rc = check_shape(dtype, dy, M, K, false, "layer_norm backward: dy must be [M, K]")) return rc;
  if (int rc = check_shape(dtype, dx, M, K, true, "layer_norm backward: dx must be a dense [M, K]")) return rc;
  if (!r.dry && M && !stats) return bad("layer_norm backward: stats is required");
  Summer sums{r, dtype};
  if (M == 0) {
    if (dw) sums.add(SumJob{nullptr, 0, 0, 0, 0, 1, K, nullptr, View{dw, 0, 1}});
    if (db) sums.add(SumJob{nullptr, 0, 0, 0, 0, 1, K, nullptr, View{db, 0, 1}});
    sums.run();
    return VI_OK;
  }
  NormArgs a{M, (int)K, view(x), view(dy), view(dx), w, nullptr, 0.0f, const_cast<float*>(stats), nullptr};
  const int pieces = norm_pieces(dtype, a, r.sms);
  if (dw || db) a.part = (float*)r.take((size_t)pieces * 2 * K * 4);
  if (!r.dry) {
    const cudaError_t rc = launch_norm(dtype, a, true, r.sms, r.s, &r.launches);
    if (rc != cudaSuccess) return set_error(VI_ERR_CUDA, cudaGetErrorString(rc));
  }
  if (dw) sums.add(SumJob{a.part, pieces, 2 * K, 0, 1, 1, K, nullptr, View{dw, 0, 1}});
  if (db) sums.add(SumJob{a.part + K, pieces, 2 * K, 0, 1, 1, K, nullptr, View{db, 0, 1}});
  sums.run();
  return VI_OK;
}

// ---- 8-bit integers ----
int quantize_rows(Run& r, int dtype, const vi_matrix* x, const vi_matrix* q, float* scale) {
  if (dtype < VI_F32 || dtype > VI_BF16) return bad("quantize_rows: unknown element type");
  if (!x || x->rows < 0 || x->cols < 1) return bad("quantize_rows: x needs at least one column");
  if (x->rows > kMaxSize || x->cols > kMaxSize) return bad("quantize_rows: sizes are limited to 2^30");
  if (!x->data && x->rows) return bad("quantize_rows: x needs data");
  if (x->row_stride < 0 || x->col_stride < 0) return bad("quantize_rows: strides must not be negative");
  if (int rc = check_vector(dtype, x->data)) return rc;
  if (!q || q->rows != x->rows || q->cols != x->cols || q->col_stride != 1 || (q->rows > 1 && q->row_stride < q->cols))
    return bad("quantize_rows: q must be [M, K] with contiguous rows");
  if (x->rows == 0 || r.dry) return VI_OK;
  if (!q->data || !scale || (uintptr_t)scale % 4) return bad("quantize_rows: q and scale are required");
  const cudaError_t rc =
      launch_quantize(dtype, QuantArgs{x->rows, (int)x->cols, view(x), (int8_t*)q->data, q->row_stride, scale}, r.sms, r.s);
  r.launches++;
  return rc == cudaSuccess ? VI_OK : set_error(VI_ERR_CUDA, cudaGetErrorString(rc));
}

// Rows of 8-bit integers as the tensor cores' copies read them: in place, or copied.
int operand8(Run& r, const vi_matrix* m, Operand& o) {
  o = Operand{m->data, m->rows, m->cols, m->row_stride, 0, true};
  if (m->col_stride == 1 && (m->row_stride >= m->cols || m->rows == 1) && (uintptr_t)m->data % 16 == 0 &&
      (m->row_stride % 16 == 0 || m->rows == 1) && m->row_stride < (1ll << 38)) {
    if (m->rows == 1) o.ld = ceil_div(m->cols, 16) * 16;
    return VI_OK;
  }
  o.ld = ceil_div(m->cols, 16) * 16;
  int8_t* dst = (int8_t*)r.take((size_t)m->rows * o.ld);
  o.p = dst;
  if (r.dry) return VI_OK;
  const cudaError_t rc = launch_pack8(view(m), m->rows, m->cols, dst, o.ld, r.s);
  r.launches++;
  return rc == cudaSuccess ? VI_OK : set_error(VI_ERR_CUDA, cudaGetErrorString(rc));
}

int int8_forward(Run& r, int dtype, int act, const vi_matrix* x, const float* x_scale, const vi_matrix* w, const float* w_scale,
                 const void* bias, const vi_matrix* res, const vi_matrix* y) {
  if (dtype < VI_F32 || dtype > VI_BF16) return bad("linear_act_int8: unknown element type");
  if (act < VI_ACT_NONE || act > VI_ACT_SIGMOID) return bad("linear_act_int8: unknown activation");
  if (!x || !w) return bad("linear_act_int8: x and weight are required");
  if (x->rows < 0 || x->cols < 1 || w->rows < 1) return bad("linear_act_int8: x needs at least one column and weight one row");
  if (w->cols != x->cols) return bad("linear_act_int8: weight and x differ in their number of columns");
  if (x->cols > kInt8Terms) return bad("linear_act_int8: sums of 2^17 columns and more do not fit 32 bits");
  if (x->rows > kMaxSize || w->rows > kMaxSize) return bad("linear_act_int8: sizes are limited to 2^30");
  if ((!x->data && x->rows) || !w->data || !w_scale) return bad("linear_act_int8: x, weight and its scale need data");
  if (x->row_stride < 0 || x->col_stride < 0 || w->row_stride < 0 || w->col_stride < 0)
    return bad("linear_act_int8: strides must not be negative");
  if ((!x_scale && (uintptr_t)x->data % elem(dtype)) || (uintptr_t)x_scale % 4 || (uintptr_t)w_scale % 4)
    return bad("linear_act_int8: data must lie on whole elements");
  if (int rc = check_vector(dtype, bias)) return rc;
  const int64_t M = x->rows, K = x->cols, N = w->rows;
  if (!given(y) || y->rows != M) return bad("linear_act_int8: y is required, [M, N]");
  if (int rc = check_shape(dtype, res, M, N, false, "linear_act_int8: residual must be [M, N]")) return rc;
  if (int rc = check_shape(dtype, y, M, N, true, "linear_act_int8: y must be a dense [M, N]")) return rc;
  if (M == 0) return VI_OK;
  Operand A{}, B{};
  Epilogue e{};
  e.act = act;
  e.bias = bias;
  e.res = view(res);
  e.out = view(y);
  e.col_scale = w_scale;
  e.row_scale = x_scale;
  if (!x_scale && int8_few(M, K)) {
    if (int rc = operand8(r, w, B)) return rc;
    if (r.dry) return VI_OK;
    const cudaError_t rc = launch_int8_few(dtype, M, view(x), B, e, r.s);
    r.launches++;
    return rc == cudaSuccess ? VI_OK : set_error(VI_ERR_CUDA, cudaGetErrorString(rc));
  }
  if (!x_scale && int8_fused(dtype, M, N, K, view(x))) {
    if (int rc = operand8(r, w, B)) return rc;
    return r.dry ? VI_OK : launch_int8_fused(dtype, M, view(x), B, e, r.sms, r.s);
  }
  if (x_scale) {
    if (int rc = operand8(r, x, A)) return rc;
  } else {
    A = Operand{nullptr, M, K, ceil_div(K, 16) * 16, 0, true};
    int8_t* q = (int8_t*)r.take((size_t)M * A.ld);
    float* s = (float*)r.take((size_t)M * 4);
    A.p = q;
    e.row_scale = s;
    if (!r.dry) {
      const cudaError_t rc = launch_quantize(dtype, QuantArgs{M, (int)K, view(x), q, A.ld, s}, r.sms, r.s);
      r.launches++;
      if (rc != cudaSuccess) return set_error(VI_ERR_CUDA, cudaGetErrorString(rc));
    }
  }
  if (int rc = operand8(r, w, B)) return rc;
  if (r.dry) return VI_OK;
  Plan p{};
  p.splits = 1;
  p.kps = (int)ceil_div(K, 128);
  if (e.out.rs == 1 && e.out.cs != 1 && 4 * N >= 3 * 128 * ceil_div(N, 128)) {  // as gemm()
    e.out = transposed(e.out);
    e.res = transposed(e.res);
    e.bias_rows = bias != nullptr;
    std::swap(e.row_scale, e.col_scale);
    std::swap(A, B);
  }
  // The float products' costs of tiles serve: within 6% of the best width of 64, 128 and 256 at 14 of 15 sizes from 100 x 4096 ->
  // 4096 to 65536 x 1024 -> 1024 and 2073600 x 96 -> 96; 14% at 65 channels of an image.
  p.bn = tile_width(dtype == VI_F32 ? VI_BF16 : dtype, kEpiInt8, A.rows, B.rows, 1, r.sms);
  return launch_int8_gemm(dtype, A, B, p, e, r.sms, r.s);
}

// ---- sample_labels ----
int sample_labels(Run& r, int dtype, const vi_matrix* z, const float* u, const vi_sampling* s, int64_t* label) {
  if (dtype < VI_F32 || dtype > VI_BF16) return bad("sample_labels: unknown element type");
  if (!z || !s) return bad("sample_labels: logits and settings are required");
  if (z->rows < 0 || z->cols < 1) return bad("sample_labels: logits need at least one column");
  if (z->rows > kMaxSize || z->cols > kMaxSize) return bad("sample_labels: sizes are limited to 2^30");
  if (z->row_stride < 0 || z->col_stride < 0) return bad("sample_labels: strides must not be negative");
  if (int rc = check_vector(dtype, z->data)) return rc;
  if (!s->temperatures && !(s->temperature >= 0.0)) return bad("sample_labels: temperature must be at least 0");
  if (!s->top_ks && s->top_k < 0) return bad("sample_labels: top_k must be at least 0");
  if (!s->top_ps && !(s->top_p > 0.0)) return bad("sample_labels: top_p must be above 0");
  if (!s->min_ps && !(s->min_p >= 0.0 && s->min_p <= 1.0)) return bad("sample_labels: min_p must lie in [0, 1]");
  if (z->rows == 0) return VI_OK;
  if (!z->data || (!r.dry && (!u || !label))) return bad("sample_labels: logits, u and label need data");
  if ((uintptr_t)u % 4 || (uintptr_t)s->temperatures % 4 || (uintptr_t)s->top_ps % 4 || (uintptr_t)s->min_ps % 4 ||
      (uintptr_t)s->top_ks % 8 || (uintptr_t)label % 8)
    return bad("sample_labels: data must lie on whole elements");
  // long rows keep candidates: as many rows at a time as fill the device many times over
  constexpr int64_t kRows = 16384;
  const uint64_t bytes = sample_scratch(std::min(z->rows, kRows), z->cols, r.sms);
  void* scratch = bytes ? r.take(bytes) : nullptr;
  if (r.dry) return VI_OK;
  const int64_t step = bytes ? kRows : z->rows;
  const size_t es = elem(dtype);
  for (int64_t m = 0; m < z->rows; m += step) {
    const auto from = [&](auto* p) { return p ? p + m : nullptr; };
    SampleArgs a{};
    a.M = std::min(step, z->rows - m);
    a.V = (int)z->cols;
    a.z = view(z);
    a.z.p = (char*)a.z.p + m * a.z.rs * es;
    a.u = u + m;
    a.temperature = from(s->temperatures);
    a.top_k = from(s->top_ks);
    a.top_p = from(s->top_ps);
    a.min_p = from(s->min_ps);
    a.temperature_all = s->temperature;
    a.top_p_all = s->top_p;
    a.min_p_all = s->min_p;
    a.top_k_all = s->top_k;
    a.label = label + m;
    a.scratch = scratch;
    const cudaError_t rc = launch_sample(dtype, a, r.sms, r.s);
    r.launches += bytes ? 2 : 1;
    if (rc != cudaSuccess) return set_error(VI_ERR_CUDA, cudaGetErrorString(rc));
  }
  return VI_OK;
}

}  // namespace
}  // namespace heads
}  // namespace vi

using namespace vi::heads;

extern "C" int vi_layer_norm_forward(int dtype, const vi_matrix* x, const void* weight, const void* bias, float eps,
                                     const vi_matrix* y, float* stats, void* stream) {
  return execute([&](Run& r) { return norm_forward(r, dtype, x, weight, bias, eps, y, stats); }, nullptr, 0, stream, "layer_norm");
}

extern "C" uint64_t vi_layer_norm_backward_scratch_bytes(int dtype, const vi_matrix* dy, const vi_matrix* x, const void* weight,
                                                         const vi_matrix* dx, const void* dweight, const void* dbias) {
  return count_bytes([&](Run& r) {
    return norm_backward(r, dtype, dy, x, weight, nullptr, dx, const_cast<void*>(dweight), const_cast<void*>(dbias));
  });
}

extern "C" int vi_layer_norm_backward(int dtype, const vi_matrix* dy, const vi_matrix* x, const void* weight, const float* stats,
                                      const vi_matrix* dx, void* dweight, void* dbias, void* scratch, uint64_t scratch_bytes,
                                      void* stream) {
  return execute([&](Run& r) { return norm_backward(r, dtype, dy, x, weight, stats, dx, dweight, dbias); }, scratch, scratch_bytes,
                 stream, "layer_norm backward");
}

extern "C" int vi_quantize_rows(int dtype, const vi_matrix* x, const vi_matrix* q, float* scale, void* stream) {
  return execute([&](Run& r) { return quantize_rows(r, dtype, x, q, scale); }, nullptr, 0, stream, "quantize_rows");
}

extern "C" uint64_t vi_linear_act_int8_scratch_bytes(int dtype, int activation, const vi_matrix* x, const float* x_scale,
                                                     const vi_matrix* weight, const float* weight_scale, const void* bias,
                                                     const vi_matrix* residual, const vi_matrix* y) {
  return count_bytes(
      [&](Run& r) { return int8_forward(r, dtype, activation, x, x_scale, weight, weight_scale, bias, residual, y); });
}

extern "C" int vi_linear_act_int8(int dtype, int activation, const vi_matrix* x, const float* x_scale, const vi_matrix* weight,
                                  const float* weight_scale, const void* bias, const vi_matrix* residual, const vi_matrix* y,
                                  void* scratch, uint64_t scratch_bytes, void* stream) {
  return execute(
      [&](Run& r) { return int8_forward(r, dtype, activation, x, x_scale, weight, weight_scale, bias, residual, y); }, scratch,
      scratch_bytes, stream, "linear_act_int8");
}

extern "C" uint64_t vi_sample_labels_scratch_bytes(int dtype, const vi_matrix* logits, const vi_sampling* settings) {
  return count_bytes([&](Run& r) { return sample_labels(r, dtype, logits, nullptr, settings, nullptr); });
}

extern "C" int vi_sample_labels(int dtype, const vi_matrix* logits, const float* u, const vi_sampling* settings, int64_t* label,
                                void* scratch, uint64_t scratch_bytes, void* stream) {
  return execute([&](Run& r) { return sample_labels(r, dtype, logits, u, settings, label); }, scratch, scratch_bytes, stream,
                 "sample_labels");
}

extern "C" uint64_t vi_linear_act_forward_scratch_bytes(int dtype, int activation, const vi_matrix* x,
                                                        const vi_matrix* weight, const void* bias,
                                                        const vi_matrix* residual, const vi_matrix* y,
                                                        const vi_matrix* dact) {
  return count_bytes([&](Run& r) { return act_forward(r, dtype, activation, x, weight, bias, residual, y, dact); });
}

extern "C" int vi_linear_act_forward(int dtype, int activation, const vi_matrix* x, const vi_matrix* weight,
                                     const void* bias, const vi_matrix* residual, const vi_matrix* y,
                                     const vi_matrix* dact, void* scratch, uint64_t scratch_bytes, void* stream) {
  return execute([&](Run& r) { return act_forward(r, dtype, activation, x, weight, bias, residual, y, dact); }, scratch,
                 scratch_bytes, stream, "linear_act");
}

extern "C" int vi_linear_act_keeps_dact(int dtype, int activation, const vi_matrix* x, const vi_matrix* weight) {
  if (check_operands(dtype, x, weight) || activation == VI_ACT_NONE) return 0;
  const View v = view(x);
  return !narrow_backward(weight->rows, x->cols, v, View{v.p, 1, 2}, View{v.p, 1, 2});
}

extern "C" uint64_t vi_linear_act_backward_scratch_bytes(int dtype, int activation, const vi_matrix* dy,
                                                         const vi_matrix* dact, const vi_matrix* x,
                                                         const vi_matrix* weight, const void* bias,
                                                         const vi_matrix* dx, const vi_matrix* dweight,
                                                         const void* dbias) {
  return count_bytes([&](Run& r) {
    return act_backward(r, dtype, activation, dy, dact, x, weight, bias, dx, dweight, const_cast<void*>(dbias));
  });
}

extern "C" int vi_linear_act_backward(int dtype, int activation, const vi_matrix* dy, const vi_matrix* dact,
                                      const vi_matrix* x, const vi_matrix* weight, const void* bias,
                                      const vi_matrix* dx, const vi_matrix* dweight, void* dbias, void* scratch,
                                      uint64_t scratch_bytes, void* stream) {
  return execute(
      [&](Run& r) { return act_backward(r, dtype, activation, dy, dact, x, weight, bias, dx, dweight, dbias); }, scratch,
      scratch_bytes, stream, "linear_act backward");
}

extern "C" uint64_t vi_linear_ce_forward_scratch_bytes(int dtype, const vi_matrix* x, const vi_matrix* weight,
                                                       const void* bias) {
  return count_bytes([&](Run& r) { return ce_forward(r, dtype, x, weight, bias, nullptr, 0, 0, nullptr, nullptr); });
}

extern "C" int vi_linear_ce_forward(int dtype, const vi_matrix* x, const vi_matrix* weight, const void* bias,
                                    const int64_t* target, int64_t ignore_index, int reduction, float* loss, float* lse,
                                    void* scratch, uint64_t scratch_bytes, void* stream) {
  return execute(
      [&](Run& r) { return ce_forward(r, dtype, x, weight, bias, target, ignore_index, reduction, loss, lse); }, scratch,
      scratch_bytes, stream, "linear_ce");
}

extern "C" uint64_t vi_linear_ce_backward_scratch_bytes(int dtype, const vi_matrix* x, const vi_matrix* weight,
                                                        const void* bias, const vi_matrix* dx,
                                                        const vi_matrix* dweight, const void* dbias) {
  return count_bytes([&](Run& r) {
    return ce_backward(r, dtype, x, weight, bias, nullptr, 0, 0, nullptr, nullptr, dx, dweight,
                       const_cast<void*>(dbias));
  });
}

extern "C" int vi_linear_ce_backward(int dtype, const vi_matrix* x, const vi_matrix* weight, const void* bias,
                                     const int64_t* target, int64_t ignore_index, int reduction, const float* lse,
                                     const float* dloss, const vi_matrix* dx, const vi_matrix* dweight, void* dbias,
                                     void* scratch, uint64_t scratch_bytes, void* stream) {
  return execute(
      [&](Run& r) {
        return ce_backward(r, dtype, x, weight, bias, target, ignore_index, reduction, lse, dloss, dx, dweight, dbias);
      },
      scratch, scratch_bytes, stream, "linear_ce backward");
}
