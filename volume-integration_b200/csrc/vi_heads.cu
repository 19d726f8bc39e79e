// Per-pixel heads: dense layers and the label loss on rendered feature images.
//
// Mathematics.  Both operators are one product z = x W^T + b with an epilogue:
//   linear_act            y = act(z) + r
//                         s = dy * act'(z); dx = s W; dW = s^T x; db = sum_m s
//   linear_cross_entropy  l_m = log sum_v exp z_mv - z_m,t
//                         G = g_m (softmax(z) - onehot(t)); dx = G W; dW = G^T x; db = sum_m G
// Sums, the softmax's maximum and sum, and biases' gradients are float32; sums over
// rows are split into pieces that are added in a fixed order, so results do not
// depend on scheduling.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdio>

#include "vi_heads.h"
#include "vi_internal.h"

namespace vi {
namespace heads {
namespace {

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

// act(z) and act'(z).  A NaN stays a NaN.
__device__ __forceinline__ void activate(int act, float z, float& y, float& d) {
  switch (act) {
    case VI_ACT_RELU:
      y = z <= 0.0f ? 0.0f : z;
      d = z > 0.0f ? 1.0f : 0.0f;
      break;
    case VI_ACT_SILU: {
      const float s = 1.0f / (1.0f + expf(-z)), c = 1.0f / (1.0f + expf(z));
      y = z * s;
      d = s * (1.0f + z * c);
      break;
    }
    case VI_ACT_GELU: {
      const float cdf = normcdff(z);
      y = z * cdf;
      d = cdf + z * 0.3989422804f * expf(-0.5f * z * z);
      break;
    }
    case VI_ACT_SIGMOID: {
      const float s = 1.0f / (1.0f + expf(-z)), c = 1.0f / (1.0f + expf(z));
      y = s;
      d = s * c;
      break;
    }
    default:
      y = z;
      d = 1.0f;
  }
}

constexpr int kTile = 64;  // output tile of one block, and of its 256 threads' 4x4 pieces
constexpr int kDepth = 16;

// acc(m, n) = sum_k A(m, k) B(n, k) on the FP32 cores, any strides; blockIdx.z
// takes columns [z * ksplit, (z + 1) * ksplit) of the sum (kEpiPartial).
template <typename T>
__global__ void __launch_bounds__(256) gemm_kernel(View A, View B, int64_t M, int64_t N, int64_t K, int64_t ksplit,
                                                   Epilogue e) {
  __shared__ float sa[kDepth][kTile + 4], sb[kDepth][kTile + 4];
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  const int64_t m0 = (int64_t)blockIdx.x * kTile, n0 = (int64_t)blockIdx.y * kTile;
  const int64_t k_begin = blockIdx.z * ksplit, k_end = min(K, k_begin + ksplit);
  const T* a = (const T*)A.p;
  const T* b = (const T*)B.p;
  float acc[4][4] = {};
  for (int64_t k0 = k_begin; k0 < k_end; k0 += kDepth) {
    for (int i = tid; i < kTile * kDepth; i += 256) {
      // neighbouring threads along whichever axis is contiguous
      const int ra = A.cs == 1 ? i / kDepth : i % kTile, ca = A.cs == 1 ? i % kDepth : i / kTile;
      const int rb = B.cs == 1 ? i / kDepth : i % kTile, cb = B.cs == 1 ? i % kDepth : i / kTile;
      sa[ca][ra] = m0 + ra < M && k0 + ca < k_end ? to_f(a[(m0 + ra) * A.rs + (k0 + ca) * A.cs]) : 0.0f;
      sb[cb][rb] = n0 + rb < N && k0 + cb < k_end ? to_f(b[(n0 + rb) * B.rs + (k0 + cb) * B.cs]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; k++) {
      float fa[4], fb[4];
#pragma unroll
      for (int i = 0; i < 4; i++) fa[i] = sa[k][ty * 4 + i], fb[i] = sb[k][tx * 4 + i];
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = fmaf(fa[i], fb[j], acc[i][j]);
    }
    __syncthreads();
  }
  const float alpha = e.alpha ? *e.alpha : 1.0f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int64_t m = m0 + ty * 4 + i;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t n = n0 + tx * 4 + j;
      if (m >= M || n >= N) continue;
      float z = acc[i][j];
      if (e.bias) z += to_f(((const T*)e.bias)[n]);
      if (e.kind == kEpiAct) {
        float y, d;
        activate(e.act, z, y, d);
        if (e.res.p) y += to_f(((const T*)e.res.p)[m * e.res.rs + n * e.res.cs]);
        ((T*)e.out.p)[m * e.out.rs + n * e.out.cs] = from_f<T>(y);
        if (e.dact.p) ((T*)e.dact.p)[m * e.dact.rs + n * e.dact.cs] = from_f<T>(d);
      } else if (e.kind == kEpiStore) {
        ((T*)e.out.p)[m * e.out.rs + n * e.out.cs] = from_f<T>(alpha * z);
      } else if (e.kind == kEpiPartial) {
        e.part[((int64_t)blockIdx.z * M + m) * N + n] = z;
      } else if (e.kind == kEpiLse) {
        acc[i][j] = z;
        top = fmaxf(top, z);
        if (n == e.target[m]) e.ztarget[m] = z;
      } else {
        const float c = e.coef[m];
        const float p = c == 0.0f ? 0.0f : expf(z - e.lse[m]) - (n + e.col0 == e.target[m] ? 1.0f : 0.0f);
        ((T*)e.out.p)[m * e.out.rs + n * e.out.cs] = from_f<T>(p * c);
      }
    }
    if (e.kind == kEpiLse) {  // the 16 threads of a row are 16 neighbouring lanes
      for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      float sum = 0.0f;
      for (int j = 0; j < 4; j++)
        if (m < M && n0 + tx * 4 + j < N) sum += top == -INFINITY && acc[i][j] == top ? 0.0f : expf(acc[i][j] - top);
      for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (tx == 0 && m < M) {
        e.pmax[(int64_t)blockIdx.y * M + m] = top;
        e.psum[(int64_t)blockIdx.y * M + m] = sum;
      }
    }
  }
}

// s = dy * dact (dact null: a copy of dy), in dact's order; columns' sums in pieces.
template <typename T>
__global__ void scale_kernel(View dy, View dact, View s, int64_t M, int64_t N) {
  const int64_t total = M * N;
  const bool by_col = s.cs == 1;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t m = by_col ? i / N : i % M, n = by_col ? i % N : i / M;
    ((T*)s.p)[m * s.rs + n * s.cs] = from_f<T>(to_f(((const T*)dy.p)[m * dy.rs + n * dy.cs]) *
                                               to_f(((const T*)dact.p)[m * dact.rs + n * dact.cs]));
  }
}

// part[piece][n] = sum of column n over the piece's rows.
template <typename T>
__global__ void column_sums_kernel(View s, int64_t M, int64_t N, int64_t rows, float* part) {
  __shared__ float sh[8][33];
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  const int64_t n = (int64_t)blockIdx.x * 32 + lane, m_end = min(M, (blockIdx.y + 1) * rows);
  float sum = 0.0f;
  if (n < N)
    for (int64_t m = blockIdx.y * rows + w; m < m_end; m += 8) sum += to_f(((const T*)s.p)[m * s.rs + n * s.cs]);
  sh[w][lane] = sum;
  __syncthreads();
  if (w == 0 && n < N) {
    for (int i = 1; i < 8; i++) sum += sh[i][lane];
    part[(int64_t)blockIdx.y * N + n] = sum;
  }
}

// out(i / cols, i % cols) = alpha * sum of the pieces, added in order.
template <typename T>
__global__ void sum_pieces_kernel(const float* part, int pieces, int64_t rows, int64_t cols, const float* alpha,
                                  View out) {
  const int64_t total = rows * cols;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    float sum = 0.0f;
    for (int p = 0; p < pieces; p++) sum += part[(int64_t)p * total + i];
    ((T*)out.p)[i / cols * out.rs + i % cols * out.cs] = from_f<T>(sum * (alpha ? *alpha : 1.0f));
  }
}

// Rows' losses from the spans' maxima and sums; per block the sum of its rows' losses and their count.
__global__ void __launch_bounds__(256) loss_kernel(const float* pmax, const float* psum, const float* ztarget,
                                                   int spans, int64_t M, int64_t V, const int64_t* target,
                                                   int64_t ignore, float* rows, float* lse, float* bsum,
                                                   float* bcount) {
  __shared__ float sh[2][8];
  const int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x;
  float loss = 0.0f, live = 0.0f;
  if (m < M) {
    float top = -INFINITY, sum = 0.0f;
    for (int i = 0; i < spans; i++) top = fmaxf(top, pmax[(int64_t)i * M + m]);
    for (int i = 0; i < spans; i++) {
      const float p = pmax[(int64_t)i * M + m];
      sum += psum[(int64_t)i * M + m] * (p == top ? 1.0f : expf(p - top));
    }
    const float l = top + logf(sum);
    const int64_t t = target[m];
    const bool ignored = t == ignore, bad = !ignored && (t < 0 || t >= V);
    lse[m] = bad ? NAN : l;
    loss = ignored ? 0.0f : bad ? NAN : l - ztarget[m];
    live = ignored ? 0.0f : 1.0f;
    if (rows) rows[m] = loss;
  }
  for (int o = 16; o; o >>= 1) {
    loss += __shfl_xor_sync(0xffffffffu, loss, o);
    live += __shfl_xor_sync(0xffffffffu, live, o);
  }
  if (threadIdx.x % 32 == 0) sh[0][threadIdx.x / 32] = loss, sh[1][threadIdx.x / 32] = live;
  __syncthreads();
  if (threadIdx.x == 0 && bsum) {
    for (int i = 1; i < 8; i++) loss += sh[0][i], live += sh[1][i];
    bsum[blockIdx.x] = loss;
    bcount[blockIdx.x] = live;
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
// products' epilogue instead (alpha): G is kept in T, and float16 would lose
// probabilities divided by a pixel count.  lift (a power of two) moves float16's G
// up further, so that a probability keeps float16's full precision down to 4e-9.
// One block.
__global__ void __launch_bounds__(1024) coef_kernel(const int64_t* target, int64_t ignore, int64_t M, int reduction,
                                                    const float* dloss, float lift, float* coef, float* alpha) {
  __shared__ float shm[32];
  __shared__ unsigned long long shc[32];
  float top = 0.0f;
  unsigned long long live = 0;
  for (int64_t m = threadIdx.x; m < M; m += 1024) {
    const bool on = target[m] != ignore;
    live += on;
    if (reduction == VI_REDUCE_NONE && on && isfinite(dloss[m])) top = fmaxf(top, fabsf(dloss[m]));
  }
  for (int o = 16; o; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    live += __shfl_xor_sync(0xffffffffu, live, o);
  }
  if (threadIdx.x % 32 == 0) shm[threadIdx.x / 32] = top, shc[threadIdx.x / 32] = live;
  __syncthreads();
  top = 0.0f;
  live = 0;
  for (int i = 0; i < 32; i++) top = fmaxf(top, shm[i]), live += shc[i];
  int ex = 0;
  frexpf(top, &ex);
  ex = min(max(ex, -100), 100);  // a power of two at or above every finite |g|: the division is exact
  if (threadIdx.x == 0)
    *alpha = (reduction == VI_REDUCE_NONE ? ldexpf(1.0f, ex)
              : reduction == VI_REDUCE_SUM ? *dloss
              : live                       ? *dloss / (float)live
                                           : 0.0f) / lift;
  for (int64_t m = threadIdx.x; m < M; m += 1024) {
    const float g = reduction == VI_REDUCE_NONE ? ldexpf(dloss[m], -ex) : 1.0f;
    coef[m] = target[m] != ignore ? g * lift : 0.0f;
  }
}

// x with the rows of ignored targets set to zero: their zero gradient times a
// NaN or an infinity would else reach the weights' gradient.  In x's own order.
template <typename T>
__global__ void live_rows_kernel(View x, const float* coef, View out, int64_t M, int64_t K) {
  const int64_t total = M * K;
  const bool by_col = out.cs == 1;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t m = by_col ? i / K : i % M, k = by_col ? i % K : i / M;
    ((T*)out.p)[m * out.rs + k * out.cs] = coef[m] == 0.0f ? from_f<T>(0.0f) : ((const T*)x.p)[m * x.rs + k * x.cs];
  }
}

// ---------------------------------------------------------------------------
// Host side.  One function per operator carves the scratch and launches; with
// `dry` it only carves, which is how the _scratch_bytes queries count.
// ---------------------------------------------------------------------------
struct Run {
  char* base;
  cudaStream_t s;
  bool dry;
  size_t cur = 0;
  int launches = 0;
  void* take(size_t bytes) {
    cur = align_up(cur);
    char* p = base + cur;
    cur += bytes;
    return p;
  }
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int grid_for(int64_t n) { return (int)std::min<int64_t>(ceil_div(n, 256), 148 * 16); }
size_t elem(int dtype) { return dtype == VI_F32 ? 4 : 2; }
View view(const vi_matrix* m) { return m ? View{m->data, m->row_stride, m->col_stride} : View{nullptr, 0, 0}; }
View transposed(View v) { return View{v.p, v.cs, v.rs}; }
bool by_rows(const View& v) { return v.cs == 1; }
// An [rows, cols] scratch matrix in the memory order of `like`.
View scratch_like(void* p, const View& like, int64_t rows, int64_t cols) {
  return by_rows(like) ? View{p, cols, 1} : View{p, 1, rows};
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

void gemm(Run& r, int dtype, View A, View B, int64_t M, int64_t N, int64_t K, int64_t ksplit, int splits,
          const Epilogue& e) {
  if (r.dry) return;
  const dim3 grid((unsigned)ceil_div(M, kTile), (unsigned)ceil_div(N, kTile), splits);
  VI_DISPATCH(dtype, (gemm_kernel<T><<<grid, 256, 0, r.s>>>(A, B, M, N, K, ksplit, e)));
  r.launches++;
}

// out = alpha * A B^T with a long sum: pieces of it in float32, added in order.
void gemm_split(Run& r, int dtype, View A, View B, int64_t M, int64_t N, int64_t K, const float* alpha, View out) {
  const int64_t tiles = ceil_div(M, kTile) * ceil_div(N, kTile);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(ceil_div(148 * 4, tiles), ceil_div(K, 512)));
  const int64_t ksplit = ceil_div(ceil_div(K, want), kDepth) * kDepth;
  const int splits = (int)ceil_div(K, ksplit);
  float* part = (float*)r.take((size_t)splits * M * N * 4);
  Epilogue e{};
  e.kind = kEpiPartial;
  e.part = part;
  gemm(r, dtype, A, B, M, N, K, ksplit, splits, e);
  if (r.dry) return;
  VI_DISPATCH(dtype, (sum_pieces_kernel<T><<<grid_for(M * N), 256, 0, r.s>>>(part, splits, M, N, alpha, out)));
  r.launches++;
}

// out[n] = alpha * sum over rows of s.
void column_sums(Run& r, int dtype, View s, int64_t M, int64_t N, const float* alpha, void* out) {
  const int64_t blocks = ceil_div(N, 32);
  const int64_t pieces = std::max<int64_t>(1, std::min<int64_t>(ceil_div(148 * 8, blocks), ceil_div(M, 64)));
  const int64_t rows = ceil_div(M, pieces);
  float* part = (float*)r.take((size_t)pieces * N * 4);
  if (r.dry) return;
  VI_DISPATCH(dtype, (column_sums_kernel<T><<<dim3((unsigned)blocks, (unsigned)pieces), 256, 0, r.s>>>(s, M, N, rows, part)));
  VI_DISPATCH(dtype, (sum_pieces_kernel<T><<<grid_for(N), 256, 0, r.s>>>(part, (int)pieces, 1, N, alpha, View{out, 0, 1})));
  r.launches += 2;
}

// Gradients of the weights over no rows at all.
void zero_gradients(Run& r, int dtype, int64_t N, int64_t K, const vi_matrix* dw, void* db) {
  if (r.dry) return;
  if (dw && dw->data) {
    VI_DISPATCH(dtype, (sum_pieces_kernel<T><<<grid_for(N * K), 256, 0, r.s>>>(nullptr, 0, N, K, nullptr, view(dw))));
    r.launches++;
  }
  if (db) {
    VI_DISPATCH(dtype, (sum_pieces_kernel<T><<<grid_for(N), 256, 0, r.s>>>(nullptr, 0, 1, N, nullptr, View{db, 0, 1})));
    r.launches++;
  }
}

// ---- argument checks ----
int bad(const char* msg) { return set_error(VI_ERR_INVALID_ARGUMENT, msg); }

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
  if (x->rows > INT32_MAX || w->rows > INT32_MAX || x->cols > INT32_MAX) return bad("heads: sizes are limited to 2^31 - 1");
  if ((!x->data && x->rows) || !w->data) return bad("heads: x and weight need data");
  if (x->row_stride < 0 || x->col_stride < 0 || w->row_stride < 0 || w->col_stride < 0)
    return bad("heads: strides must not be negative");
  return VI_OK;
}
int check_shape(const vi_matrix* m, int64_t rows, int64_t cols, bool need_dense, const char* msg) {
  if (!m || !m->data) return VI_OK;
  if (m->rows != rows || m->cols != cols || m->row_stride < 0 || m->col_stride < 0) return bad(msg);
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

template <class F>
uint64_t count_bytes(F&& f) {
  Run r{nullptr, nullptr, true};
  return f(r) == VI_OK ? align_up(r.cur) + 256 : 0;
}
template <class F>
int execute(F&& f, void* scratch, uint64_t bytes, void* stream, const char* where) {
  Run d{nullptr, nullptr, true};
  int rc = f(d);
  if (rc) return rc;
  if (d.cur > bytes || (d.cur && (!scratch || (uintptr_t)scratch % 256)))
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
  const int64_t M = x->rows, K = x->cols, N = w->rows;
  if (!given(y) || y->rows != M) return bad("linear_act: y is required, [M, N]");
  if (int rc = check_shape(res, M, N, false, "linear_act: residual must be [M, N]")) return rc;
  if (int rc = check_shape(y, M, N, true, "linear_act: y must be a dense [M, N]")) return rc;
  if (int rc = check_shape(dact, M, N, true, "linear_act: dact must be a dense [M, N]")) return rc;
  if (dact && dact->data && (dact->row_stride != y->row_stride || dact->col_stride != y->col_stride))
    return bad("linear_act: dact must have y's strides");
  if (M == 0) return VI_OK;
  Epilogue e{};
  e.kind = kEpiAct;
  e.act = act;
  e.bias = bias;
  e.res = view(res);
  e.out = view(y);
  e.dact = view(dact);
  gemm(r, dtype, view(x), view(w), M, N, K, K, 1, e);
  return VI_OK;
}

int act_backward(Run& r, int dtype, const vi_matrix* dy, const vi_matrix* dact, const vi_matrix* x,
                 const vi_matrix* w, const vi_matrix* dx, const vi_matrix* dw, void* db) {
  if (int rc = check_operands(dtype, x, w)) return rc;
  const int64_t M = x->rows, K = x->cols, N = w->rows;
  if (!given(dy) || dy->rows != M) return bad("linear_act backward: dy is required, [M, N]");
  if (int rc = check_shape(dy, M, N, false, "linear_act backward: dy must be [M, N]")) return rc;
  if (int rc = check_shape(dact, M, N, true, "linear_act backward: dact must be a dense [M, N]")) return rc;
  if (int rc = check_shape(dx, M, K, true, "linear_act backward: dx must be a dense [M, K]")) return rc;
  if (int rc = check_shape(dw, N, K, true, "linear_act backward: dweight must be a dense [N, K]")) return rc;
  const size_t es = elem(dtype);
  if (M == 0) {
    zero_gradients(r, dtype, N, K, dw, db);
    return VI_OK;
  }
  View s = view(dy);
  if (dact && dact->data) {
    s = scratch_like(r.take((size_t)M * N * es), view(dact), M, N);
    if (!r.dry) {
      VI_DISPATCH(dtype, (scale_kernel<T><<<grid_for(M * N), 256, 0, r.s>>>(view(dy), view(dact), s, M, N)));
      r.launches++;
    }
  }
  if (dx && dx->data) {
    Epilogue e{};
    e.kind = kEpiStore;
    e.out = view(dx);
    gemm(r, dtype, s, transposed(view(w)), M, K, N, N, 1, e);
  }
  if (dw && dw->data) gemm_split(r, dtype, transposed(s), transposed(view(x)), N, K, M, nullptr, view(dw));
  if (db) column_sums(r, dtype, s, M, N, nullptr, db);
  return VI_OK;
}

// ---- linear_cross_entropy ----
int ce_forward(Run& r, int dtype, const vi_matrix* x, const vi_matrix* w, const void* bias, const int64_t* target,
               int64_t ignore, int reduction, float* loss, float* lse) {
  if (int rc = check_operands(dtype, x, w)) return rc;
  if (reduction < VI_REDUCE_NONE || reduction > VI_REDUCE_SUM) return bad("linear_ce: unknown reduction");
  const int64_t M = x->rows, K = x->cols, V = w->rows;
  if (!r.dry && M && (!target || !loss || !lse)) return bad("linear_ce: target, loss and lse are required");
  const int spans = (int)ceil_div(V, kTile);
  const int64_t blocks = ceil_div(M, 256);
  float* pmax = (float*)r.take((size_t)spans * M * 4);
  float* psum = (float*)r.take((size_t)spans * M * 4);
  float* zt = (float*)r.take((size_t)M * 4);
  float* bsum = (float*)r.take((size_t)blocks * 4);
  float* bcount = (float*)r.take((size_t)blocks * 4);
  if (r.dry) return VI_OK;
  if (M) {
    Epilogue e{};
    e.kind = kEpiLse;
    e.bias = bias;
    e.pmax = pmax;
    e.psum = psum;
    e.ztarget = zt;
    e.target = target;
    gemm(r, dtype, view(x), view(w), M, V, K, K, 1, e);
    const bool none = reduction == VI_REDUCE_NONE;
    loss_kernel<<<(unsigned)blocks, 256, 0, r.s>>>(pmax, psum, zt, spans, M, V, target, ignore, none ? loss : nullptr,
                                                   lse, none ? nullptr : bsum, bcount);
    r.launches++;
  }
  if (reduction != VI_REDUCE_NONE) {
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
  const int64_t M = x->rows, K = x->cols, V = w->rows;
  if (int rc = check_shape(dx, M, K, true, "linear_ce backward: dx must be a dense [M, K]")) return rc;
  if (int rc = check_shape(dw, V, K, true, "linear_ce backward: dweight must be a dense [V, K]")) return rc;
  if (!r.dry && M && (!target || !lse || !dloss)) return bad("linear_ce backward: target, lse and dloss are required");
  const size_t es = elem(dtype);
  if (M == 0) {
    zero_gradients(r, dtype, V, K, dw, db);
    return VI_OK;
  }
  float* coef = (float*)r.take((size_t)M * 4);
  float* alpha = (float*)r.take(4);
  View G{r.take((size_t)M * V * es), V, 1};
  View xl = view(x);
  if (dw && dw->data) xl = scratch_like(r.take((size_t)M * K * es), view(x), M, K);
  if (!r.dry) {
    coef_kernel<<<1, 1024, 0, r.s>>>(target, ignore, M, reduction, dloss, dtype == VI_F16 ? 16384.0f : 1.0f, coef, alpha);
    r.launches++;
    if (dw && dw->data) {
      VI_DISPATCH(dtype, (live_rows_kernel<T><<<grid_for(M * K), 256, 0, r.s>>>(view(x), coef, xl, M, K)));
      r.launches++;
    }
  }
  Epilogue e{};
  e.kind = kEpiGrad;
  e.bias = bias;
  e.out = G;
  e.target = target;
  e.lse = lse;
  e.coef = coef;
  gemm(r, dtype, view(x), view(w), M, V, K, K, 1, e);
  if (dx && dx->data) {
    Epilogue d{};
    d.kind = kEpiStore;
    d.out = view(dx);
    d.alpha = alpha;
    gemm(r, dtype, G, transposed(view(w)), M, K, V, V, 1, d);
  }
  if (dw && dw->data) gemm_split(r, dtype, transposed(G), transposed(xl), V, K, M, alpha, view(dw));
  if (db) column_sums(r, dtype, G, M, V, alpha, db);
  return VI_OK;
}

}  // namespace
}  // namespace heads
}  // namespace vi

using namespace vi::heads;

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

extern "C" uint64_t vi_linear_act_backward_scratch_bytes(int dtype, const vi_matrix* dy, const vi_matrix* dact,
                                                         const vi_matrix* x, const vi_matrix* weight,
                                                         const vi_matrix* dx, const vi_matrix* dweight,
                                                         const void* dbias) {
  return count_bytes(
      [&](Run& r) { return act_backward(r, dtype, dy, dact, x, weight, dx, dweight, const_cast<void*>(dbias)); });
}

extern "C" int vi_linear_act_backward(int dtype, const vi_matrix* dy, const vi_matrix* dact, const vi_matrix* x,
                                      const vi_matrix* weight, const vi_matrix* dx, const vi_matrix* dweight,
                                      void* dbias, void* scratch, uint64_t scratch_bytes, void* stream) {
  return execute([&](Run& r) { return act_backward(r, dtype, dy, dact, x, weight, dx, dweight, dbias); }, scratch,
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
