// Rows of 8-bit integers with a scale each.
//
// Mathematics.  s = f32(max_k |x_k| / 127), q_k = x_k / s rounded to the nearest whole number, ties to even: |q| <= 127.
// The rounding is that of the exact quotient: x times the rounded 1 / s decides it, but near halves, where the exact rest
// x - q s does.  A row of zeros has s = 0 and q = 0; one that holds an infinity or a NaN has s = NaN and q = 0, so
// that what is made of it is NaN.
//
// One pass over x, held in registers between the maximum and the rounding; memory bounds long rows (32768 x 1024 in float16: 25 us,
// 15 at the copy rate), instructions short ones (2073600 x 64 in bfloat16: 132 us, 61; as an image 285).
#include <algorithm>
#include <type_traits>

#include "vi_heads.h"
#include "vi_heads_math.cuh"
#include "vi_internal.h"
#include "vi_quant.cuh"
#include "vi_rows.cuh"

namespace vi {
namespace heads {
namespace {

constexpr int kThreads = 256;

// The bits of magnitudes, which order as they do, infinities and NaNs last.  Two 16-bit ones at a time.
template <typename T, int N>
__device__ __forceinline__ uint32_t magnitude(const Chunk<T, N>& c, uint32_t top) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; i++) top = max(top, __float_as_uint(to_f(c.v[i])) & 0x7fffffffu);
  } else if constexpr (N == 1) {
    top = max(top, (uint32_t)(*(const uint16_t*)&c.v[0] & 0x7fff));
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; i++) top = __vmaxu2(top, ((const uint32_t*)c.v)[i] & 0x7fff7fffu);
  }
  return top;
}
// The magnitude as float32's bits: of one, or the larger of two.
template <typename T>
__device__ __forceinline__ uint32_t magnitude_bits(uint32_t top) {
  if constexpr (sizeof(T) == 4) {
    return top;
  } else {
    const uint16_t m = (uint16_t)max(top & 0xffffu, top >> 16);
    return __float_as_uint(to_f(*(const T*)&m));
  }
}

// Rows of contiguous features: a row belongs to `lanes` lanes, or to a block; R rows at a time.
template <typename T, int VEC, int NV, int R, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : kThreads) quantize_rows_kernel(const __grid_constant__ QuantArgs a, int lanes) {
  __shared__ uint32_t sh[2][16];
  int turn = 0;
  const int lane = BLOCK ? threadIdx.x : threadIdx.x % lanes, group = BLOCK ? 0 : threadIdx.x / lanes;
  const int groups = BLOCK ? 1 : kThreads / lanes;
  for (int64_t m0 = (int64_t)blockIdx.x * groups * R; m0 < a.M; m0 += (int64_t)gridDim.x * groups * R) {
    Chunk<T, VEC> x[R][NV];
#pragma unroll
    for (int r = 0; r < R; r++) load_row(x[r], a.x, min(m0 + r * groups + group, a.M - 1), a.K, lanes, lane);
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int64_t m = m0 + r * groups + group;
      uint32_t top = 0;
#pragma unroll
      for (int v = 0; v < NV; v++) top = magnitude(x[r][v], top);
      top = magnitude_bits<T>(top);
      if constexpr (BLOCK) {
        top = __reduce_max_sync(0xffffffffu, top);
        if (threadIdx.x % 32 == 0) sh[turn][threadIdx.x / 32] = top;
        __syncthreads();
        for (int w = 0; w < blockDim.x / 32; w++) top = max(top, sh[turn][w]);
        turn ^= 1;
      } else if (lanes == 32) {
        top = __reduce_max_sync(0xffffffffu, top);
      } else {
        for (int o = lanes / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      }
      const Scale s(top);
      if (m >= a.M) continue;
      int8_t* q = a.q + m * a.ld;
#pragma unroll
      for (int v = 0; v < NV; v++) {
        const int at = (v * lanes + lane) * VEC;
        if (at >= a.K) continue;
        float f[VEC];
        int b[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) f[i] = to_f(x[r][v].v[i]);
        quantize(f, s, b);
        if constexpr (VEC == 1) q[at] = (int8_t)b[0];
        else if constexpr (VEC == 4) *(uint32_t*)(q + at) = bytes4(b[0], b[1], b[2], b[3]);
        else *(uint2*)(q + at) = make_uint2(bytes4(b[0], b[1], b[2], b[3]), bytes4(b[4], b[5], b[6], b[7]));
      }
      if (lane == 0) a.scale[m] = s.s;
    }
  }
}

// Any strides and lengths: a block a row, which it reads twice.
template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_long_kernel(const __grid_constant__ QuantArgs a) {
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
    for (int k = threadIdx.x; k < a.K; k += kThreads) {
      const float f[1] = {to_f(x[k * a.x.cs])};
      int q[1];
      quantize(f, s, q);
      a.q[m * a.ld + k] = (int8_t)q[0];
    }
    if (threadIdx.x == 0) a.scale[m] = s.s;
  }
}

// Images: a lane holds VP neighbouring pixels, a warp every warps-th group of 4 channels, up to R channels; the bytes go to
// their pixels' rows through shared memory, in words whose pitch is odd so that no two lanes meet in a bank.
// LONG: more channels than the warps hold, so they are read twice.
template <typename T, int VP, int R, bool LONG>
__global__ void __launch_bounds__(512) quantize_image_kernel(const __grid_constant__ QuantArgs a) {
  extern __shared__ uint32_t sh[];
  constexpr int kPixels = 32 * VP;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  const int words = (a.K + 3) / 4, pitch = words | 1;
  uint32_t* const tops = sh + kPixels * pitch;  // [2][warps][up to kPixels]
  int turn = 0;
  const int64_t tiles = (a.M + kPixels - 1) / kPixels;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, turn ^= 1) {
    const int64_t m = (tile * 32 + lane) * VP;
    Chunk<T, VP> x[R];
    const auto load = [&](int k0) {
#pragma unroll
      for (int i = 0; i < R; i++) {
        const int c = k0 + (i / 4 * warps + warp) * 4 + i % 4;
        x[i] = c < a.K && m < a.M ? load_pixels<T, VP>(a.x, m, c, a.M) : chunk_zero<T, VP>();
      }
    };
    // magnitudes of 16-bit neighbours stay in pairs
    constexpr int kTops = sizeof(T) == 2 && VP > 1 ? VP / 2 : VP;
    const auto larger = [](uint32_t p, uint32_t q) { return kTops < VP ? __vmaxu2(p, q) : max(p, q); };
    uint32_t top[kTops] = {};
    load(0);
    for (int k0 = 0; k0 < (LONG ? a.K : 1); k0 += R * warps) {
      if (LONG && k0) load(k0);
#pragma unroll
      for (int i = 0; i < R; i++)
#pragma unroll
        for (int j = 0; j < kTops; j++) {
          if constexpr (kTops < VP) top[j] = __vmaxu2(top[j], ((const uint32_t*)x[i].v)[j] & 0x7fff7fffu);
          else top[j] = max(top[j], __float_as_uint(to_f(x[i].v[j])) & 0x7fffffffu);
        }
    }
    uint32_t* const own = tops + turn * warps * 32 * kTops + lane;
#pragma unroll
    for (int j = 0; j < kTops; j++) own[(warp * kTops + j) * 32] = top[j];
    __syncthreads();
    Scale s[VP];
#pragma unroll
    for (int j = 0; j < kTops; j++) {
      for (int w = 0; w < warps; w++) top[j] = larger(top[j], own[(w * kTops + j) * 32]);
    }
#pragma unroll
    for (int j = 0; j < VP; j++) {
      if constexpr (kTops < VP) {
        const uint16_t h = (uint16_t)(j % 2 ? top[j / 2] >> 16 : top[j / 2] & 0xffffu);
        s[j] = Scale(__float_as_uint(to_f(*(const T*)&h)));
      } else {
        s[j] = Scale(top[j]);
      }
      if (warp == 0 && m + j < a.M) a.scale[m + j] = s[j].s;
    }
    if (LONG) load(0);
    for (int k0 = 0; k0 < (LONG ? a.K : 1); k0 += R * warps) {
      if (LONG && k0) load(k0);
#pragma unroll
      for (int i = 0; i < R; i += 4) {
        const int w = k0 / 4 + i / 4 * warps + warp;
        if (w < words) {
#pragma unroll
          for (int j = 0; j < VP; j++) {
            const float f[4] = {to_f(x[i].v[j]), to_f(x[i + 1].v[j]), to_f(x[i + 2].v[j]), to_f(x[i + 3].v[j])};
            int q[4];
            quantize(f, s[j], q);
            sh[(j * 32 + lane) * pitch + w] = bytes4(q[0], q[1], q[2], q[3]);
          }
        }
      }
    }
    __syncthreads();
    const int64_t first = tile * kPixels;
    // a pixel's words by as many lanes as a power of two holds
    const int count = (int)min((int64_t)kPixels, a.M - first);
    int span = 1;
    while (span < words && span < 32) span *= 2;
    for (int p = threadIdx.x / span; p < count; p += blockDim.x / span)
      for (int w = threadIdx.x % span; w < words; w += span) {
        const uint32_t v = sh[(p % VP * 32 + p / VP) * pitch + w];
        int8_t* to = a.q + (first + p) * a.ld + 4 * w;
        if (4 * w + 4 <= a.K) *(uint32_t*)to = v;
        else
          for (int i = 0; i < a.K - 4 * w; i++) to[i] = (int8_t)(v >> (8 * i));  // what lies behind the row stays
      }
  }
}

__global__ void __launch_bounds__(kThreads) pack8_kernel(View src, int64_t rows, int64_t k, int8_t* dst, int64_t ld) {
  const int8_t* p = (const int8_t*)src.p;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows * k; i += (int64_t)gridDim.x * kThreads)
    dst[i / k * ld + i % k] = p[i / k * src.rs + i % k * src.cs];
}

// ---- a few rows: quantised and multiplied by one launch ----
// At up to 8 rows the launches cost more than the product does.  Every block quantises all rows into its shared memory, and each
// of its warps makes 4 channels: lanes along the sum, 16 products an instruction quartet, one reduction a result.
constexpr int kFewRows = 8, kFewTerms = 4096, kFewColumns = 4;
struct FewArgs {
  int M, N, K, act;
  View x, res, y;
  const int8_t* w;
  int64_t ld;
  const float* w_scale;
  const void* bias;
};
template <typename T>
__device__ __forceinline__ float act_of(int act, float z) {
  constexpr bool kExact = sizeof(T) == 4;
  float2 y, d;
  switch (act) {
    case VI_ACT_RELU:
      activate<VI_ACT_RELU, kExact, false>(pair(z), y, d);
      return relu_signed_zero<T>(y).x;
    case VI_ACT_SILU: activate<VI_ACT_SILU, kExact, false>(pair(z), y, d); return y.x;
    case VI_ACT_GELU: activate<VI_ACT_GELU, kExact, false>(pair(z), y, d); return y.x;
    case VI_ACT_SIGMOID: activate<VI_ACT_SIGMOID, kExact, false>(pair(z), y, d); return y.x;
    default: return z;
  }
}
template <typename T, int ROWS>
__global__ void __launch_bounds__(kThreads) few_rows_kernel(const __grid_constant__ FewArgs a) {
  extern __shared__ __align__(16) int8_t terms_of[];  // [ROWS][terms]
  __shared__ uint32_t tops[kThreads / 32];
  __shared__ float scales[ROWS];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, terms = (a.K + 15) / 16 * 16;
  // the weights are asked for before the rows are known
  const int n0 = (blockIdx.x * (kThreads / 32) + warp) * kFewColumns;
  int4 first[kFewColumns];
  const bool ahead = lane * 16 + 16 <= a.K;
#pragma unroll
  for (int c = 0; c < kFewColumns; c++)
    if (ahead && n0 + c < a.N) first[c] = *(const int4*)(a.w + (n0 + c) * a.ld + lane * 16);
  {
    constexpr int kTeam = kThreads / ROWS;
    const int r = threadIdx.x / kTeam, t = threadIdx.x % kTeam;
    const T* x = (const T*)a.x.p + r * a.x.rs;
    uint32_t top = 0;
    if (r < a.M)
      for (int k = t; k < a.K; k += kTeam) top = max(top, __float_as_uint(to_f(x[k * a.x.cs])) & 0x7fffffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kTeam / 32; w++) top = max(top, tops[r * (kTeam / 32) + w]);
    const Scale s(top);
    if (t == 0) scales[r] = s.s;
    for (int k = t; k < terms; k += kTeam) {
      int q[1] = {0};
      if (r < a.M && k < a.K) {
        const float f[1] = {to_f(x[k * a.x.cs])};
        quantize(f, s, q);
      }
      terms_of[r * terms + k] = (int8_t)q[0];
    }
  }
  __syncthreads();
  if (n0 >= a.N) return;
  int acc[kFewColumns][ROWS] = {};
  for (int k = lane * 16; k < a.K; k += 512) {
    int4 w[kFewColumns];
#pragma unroll
    for (int c = 0; c < kFewColumns; c++) {
      w[c] = make_int4(0, 0, 0, 0);
      if (n0 + c < a.N) {
        const int8_t* p = a.w + (n0 + c) * a.ld + k;
        if (k == lane * 16 && ahead) w[c] = first[c];
        else if (k + 16 <= a.K) w[c] = *(const int4*)p;
        else
          for (int i = 0; i < a.K - k; i++) ((int8_t*)&w[c])[i] = p[i];
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
      const int4 x = *(const int4*)(terms_of + r * terms + k);
#pragma unroll
      for (int c = 0; c < kFewColumns; c++)
        acc[c][r] = __dp4a(w[c].x, x.x, __dp4a(w[c].y, x.y, __dp4a(w[c].z, x.z, __dp4a(w[c].w, x.w, acc[c][r]))));
    }
  }
  int mine = 0;  // lane c * ROWS + r keeps that result
#pragma unroll
  for (int c = 0; c < kFewColumns; c++)
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
      const int sum = __reduce_add_sync(0xffffffffu, acc[c][r]);
      if (lane == c * ROWS + r) mine = sum;
    }
  const int r = lane % ROWS, n = n0 + lane / ROWS;
  if (lane >= kFewColumns * ROWS || r >= a.M || n >= a.N) return;
  float z = (float)mine * (scales[r] * a.w_scale[n]);
  if (a.bias) z += to_f(((const T*)a.bias)[n]);
  z = act_of<T>(a.act, z);
  if (a.res.p) z += to_f(((const T*)a.res.p)[r * a.res.rs + n * a.res.cs]);
  ((T*)a.y.p)[r * a.y.rs + n * a.y.cs] = from_f<T>(z);
}
static_assert(kFewColumns * kFewRows <= 32, "a result a lane");

// ---- host ----
struct Call {
  const QuantArgs& a;
  int sms;
  cudaStream_t s;

  template <typename T, int VEC, int NV, int R, bool BLOCK>
  bool rows(int64_t units) {
    if (units > (BLOCK ? 512 : 32) * NV) return false;
    const int threads = BLOCK ? (int)ceil_div(ceil_div(units, NV), 32) * 32 : kThreads;
    const int lanes = BLOCK ? threads : NV > 1 ? 32 : pow2_at_least(units);
    const int64_t work = BLOCK ? a.M : ceil_div(a.M, (int64_t)kThreads / lanes * R);
    quantize_rows_kernel<T, VEC, NV, R, BLOCK><<<(unsigned)std::min<int64_t>(work, (int64_t)sms * 16), threads, 0, s>>>(a, lanes);
    return true;
  }
  template <typename T, int VP, int R, bool LONG>
  bool image() {
    const int warps = (int)std::min<int64_t>(16, ceil_div(ceil_div(a.K, 4), R / 4));
    const size_t smem = (size_t)32 * VP * ((ceil_div(a.K, 4) | 1) + 2 * warps) * 4;
    constexpr int kMost = 200 * 1024;
    if (smem > kMost) return false;
    auto* kernel = quantize_image_kernel<T, VP, R, LONG>;
    // the most that any call asks for, as another thread's call may need more than this one
    if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost) != cudaSuccess) {
      cudaGetLastError();
      return false;
    }
    const int per_sm = (int)std::max<int64_t>(1, std::min<int64_t>(16 / warps * 2, (int64_t)(220 * 1024 / (smem + 1024))));
    kernel<<<(unsigned)std::min<int64_t>(ceil_div(a.M, 32 * VP), (int64_t)sms * per_sm), warps * 32, smem, s>>>(a);
    return true;
  }
  template <typename T>
  void run() {
    constexpr int VEC = 16 / (int)sizeof(T), VP = 4 / (int)sizeof(T);
    const int64_t K = a.K;
    const bool words = a.ld % 8 == 0 && (uintptr_t)a.q % 8 == 0;  // as this library lays rows out
    if (a.x.rs == 1 && a.x.cs != 1 && a.M > 1 && a.ld % 4 == 0 && (uintptr_t)a.q % 4 == 0) {
      if (K <= 128 && moves<T>(a.x, VEC, true)) {
        if (image<T, VEC, 8, false>()) return;
      } else if (K <= 512) {
        if (moves<T>(a.x, VP, true) ? image<T, VP, 32, false>() : image<T, 1, 32, false>()) return;
      } else if (moves<T>(a.x, VP, true) ? image<T, VP, 32, true>() : image<T, 1, 32, true>()) {
        return;
      }
    } else if (words && K % VEC == 0 && moves<T>(a.x, VEC, false)) {
      const int64_t n = K / VEC;
      if (rows<T, VEC, 1, 4, false>(n) || rows<T, VEC, 2, 2, false>(n) || rows<T, VEC, 4, 1, false>(n) || rows<T, VEC, 4, 1, true>(n)) return;
    } else if (a.x.cs == 1 || a.x.rs != 1) {
      if (rows<T, 1, 1, 4, false>(K) || rows<T, 1, 4, 1, false>(K) || rows<T, 1, 16, 1, false>(K) || rows<T, 1, 16, 1, true>(K)) return;
    }
    quantize_long_kernel<T><<<(unsigned)std::min<int64_t>(a.M, (int64_t)sms * 8), kThreads, 0, s>>>(a);
  }
};

}  // namespace

cudaError_t launch_quantize(int dtype, const QuantArgs& a, int sms, cudaStream_t s) {
  Call c{a, sms, s};
  if (dtype == VI_F32) c.run<float>();
  else if (dtype == VI_F16) c.run<__half>();
  else c.run<__nv_bfloat16>();
  return cudaPeekAtLastError();
}
bool int8_few(int64_t M, int64_t K) { return M <= kFewRows && K <= kFewTerms; }
cudaError_t launch_int8_few(int dtype, int64_t M, const View& x, const Operand& w, const Epilogue& e, cudaStream_t s) {
  FewArgs a{(int)M, (int)w.rows, (int)w.k, e.act, x, e.res, e.out, (const int8_t*)w.p, w.ld, e.col_scale, e.bias};
  const unsigned blocks = (unsigned)ceil_div(w.rows, kThreads / 32 * kFewColumns);
  const auto run = [&](auto rows) {
    constexpr int ROWS = decltype(rows)::value;
    const size_t smem = (size_t)ROWS * ceil_div(w.k, 16) * 16;
    if (dtype == VI_F32) few_rows_kernel<float, ROWS><<<blocks, kThreads, smem, s>>>(a);
    else if (dtype == VI_F16) few_rows_kernel<__half, ROWS><<<blocks, kThreads, smem, s>>>(a);
    else few_rows_kernel<__nv_bfloat16, ROWS><<<blocks, kThreads, smem, s>>>(a);
  };
  if (M == 1) run(std::integral_constant<int, 1>());
  else if (M == 2) run(std::integral_constant<int, 2>());
  else if (M <= 4) run(std::integral_constant<int, 4>());
  else run(std::integral_constant<int, 8>());
  return cudaPeekAtLastError();
}
cudaError_t launch_pack8(const View& src, int64_t rows, int64_t k, int8_t* dst, int64_t ld, cudaStream_t s) {
  const unsigned blocks = (unsigned)std::min<int64_t>((rows * k + kThreads - 1) / kThreads, 148 * 16);
  pack8_kernel<<<blocks, kThreads, 0, s>>>(src, rows, k, dst, ld);
  return cudaPeekAtLastError();
}

}  // namespace heads
}  // namespace vi
