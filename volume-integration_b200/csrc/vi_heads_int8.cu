// The dense layer in 8-bit integers: vi_heads_gemm.cuh's product with kEpiInt8.
//
// Mathematics.  x_mk is about s_m q_mk and w_nk about t_n p_nk with whole q and p in [-127, 127]; the sum over k of
// q p is exact in 32 bits (under 2^17 terms), and y = act(s_m t_n sum + b_n) + res is rounded once to the type.
// 32768 x 1024 -> 4096 with relu, x quantised before: 156 us at 1965 MHz, 1.8 * 10^15 operations a second; the float16 layer 229.
#include "vi_heads_gemm.cuh"
#include "vi_quant.cuh"

namespace vi {
namespace heads {
namespace {

// ---- few features: quantised on the way into the product ----
// Up to 64 features and 64 channels of 16-bit types are bound by memory and by the epilogue, and a pass that quantises would
// write and read the features once more (2M x 64 -> 64 with gelu and a residual: 284 us + 235 apart).  Here one warp copies 256
// rows of x at a time into shared memory, eight find their scales and write the tensor core's operand, two products of 128 rows
// follow, and 16 warps run the epilogue: 317 us in all, the latency of 26 warps at 72 registers.
constexpr int kFusedK = 64, kFusedN = 64;
template <typename T>
struct Fused {
  static constexpr int kEpi = 16, kMake = 8, kThreads = (kEpi + kMake + 2) * 32, kRows = 256;
  static constexpr int kStage = kRows * 128, kStages = 2, kScales = 4;
  static constexpr int kX = kStages * kStage, kXBytes = kRows * kFusedK * 2, kXStages = 3;
  static constexpr int kB = kX + kXStages * kXBytes, kStaging = kB + kFusedN * 128;
  static constexpr int kWarpBytes = 32 * 32 * (int)sizeof(T) + 256;
  static constexpr int kScale = kStaging + kEpi * kWarpBytes, kBars = kScale + kScales * kRows * 4;
  static constexpr int kSmem = kBars + 28 * 8;
  static_assert(kSmem <= 227 * 1024, "shared memory of a block");
};
struct FusedArgs {
  int64_t M;
  int K, N, image;
  uint32_t idesc;
  int64_t wait_limit;  // cycles
  int withhold;        // testing hooks: the first load is never issued;
  int lapse;           // one lane's wait counts as run out
  uint32_t* status;
  Epilogue e;
};

// 16 bytes c of row r of a 128-byte swizzled operand.
__device__ __forceinline__ uint32_t swizzled(uint32_t base, int r, int c) { return base + r * 128 + ((c ^ (r & 7)) << 4); }

template <typename T, int ACT>
__global__ void __launch_bounds__(Fused<T>::kThreads, 1) int8_fused_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ FusedArgs a) {
  using S = Fused<T>;
  extern __shared__ __align__(1024) char smem[];
  uint64_t* bars = (uint64_t*)(smem + S::kBars);
  uint32_t* tmem_slot = (uint32_t*)(bars + 24);
  volatile int* dead = (int*)(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t afull = smem_u32(bars), aempty = afull + 16, tfull = afull + 32, tempty = afull + 48, sfull = afull + 64, bfull = afull + 96,
                 drain = afull + 104, xfull = afull + 112, xempty = xfull + 8 * S::kXStages;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kXStages; i++) {
      mbar_init(xfull + 8 * i, 1);
      mbar_init(xempty + 8 * i, S::kMake);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(afull + 8 * i, S::kMake);
      mbar_init(aempty + 8 * i, 1);
      mbar_init(tfull + 8 * i, 1);
      mbar_init(tempty + 8 * i, S::kEpi);
    }
    for (int i = 0; i < S::kScales; i++) mbar_init(sfull + 8 * i, S::kMake);
    mbar_init(bfull, 1);
    mbar_init(drain, 1);
    *dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  constexpr uint32_t kCols = 256;  // two accumulators of two products of 64 columns
  if (warp == S::kEpi + S::kMake) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  const int64_t tiles = (a.M + S::kRows - 1) / S::kRows;
  float* const scales = (float*)(smem + S::kScale);

  if (warp >= S::kEpi && warp < S::kEpi + S::kMake) {
    // ---- quantise: 32 rows a warp ----
    const int first = (warp - S::kEpi) * (S::kRows / S::kMake);
    int i = 0, xs = 0;
    uint32_t xphase = 0;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x, i++) {
      const uint32_t base = smem_u32(smem) + (i & 1) * S::kStage, x = smem_u32(smem + S::kX) + xs * S::kXBytes;
      // the last product that read this stage has ended, and with it the epilogue of four tiles ago
      bool on = mbar_wait(xfull + 8 * xs, xphase, dead, a.wait_limit) && mbar_wait(aempty + 8 * (i & 1), (i / 2 & 1) ^ 1, dead, a.wait_limit);
      if (a.lapse && lane == 5) on = false, *dead = 1;
      if (!__all_sync(0xffffffffu, on)) break;  // the lanes leave together: what follows exchanges between them
      if (a.image) {  // a lane: two neighbouring pixels, half of the channels
        const int pair_row = first + lane % 16 * 2, k0 = lane / 16 * (kFusedK / 2);
        const uint32_t own = x + pair_row * 2 + k0 * (S::kRows * 2);
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < kFusedK / 2; k++) top = __vmaxu2(top, lds_cell(own + k * (S::kRows * 2), 0u) & 0x7fff7fffu);
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 16));
        Scale s[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const uint16_t h = (uint16_t)(j ? top >> 16 : top & 0xffffu);
          s[j] = Scale(__float_as_uint(to_f(*(const T*)&h)));
          if (lane < 16) scales[(i & 3) * S::kRows + pair_row + j] = s[j].s;
        }
#pragma unroll
        for (int c = 0; c < kFusedK / 32; c++) {
          uint32_t w[2][4];
#pragma unroll
          for (int g = 0; g < 4; g++) {
            float f[2][4];
#pragma unroll
            for (int b = 0; b < 4; b++) {
              const float2 v = unpack2(lds_cell(own + (c * 16 + g * 4 + b) * (S::kRows * 2), 0u), T());
              f[0][b] = v.x, f[1][b] = v.y;
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
              int q[4];
              quantize(f[j], s[j], q);
              w[j][g] = bytes4(q[0], q[1], q[2], q[3]);
            }
          }
#pragma unroll
          for (int j = 0; j < 2; j++) sts128(swizzled(base, pair_row + j, k0 / 16 + c), make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]));
        }
      } else {  // 8 lanes a row, 8 features each
#pragma unroll
        for (int n = 0; n < S::kRows / S::kMake / 4; n++) {
          const int r = first + n * 4 + lane / 8;
          const uint4 u = lds128(x + r * (kFusedK * 2) + lane % 8 * 16);
          uint32_t top = __vmaxu2(__vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu), __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
#pragma unroll
          for (int o = 4; o; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
          const uint16_t h = (uint16_t)max(top & 0xffffu, top >> 16);
          const Scale s(__float_as_uint(to_f(*(const T*)&h)));
          const float2 v0 = unpack2(u.x, T()), v1 = unpack2(u.y, T()), v2 = unpack2(u.z, T()), v3 = unpack2(u.w, T());
          const float f[8] = {v0.x, v0.y, v1.x, v1.y, v2.x, v2.y, v3.x, v3.y};
          int q[8];
          quantize(f, s, q);
          const uint32_t to = swizzled(base, r, lane % 8 / 2) + lane % 2 * 8;
          asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(bytes4(q[0], q[1], q[2], q[3])), "r"(bytes4(q[4], q[5], q[6], q[7])) : "memory");
          if (lane % 8 == 0) scales[(i & 3) * S::kRows + r] = s.s;
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(xempty + 8 * xs);
        mbar_arrive(afull + 8 * (i & 1));
        mbar_arrive(sfull + 8 * (i & 3));
      }
      if (++xs == S::kXStages) xs = 0, xphase ^= 1;
    }
  } else if (warp == S::kEpi + S::kMake + 1) {
    // ---- loads ----
    if (lane == 0) {
      int64_t n = 0;
      for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x, n++) {
        const int xs = (int)(n % S::kXStages);
        if (!mbar_wait(xempty + 8 * xs, (uint32_t)(n / S::kXStages & 1) ^ 1, dead, a.wait_limit)) break;
        if (a.withhold && n == 0) continue;  // this stage is never filled: its readers' wait runs out
        mbar_expect(xfull + 8 * xs, S::kXBytes);
        const uint32_t to = smem_u32(smem + S::kX) + xs * S::kXBytes;
        if (a.image) tma_load<false>(to, &map_x, xfull + 8 * xs, (int)(t * S::kRows), 0, 0);
        else tma_load<false>(to, &map_x, xfull + 8 * xs, 0, (int)(t * S::kRows), 0);
      }
      // the copies in flight end before the block does: the last fill of every stage
      for (int64_t f = n - 1; f >= a.withhold && f >= n - S::kXStages; f--)
        mbar_drain(xfull + 8 * (uint32_t)(f % S::kXStages), (uint32_t)(f / S::kXStages) & 1, a.wait_limit);
    }
  } else if (warp == S::kEpi + S::kMake) {
    // ---- products ----
    if (lane == 0) {
      mbar_expect(bfull, kFusedN * 128);
      tma_load<false>(smem_u32(smem + S::kB), &map_b, bfull, 0, 0, 0);
      bool on = mbar_wait(bfull, 0, dead, a.wait_limit);
      if (!on) mbar_drain(bfull, 0, a.wait_limit);
      const uint64_t db = smem_desc(smem_u32(smem + S::kB), 1);
      const int steps = (a.K + 31) / 32;
      int i = 0;
      for (int64_t t = blockIdx.x; t < tiles && on; t += gridDim.x, i++) {
        on = mbar_wait(tempty + 8 * (i & 1), (i / 2 & 1) ^ 1, dead, a.wait_limit) && mbar_wait(afull + 8 * (i & 1), i / 2 & 1, dead, a.wait_limit);
        if (!on) break;
        fence_after();
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint64_t da = smem_desc(smem_u32(smem) + (i & 1) * S::kStage + h * (S::kStage / 2), 1);
          for (int k = 0; k < steps; k++) mma_i8<false>(tmem + (i & 1) * 128 + h * 64, da + 2 * k, db + 2 * k, a.idesc, k > 0);
        }
        mma_commit<false>(aempty + 8 * (i & 1));
        mma_commit<false>(tfull + 8 * (i & 1));
      }
      // the arrivals that the products still owe come before the block leaves
      for (int j = i - 2; j < i && on; j++)
        if (j >= 0) on = mbar_wait(aempty + 8 * (j & 1), j / 2 & 1, dead, a.wait_limit);
      if (*dead) {
        mma_commit<false>(drain);
        mbar_drain(drain, 0, a.wait_limit);
      }
    }
  } else {
    // ---- epilogue: a warp 32 columns of 32 rows of each product ----
    const int quad = warp % 4, c = warp / 4 % 2 * 32;
    const uint32_t st = smem_u32(smem + S::kStaging) + warp * S::kWarpBytes, bias_slot = st + 32 * 32 * (int)sizeof(T);
    const Epilogue& e = a.e;
    const int out_access = access_of<T>(e.out), res_access = access_of<T>(e.res);
    if (c < a.N) {
      const bool in = c + lane < a.N;
      sts_cell(bias_slot + lane * 4, __float_as_uint(in && e.bias ? to_f(((const T*)e.bias)[c + lane]) : 0.0f));
      sts_cell(bias_slot + 128 + lane * 4, __float_as_uint(in ? e.col_scale[c + lane] : 0.0f));
    }
    __syncwarp();
    int i = 0;
    bool on = true;
    for (int64_t t = blockIdx.x; t < tiles && on; t += gridDim.x, i++) {
      const int half = warp / 8, row = half * 128 + quad * 32;
      const int64_t m0 = t * S::kRows + row;
      const bool some = m0 < a.M && c < a.N;
      const Place here{(int)m0, c, (int)min((int64_t)32, a.M - m0), min(32, a.N - c)};
      Row<T> extra, y;
      int way = kNone;
      if (some && e.res.p) way = load_tile<T>(extra, e.res, res_access, st, lane, here);  // asked for before the product is waited for
      on = mbar_wait(sfull + 8 * (i & 3), i / 4 & 1, dead, a.wait_limit) && mbar_wait(tfull + 8 * (i & 1), i / 2 & 1, dead, a.wait_limit);
      on = __all_sync(0xffffffffu, on);
      if (!on) break;
      fence_after();
      if (some) {
        const float row_scale = scales[(i & 3) * S::kRows + row + lane];
        const uint32_t src = tmem + ((uint32_t)(quad * 32) << 16) + (i & 1) * 128 + half * 64 + c;
        if (e.res.p) own_row<T>(extra, way, st, lane);
#pragma unroll
        for (int h = 0; h < 2; h++) {
          float2 v[8];
          tmem_load16(src + h * 16, (float*)v);
          tmem_wait_load();
          scale_sums(bias_slot + 128 + h * 64, row_scale, v);
          if (e.bias) add_bias<16>(bias_slot + h * 64, v);
#pragma unroll
          for (int j = 0; j < 8; j++) {
            float2 w, d;
            activate<ACT, false, false>(v[j], w, d);
            v[j] = ACT == VI_ACT_RELU ? relu_signed_zero<T>(w) : w;
            if (e.res.p) v[j] = __fadd2_rn(v[j], get_pair(extra, h * 8 + j));
            set_pair(y, h * 8 + j, v[j]);
          }
#pragma unroll
          for (int j = 0; j < 8; j++) asm volatile("" : "+r"(y.w[h * 8 + j]));
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty + 8 * (i & 1));
      if (some) store_tile(y, e.out, out_access, st, lane, here);
    }
  }
  __syncwarp();
  __syncthreads();
  if (warp == S::kEpi + S::kMake)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
  if (threadIdx.x == 0 && *dead) atomicOr(a.status, VI_DEVICE_HEAD_TIMEOUT);
}

template <typename T, int ACT>
cudaError_t run_fused(const CUtensorMap& mx, const CUtensorMap& mb, const FusedArgs& a, int sms, cudaStream_t s) {
  using S = Fused<T>;
  auto* k = int8_fused_kernel<T, ACT>;
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (dev >= 64 || !(done.load(std::memory_order_relaxed) & bit)) {
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  }
  k<<<(unsigned)std::min<int64_t>((a.M + S::kRows - 1) / S::kRows, sms), S::kThreads, S::kSmem, s>>>(mx, mb, a);
  return cudaPeekAtLastError();
}
template <typename T>
cudaError_t run_fused_act(const CUtensorMap& mx, const CUtensorMap& mb, const FusedArgs& a, int sms, cudaStream_t s) {
  switch (a.e.act) {
    case VI_ACT_RELU: return run_fused<T, VI_ACT_RELU>(mx, mb, a, sms, s);
    case VI_ACT_SILU: return run_fused<T, VI_ACT_SILU>(mx, mb, a, sms, s);
    case VI_ACT_GELU: return run_fused<T, VI_ACT_GELU>(mx, mb, a, sms, s);
    case VI_ACT_SIGMOID: return run_fused<T, VI_ACT_SIGMOID>(mx, mb, a, sms, s);
    default: return run_fused<T, VI_ACT_NONE>(mx, mb, a, sms, s);
  }
}

template <typename T, int ACT>
cudaError_t run_width(int bn, const CUtensorMap& ma, const CUtensorMap& mb, const Args& a, int sms, cudaStream_t s) {
  return bn == 256  ? run<T, 256, kEpiInt8, 1, ACT, false>(ma, mb, a, sms, s)
         : bn == 64 ? run<T, 64, kEpiInt8, 1, ACT, false>(ma, mb, a, sms, s)
                    : run<T, 128, kEpiInt8, 1, ACT, false>(ma, mb, a, sms, s);
}
template <typename T>
cudaError_t run_act(int bn, const CUtensorMap& ma, const CUtensorMap& mb, const Args& a, int sms, cudaStream_t s) {
  switch (a.e.act) {
    case VI_ACT_RELU: return run_width<T, VI_ACT_RELU>(bn, ma, mb, a, sms, s);
    case VI_ACT_SILU: return run_width<T, VI_ACT_SILU>(bn, ma, mb, a, sms, s);
    case VI_ACT_GELU: return run_width<T, VI_ACT_GELU>(bn, ma, mb, a, sms, s);
    case VI_ACT_SIGMOID: return run_width<T, VI_ACT_SIGMOID>(bn, ma, mb, a, sms, s);
    default: return run_width<T, VI_ACT_NONE>(bn, ma, mb, a, sms, s);
  }
}

}  // namespace

// Few features and channels of 16-bit types, and rows enough that their bytes count, where bulk copies reach them.  bfloat16
// 64 -> 64 with gelu and a residual, image (rows): 524288 pixels 92 us (88) here, 150 (102) apart; 32768 16 (16), 27 (19); below, this
// kernel would save up to 8 us of a call that is launches mostly: 8192 pixels 14 (14), 23 (16).
bool int8_fused(int dtype, int64_t M, int64_t N, int64_t K, const View& x) {
  if (dtype == VI_F32 || K > kFusedK || N > kFusedN || M < 32768) return false;
  if ((uintptr_t)x.p % 16) return false;
  if (x.rs == 1 && x.cs != 1) return x.cs % 8 == 0 && x.cs >= M && x.cs < (1ll << 38);
  return x.cs == 1 && x.rs % 8 == 0 && x.rs >= K && x.rs < (1ll << 38);
}
int launch_int8_fused(int dtype, int64_t M, const View& x, const Operand& B, const Epilogue& e, int sms, cudaStream_t s) {
  CUtensorMap mx, mb;
  const EncodeFn fn = encode_fn();
  const bool image = x.rs == 1 && x.cs != 1;
  const cuuint64_t dims[3] = {(cuuint64_t)(image ? M : B.k), (cuuint64_t)(image ? B.k : M), 1}, stride = (cuuint64_t)(image ? x.cs : x.rs) * 2;
  const cuuint64_t strides[2] = {stride, stride};
  const cuuint32_t box[3] = {(cuuint32_t)(image ? Fused<__half>::kRows : kFusedK), (cuuint32_t)(image ? kFusedK : Fused<__half>::kRows), 1}, unit[3] = {1, 1, 1};
  if (!fn || !encode(&mb, B, 1, kInt8, kFusedN) ||
      fn(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, x.p, dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return set_error(VI_ERR_CUDA, "heads: a tensor map could not be encoded");
  FusedArgs a{};
  a.M = M;
  a.K = (int)B.k;
  a.N = (int)B.rows;
  a.image = image;
  a.idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kFusedN >> 3) << 17) | ((128u >> 4) << 24);
  const char* test = getenv("VI_HEADS_TEST_TIMEOUT");
  a.withhold = test && test[0] == '1';
  a.lapse = test && test[0] == '2';
  a.wait_limit = a.withhold || a.lapse ? 1 << 20 : kWaitLimit;
  a.status = status_word();
  a.e = e;
  if (!a.status) return set_error(VI_ERR_CUDA, "heads: the status word has no address");
  const cudaError_t rc = dtype == VI_F16 ? run_fused_act<__half>(mx, mb, a, sms, s) : run_fused_act<__nv_bfloat16>(mx, mb, a, sms, s);
  if (rc != cudaSuccess) return set_error(VI_ERR_CUDA, cudaGetErrorString(rc));
  note_launches(1);
  return VI_OK;
}

int launch_int8_gemm(int dtype, const Operand& A, const Operand& B, const Plan& p, const Epilogue& e, int sms, cudaStream_t s) {
  const bool pair = pair_tile(kEpiInt8, p.bn);
  CUtensorMap ma, mb;
  if (!encode(&ma, A, 1, kInt8, kBM) || !encode(&mb, B, 1, kInt8, pair ? 128 : p.bn))
    return set_error(VI_ERR_CUDA, "heads: a tensor map could not be encoded");
  Args a;
  if (int rc = fill_args(a, A, B, p, kEpiInt8, 1)) return rc;
  a.e = e;
  const cudaError_t rc = dtype == VI_F32   ? run_act<float>(p.bn, ma, mb, a, sms, s)
                         : dtype == VI_F16 ? run_act<__half>(p.bn, ma, mb, a, sms, s)
                                           : run_act<__nv_bfloat16>(p.bn, ma, mb, a, sms, s);
  if (rc != cudaSuccess) {
    char msg[256];
    snprintf(msg, sizeof msg, "heads: %s", cudaGetErrorString(rc));
    return set_error(VI_ERR_CUDA, msg);
  }
  note_launches(1);
  if (pair) note_pair_launch();
  return VI_OK;
}

}  // namespace heads
}  // namespace vi
