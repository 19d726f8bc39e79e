// The heads' matrix products of float operands: the kernels of vi_heads_gemm.cuh for each type, tile and epilogue.
#include "vi_heads_gemm.cuh"

namespace vi {
namespace heads {
namespace {

__device__ uint32_t g_status;  // VI_DEVICE_HEAD_TIMEOUT when a wait ran out
std::atomic<uint64_t> g_pair_launches{0};

template <typename T, int EPI, int PL, int ACT = VI_ACT_NONE>
cudaError_t run_bn(int bn, const CUtensorMap& ma, const CUtensorMap& mb, const Args& a, int sms, cudaStream_t s) {
  constexpr bool kOwn = own_chain_kernel(EPI);
  if constexpr (kOwn)
    if (a.chain) return run<T, 128, EPI, PL, ACT, true>(ma, mb, a, sms, s);
  if constexpr (PL == 1)
    if (bn == 256) return run<T, 256, EPI, PL, ACT, !kOwn>(ma, mb, a, sms, s);
  return bn == 64 ? run<T, 64, EPI, PL, ACT, !kOwn>(ma, mb, a, sms, s) : run<T, 128, EPI, PL, ACT, !kOwn>(ma, mb, a, sms, s);
}
template <typename T>
cudaError_t run_epi(int epi, int bn, const CUtensorMap& ma, const CUtensorMap& mb, const Args& a, int sms,
                    cudaStream_t s) {
  constexpr int PL = sizeof(T) == 4 ? 3 : 1;
  switch (epi) {
    case kEpiAct:
      switch (a.e.act) {
        case VI_ACT_RELU: return run_bn<T, kEpiAct, PL, VI_ACT_RELU>(bn, ma, mb, a, sms, s);
        case VI_ACT_SILU: return run_bn<T, kEpiAct, PL, VI_ACT_SILU>(bn, ma, mb, a, sms, s);
        case VI_ACT_GELU: return run_bn<T, kEpiAct, PL, VI_ACT_GELU>(bn, ma, mb, a, sms, s);
        case VI_ACT_SIGMOID: return run_bn<T, kEpiAct, PL, VI_ACT_SIGMOID>(bn, ma, mb, a, sms, s);
        default: return run_bn<T, kEpiAct, PL>(bn, ma, mb, a, sms, s);
      }
    case kEpiStore: return run_bn<T, kEpiStore, PL>(bn, ma, mb, a, sms, s);
    case kEpiPartial: return run_bn<float, kEpiPartial, PL>(bn, ma, mb, a, sms, s);
    case kEpiLse: return run_bn<T, kEpiLse, PL>(bn, ma, mb, a, sms, s);
    default: return run_bn<T, kEpiGrad, PL>(bn, ma, mb, a, sms, s);
  }
}

}  // namespace

uint32_t* status_word() {
  static std::atomic<uint32_t*> known[64];  // by device
  int dev = 0;
  cudaGetDevice(&dev);
  uint32_t* w = known[dev & 63].load(std::memory_order_relaxed);
  if (w && dev < 64) return w;
  void* p = nullptr;
  if (cudaGetSymbolAddress(&p, g_status) != cudaSuccess) return nullptr;
  if (dev < 64) known[dev].store((uint32_t*)p, std::memory_order_relaxed);
  return (uint32_t*)p;
}
void note_pair_launch() { g_pair_launches.fetch_add(1, std::memory_order_relaxed); }

int lse_parts(int bn) { return Shape<__half, 64, kEpiLse, 1>::kParts * (bn == 256 ? 2 : 1); }
static_assert(Shape<__half, 256, kEpiLse, 1>::kParts == 2 * Shape<__half, 64, kEpiLse, 1>::kParts &&
              Shape<float, 128, kEpiLse, 3>::kParts == Shape<__half, 64, kEpiLse, 1>::kParts, "lse_parts");

int launch_gemm(int dtype, int epi, const Operand& A, const Operand& B, const Plan& p, const Epilogue& e, int sms,
                cudaStream_t s) {
  const int planes = dtype == VI_F32 ? 3 : 1;
  const bool half = dtype == VI_F16;
  const bool pair = pair_tile(epi, p.bn);
  if (long_chain_kernel(dtype, epi, p.kps) && p.bn != 128) return set_error(VI_ERR_UNSUPPORTED, "heads: a long sum's tiles are 128 wide");
  CUtensorMap ma, mb;
  if (!encode(&ma, A, planes, dtype, kBM) || !encode(&mb, B, planes, dtype, pair ? 128 : p.bn))
    return set_error(VI_ERR_CUDA, "heads: a tensor map could not be encoded");
  Args a;
  if (int rc = fill_args(a, A, B, p, epi, half ? 0 : 1)) return rc;
  if (const int most = chain_blocks(dtype, epi); p.kps > most) {
    const int chains = (p.kps + most - 1) / most;
    a.chain = (p.kps + chains - 1) / chains;
  }
  a.e = e;
  cudaError_t rc;
  if (dtype == VI_F32)
    rc = run_epi<float>(epi, p.bn, ma, mb, a, sms, s);
  else if (dtype == VI_F16)
    rc = run_epi<__half>(epi, p.bn, ma, mb, a, sms, s);
  else
    rc = run_epi<__nv_bfloat16>(epi, p.bn, ma, mb, a, sms, s);
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

extern "C" uint64_t vi_heads_pair_launches(void) { return vi::heads::g_pair_launches.load(); }

extern "C" int vi_heads_status(uint32_t* status, int reset, void* stream) {
  using namespace vi;
  const cudaStream_t s = (cudaStream_t)stream;
  void* p = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&p, heads::g_status);
  if (e == cudaSuccess) e = cudaMemcpyAsync(status, p, 4, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess && reset) e = cudaMemsetAsync(p, 0, 4, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e == cudaSuccess) return VI_OK;
  char msg[256];
  snprintf(msg, sizeof msg, "vi_heads_status: %s", cudaGetErrorString(e));
  return set_error(VI_ERR_CUDA, msg);
}
