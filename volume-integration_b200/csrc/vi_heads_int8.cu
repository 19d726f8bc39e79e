// The dense layer in 8-bit integers: vi_heads_gemm.cuh's product with kEpiInt8.
//
// Mathematics.  x_mk is about s_m q_mk and w_nk about t_n p_nk with whole q and p in [-127, 127]; the sum over k of
// q p is exact in 32 bits (up to 2^17 terms), and y = act(s_m t_n sum + b_n) + res is rounded once to the type.
#include "vi_heads_gemm.cuh"

namespace vi {
namespace heads {
namespace {

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
