// Internal declarations of the per-pixel heads: operand views, the epilogues of
// their matrix product, and its launcher.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/volume_integration_b200.h"

namespace vi {
namespace heads {

// Element (r, c) at p + r * rs + c * cs (strides in elements).
struct View {
  void* p;
  int64_t rs, cs;
};

// One operand of the product as the tensor cores read it: 16-bit elements, [rows][k]
// with either axis contiguous, 16-byte aligned, in one plane or in three whose sum it
// is (float32, see split3).
struct Operand {
  const void* p;
  int64_t rows, k;       // extents
  int64_t ld;            // elements from one row (k_major) or one k (else) to the next
  int64_t plane;         // elements from one plane to the next
  bool k_major;          // k is the contiguous axis
};

enum Epi {
  kEpiAct,      // out = act(acc + bias) + res, dact = act'
  kEpiStore,    // out = alpha * acc
  kEpiPartial,  // part[split] = acc, or += acc (float32)
  kEpiLse,      // per row the maximum and the sum of exponentials of the logits, the target's logit
  kEpiGrad,     // G = coef * (softmax - onehot)
  kEpiCount
};

// Whether a tile is 256 rows high and made by a pair of blocks.  The softmax's are not: its epilogue
// is the longer part, and two blocks that wait for each other's lose (K = 512: statistics 904 us
// apart, 974 in pairs; gradient 1027, 1095; the plain products 974, 921).
#ifdef __CUDACC__
__host__ __device__
#endif
constexpr bool pair_tile(int epi, int bn) { return bn == 256 && epi != kEpiLse && epi != kEpiGrad; }

// Blocks of k (64 terms each) that one accumulation may take.  The tensor core cuts what it adds, always towards
// zero, so a sum of terms of one sign drifts with its length: by about 0.8 * 2^-23 of it for every 16 terms (a float16 weight
// gradient over 262144 rows: 1.5e-3, three half steps).  Longer sums are made in accumulations that the epilogue
// adds up, rounded: 768 terms in float32; 4096 in logits of 16-bit features, whose loss is float32 (5e-6 of a
// logit); else as many as stay within a fifth of the type's half step.
constexpr int chain_blocks(int dtype, int epi) {
  if (dtype == VI_F32) return 12;
  return epi == kEpiLse || epi == kEpiGrad ? 64 : dtype == VI_F16 ? 256 : 2048;
}

// Whether a product's accumulations are added up by a kernel of its own, with 128-wide tiles: the epilogues that have no
// registers to spare for that code (with it in the common one: 2M x 64 -> 64 with gelu 222 us, 240; float32 logits of
// 4096 x 256, V = 8192: 113, 127).
constexpr bool own_chain_kernel(int epi) { return epi != kEpiStore && epi != kEpiPartial; }
constexpr bool long_chain_kernel(int dtype, int epi, int64_t kblocks) {
  return own_chain_kernel(epi) && kblocks > chain_blocks(dtype, epi);
}

// What happens to the product acc(m, n) = sum_k A(m, k) B(n, k).
struct Epilogue {
  int act;              // kEpiAct: vi_activation
  const void* bias;     // kEpiAct, kEpiLse, kEpiGrad: [N] or null
  int bias_rows;        // kEpiAct: bias is [M], one value per row
  View res;             // kEpiAct: residual, p null = none
  View out;             // kEpiAct, kEpiStore: T, one stride 1
  void* dact;           // kEpiAct: act'(z) in out's strides (float32, or 16 bits: pack_slope), null = not wanted
  const float* alpha;   // kEpiStore: device scalar the product is multiplied with, null = 1
  float* part;          // kEpiPartial: [splits][M][N]
  int add;              // kEpiPartial: add to what part holds
  // kEpiLse: [parts][M] the largest logit and the sum of exp(z - largest), [M] the target's logit
  float* pmax;
  float* psum;
  float* ztarget;
  const int64_t* target;
  // kEpiGrad: columns [col0, col0 + N) of the vocabulary
  const float* lse;     // [3][M]: the largest logit, log2 of the sum of exp(z - largest), the target's logit
  const float* coef;    // per row
  int64_t col0;
  void* grad;           // [planes][M][grad_ld], 16-bit
  int64_t grad_ld, grad_plane;
  float* column_part;   // 16-bit types: [4 per tile of 128 rows][N] sums of G's columns over 32 rows, of the cells as
                        // rounded, which dx and dweight use too; null = not wanted
};

// Tile shape and division of one product's work.
struct Plan {
  int bn;          // columns of a tile: 64, 128, or 256 (16-bit types only)
  int splits;      // pieces of the sum over k (kEpiPartial)
  int kps;         // 64-wide blocks of k per piece
  int span;        // column tiles one work item takes in turn (kEpiLse)
  int spans;       // work items per row of tiles (kEpiLse); partial results per row: lse_parts(bn) each
};

// Partial results of kEpiLse per span.
int lse_parts(int bn);

// dtype: of outputs, bias and residual.  Planes: 1, or 3 for float32.
// Returns a vi_status.
int launch_gemm(int dtype, int epi, const Operand& a, const Operand& b, const Plan& p, const Epilogue& e, int sms,
                cudaStream_t s);

// linear_act on images (rows contiguous) of at most kNarrowK channels, on the FP32 cores.
constexpr int kNarrowK = 8, kNarrowN = 256;
struct NarrowArgs {
  int64_t M;
  int N, K, act;
  View x, w;
  const void* bias;
  View y;        // the result; in the backward the incoming gradient
  View res, dx;  // p null = none
  float* part;   // backward: [blocks][N][narrow_sums(K)], the sums of s x[k], then zeros up to the last, of s
  bool vec;      // set by the launcher
  int span;      // set by the launcher: channels a block takes
};
bool narrow_forward(int64_t N, int64_t K, const View& x, const View& y, const View& res);
bool narrow_backward(int64_t N, int64_t K, const View& x, const View& dy, const View& dx);
int narrow_sums(int64_t K);
int narrow_blocks(int64_t M, int sms);  // of the backward
cudaError_t launch_narrow(int dtype, const NarrowArgs& a, bool backward, int blocks, int sms, cudaStream_t s);

// out(m, n) = f(sum_k A(m, k) B(n, k)) on the FP32 cores, for small products.
struct SmallJob {
  View a, slope;       // A = a * slope (p null: a)
  View b;
  const float* skip;   // B(n, k) counts as 0 where skip[k] is 0; null = nowhere
  int M, N, K;
  View out;            // p null: only the sums are wanted
  const float* alpha;  // device factor, null = 1
  void* sums;          // [M] alpha * sum_k A(m, k), null = not wanted
  // forward: act(. + bias) + res, act' to dact (in out's strides)
  const void* bias;
  int act;
  View res;
  void* dact;
  // the logits' gradient instead of act: as kEpiGrad
  const float* coef;
  const float* lse;
  const int64_t* target;
  bool relu;           // slope is positive where act' is 1
};
struct SmallJobs {
  SmallJob j[2];
  int tiles0;
};
// Whether the launches of the tensor-core path would cost more than the product does here; `longest`
// is the longest of its sums, which one block makes alone.
constexpr int64_t kSmallWork = 1 << 24, kSmallSum = 512;
bool small_product(int64_t M, int64_t N, int64_t K, int64_t longest);
cudaError_t launch_small(int dtype, const SmallJob& a, const SmallJob* b, cudaStream_t s);

}  // namespace heads
}  // namespace vi
