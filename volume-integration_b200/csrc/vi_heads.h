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

enum Epi { kEpiAct, kEpiStore, kEpiPartial, kEpiLse, kEpiGrad };

// What happens to the product acc(m, n) = sum_k A(m, k) B(n, k).
struct Epilogue {
  int kind;
  int act;              // kEpiAct: vi_activation
  const void* bias;     // kEpiAct, kEpiLse, kEpiGrad: [N] or null
  View res;             // kEpiAct: residual, p null = none
  View out;             // kEpiAct, kEpiStore, kEpiGrad: T
  View dact;            // kEpiAct: act'(z), p null = not wanted
  const float* alpha;   // kEpiStore: device scalar the product is multiplied with, null = 1
  float* part;          // kEpiPartial: [splits][M][N]
  // kEpiLse: per (span of columns, row) the maximum of the logits and the sum of
  // exp(z - maximum), [spans][M] each, and the target's logit [M]
  float* pmax;
  float* psum;
  float* ztarget;
  const int64_t* target;
  // kEpiGrad: (exp(z - lse) - onehot) * coef per row, columns [col0, col0 + N) of the vocabulary
  const float* lse;
  const float* coef;
  int64_t col0;
};

}  // namespace heads
}  // namespace vi
