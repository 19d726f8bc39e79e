// Labels drawn from rows of logits.
//
// Mathematics.  With w_v = exp((z_v - max z) / T), candidates in the order of falling z (ties: lowest index first):
// top-k keeps the first k of them; top-p of those each whose mass before it is under p times their mass, the first
// always; min-p those with w_v >= min_p.  All three keep the front of the order, so what is kept is "z above a
// threshold, or equal to it and among the first few that are".  The answer is the first index, in index order, at
// which the running sum of the kept w exceeds u times their sum.
//
// The answer is a whole number that a border decides, so weights and sums are 64 bits wide: of 65536 candidates in
// float32 (1e-7 a weight) one draw in a hundred would fall on the wrong side.  Sums of weights are added in a fixed order, or as whole
// numbers of a unit (2^-46 of the largest up to V = 65536), so the same call gives the same label.
//
// The threshold is found without sorting: the logits' bits, made to order as unsigned integers, are narrowed by 8 bits
// at a time through histograms of counts (top-k) or masses (top-p).
#include <algorithm>

#include "vi_heads.h"
#include "vi_heads_math.cuh"
#include "vi_internal.h"

namespace vi {
namespace heads {
namespace {

// Bits that order as the value does; -0 as 0.
__device__ __forceinline__ uint32_t order_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// A row's settings.
struct Setting {
  double t, p, m;
  int64_t k;
};
__device__ __forceinline__ Setting setting_of(const SampleArgs& a, int64_t row) {
  Setting s;
  s.t = a.temperature ? (double)a.temperature[row] : a.temperature_all;
  s.p = a.top_p ? (double)a.top_p[row] : a.top_p_all;
  s.m = a.min_p ? (double)a.min_p[row] : a.min_p_all;
  s.k = a.top_k ? a.top_k[row] : a.top_k_all;
  return s;
}

constexpr int kThreads = 512;

struct Shared {
  double d[kThreads / 32];
  uint32_t u[kThreads / 32];
  unsigned long long mass[256];
  uint32_t count[256];
  uint32_t key, ties;
  unsigned long long above;
  int answer;
};

// A block a row, which it reads again for each step.
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* z = (const T*)a.z.p + row * a.z.rs;
    const auto key_at = [&](int v) { return order_of(to_f(z[v * a.z.cs])); };
    const Setting s = setting_of(a, row);
    // the largest key; whether there is a NaN
    uint32_t top = 0;
    bool nan = false;
    for (int v = tid; v < a.V; v += kThreads) {
      const float x = to_f(z[v * a.z.cs]);
      nan |= x != x;
      top = max(top, order_of(x));
    }
    nan = __syncthreads_or(nan || s.t != s.t);
    top = __reduce_max_sync(0xffffffffu, top);
    if (tid % 32 == 0) sh.u[tid / 32] = top;
    __syncthreads();
    for (int i = 0; i < kThreads / 32; i++) top = max(top, sh.u[i]);
    const float best = value_of(top);
    if (nan || best == -INFINITY) {
      if (tid == 0) a.label[row] = -1;
      __syncthreads();
      continue;
    }
    const bool greedy = !(s.t > 0.0);
    const auto weight = [&](uint32_t key) {
      const double x = (double)value_of(key);
      return key == top ? 1.0 : x == -INFINITY ? 0.0 : exp((x - (double)best) / s.t);
    };

    // kept: keys above `low`, and the first `ties` of those equal to it
    uint32_t low = greedy ? top : 0;
    uint32_t ties = greedy ? 1 : 0x7fffffff;
    // narrowed from the front of the order: count (by_mass false) or mass in front of the last one kept
    const auto narrow = [&](bool by_mass, uint64_t want) {
      uint32_t prefix = 0;
      uint64_t before = 0;  // in front of the keys that share the prefix
      const uint32_t old_low = low, old_ties = ties;
      uint32_t cut = 0;
      for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (tid < 256) sh.mass[tid] = 0, sh.count[tid] = 0;
        __syncthreads();
        for (int v = tid; v < a.V; v += kThreads) {
          const uint32_t k = key_at(v);
          if (k < old_low || (shift < 24 && (k >> (shift + 8)) != prefix)) continue;
          atomicAdd(&sh.count[k >> shift & 255], 1u);
          if (by_mass && k != old_low) atomicAdd(&sh.mass[k >> shift & 255], (unsigned long long)rint(weight(k) * a.unit));
        }
        __syncthreads();
        if (tid == 0) {
          uint64_t sum = before;
          int bin = 255;
          for (;; bin--) {
            uint64_t here = sh.count[bin];
            if (by_mass) {
              here = sh.mass[bin];
              // the last step's keys are told apart; of those at the old threshold only some are left
              if (old_low && old_low >> shift == ((shift < 24 ? prefix << 8 : 0) | (uint32_t)bin) && sh.count[bin])
                here += min(old_ties, sh.count[bin]) * (uint64_t)rint(weight(old_low) * a.unit);
            }
            if (bin == 0 || sum + here >= want) break;
            sum += here;
          }
          sh.key = bin;
          sh.ties = sh.count[bin];
          sh.above = sum;
        }
        __syncthreads();
        prefix = (shift < 24 ? prefix << 8 : 0) | sh.key;
        before = sh.above;
        cut = sh.ties;
      }
      low = prefix;
      uint64_t n = want - before;  // how many, or how much, of the keys equal to it
      if (by_mass) {
        const uint64_t one = (uint64_t)rint(weight(low) * a.unit);
        n = one ? (n + one - 1) / one : cut;
      }
      ties = (uint32_t)min(n, (uint64_t)cut);
      if (low == old_low) ties = min(ties, old_ties);
    };
    if (!greedy && s.k > 0 && s.k < a.V) narrow(false, s.k);
    if (!greedy && s.p < 1.0) {
      unsigned long long part = 0;
      uint32_t equal = 0;
      for (int v = tid; v < a.V; v += kThreads) {
        const uint32_t k = key_at(v);
        if (k > low) part += (unsigned long long)rint(weight(k) * a.unit);
        equal += k == low;
      }
      __syncthreads();
      if (tid == 0) sh.mass[0] = 0, sh.count[0] = 0;
      __syncthreads();
      atomicAdd(&sh.mass[0], part);
      atomicAdd(&sh.count[0], equal);
      __syncthreads();
      const uint64_t all = sh.mass[0] + min(ties, sh.count[0]) * (uint64_t)rint(weight(low) * a.unit);
      narrow(true, max((uint64_t)1, (uint64_t)ceil(fmax(s.p, 0.0) * (double)all)));
    }
    if (!greedy && s.m > 0.0 && low < top) {
      // the threshold rises to the lowest key whose weight is enough, if that is above it
      uint32_t least = 0xffffffffu;
      for (int v = tid; v < a.V; v += kThreads) {
        const uint32_t k = key_at(v);
        if (k >= low && (k == top || weight(k) >= s.m)) least = min(least, k);
      }
      least = __reduce_min_sync(0xffffffffu, least);
      __syncthreads();
      if (tid % 32 == 0) sh.u[tid / 32] = least;
      __syncthreads();
      for (int i = 0; i < kThreads / 32; i++) least = min(least, sh.u[i]);
      if (least > low) low = least, ties = 0x7fffffff;
    }

    // kept mass in index order: a piece of the row a thread, then the piece that holds the draw
    const int per = (a.V + kThreads - 1) / kThreads, v0 = min(a.V, tid * per), v1 = min(a.V, v0 + per);
    const double w_low = weight(low);
    uint32_t equal = 0;
    for (int v = v0; v < v1; v++) equal += key_at(v) == low;
    // equal ones in front of this thread's piece
    uint32_t scan = equal;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t n = __shfl_up_sync(0xffffffffu, scan, o);
      if (tid % 32 >= o) scan += n;
    }
    __syncthreads();
    if (tid % 32 == 31) sh.u[tid / 32] = scan;
    __syncthreads();
    uint32_t ahead = scan - equal;
    for (int i = 0; i < tid / 32; i++) ahead += sh.u[i];
    double mine = 0.0;
    uint32_t seen = ahead;
    for (int v = v0; v < v1; v++) {
      const uint32_t k = key_at(v);
      if (k > low) mine += weight(k);
      else if (k == low && seen++ < ties) mine += w_low;
    }
    double sum = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const double n = __shfl_up_sync(0xffffffffu, sum, o);
      if (tid % 32 >= o) sum += n;
    }
    __syncthreads();
    if (tid % 32 == 31) sh.d[tid / 32] = sum;
    if (tid == 0) sh.answer = 0x7fffffff;
    __syncthreads();
    double front = 0.0, total = 0.0;
    for (int i = 0; i < kThreads / 32; i++) {
      if (i == tid / 32) front = total;
      total += sh.d[i];
    }
    front += sum - mine;
    const double want = (double)a.u[row] * total;
    // the first index at which the running sum exceeds `want`; else (u >= 1) the last one kept
    int last = -1, hit = 0x7fffffff;
    double run = front;
    seen = ahead;
    for (int v = v0; v < v1; v++) {
      const uint32_t k = key_at(v);
      const bool in = k > low || (k == low && seen++ < ties);
      if (!in) continue;
      const double w = k == low ? w_low : weight(k);
      if (w > 0.0) last = v;
      run += w;
      if (run > want && w > 0.0) {
        hit = v;
        break;
      }
    }
    if (hit != 0x7fffffff) atomicMin(&sh.answer, hit);
    __syncthreads();
    const bool none = sh.answer == 0x7fffffff;
    __syncthreads();
    if (none) {
      if (tid == 0) sh.answer = -1;
      __syncthreads();
      atomicMax(&sh.answer, last);
      __syncthreads();
    }
    if (tid == 0) a.label[row] = sh.answer;
    __syncthreads();
  }
}

}  // namespace

cudaError_t launch_sample(int dtype, const SampleArgs& a, int sms, cudaStream_t s) {
  SampleArgs b = a;
  int bits = 0;
  while ((1ll << bits) < a.V) bits++;
  b.unit = ldexp(1.0, 62 - std::max(bits, 16));
  const unsigned blocks = (unsigned)std::min<int64_t>(a.M, (int64_t)sms * 4);
  if (dtype == VI_F32) sample_kernel<float><<<blocks, kThreads, 0, s>>>(b);
  else if (dtype == VI_F16) sample_kernel<__half><<<blocks, kThreads, 0, s>>>(b);
  else sample_kernel<__nv_bfloat16><<<blocks, kThreads, 0, s>>>(b);
  return cudaPeekAtLastError();
}

}  // namespace heads
}  // namespace vi
