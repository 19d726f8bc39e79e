// Labels drawn from rows of logits.
//
// Mathematics.  With w_v = exp((z_v - max z) / T), candidates in the order of falling z (ties: lowest index first):
// top-k keeps the first k of them; top-p of those each whose mass before it is under p times their mass, the first
// always; min-p those with w_v >= min_p.  All three keep the front of the order, so what is kept is "z above a
// threshold, or equal to it and among the first few that are".  The answer is the first index, in index order, at
// which the running sum of the kept w exceeds u times their sum.
//
// The answer is a whole number that a border decides.  Weights and sums in 64 bits decide it; where no top-k or
// top-p is asked for, float32 does, with a bound on its error, and a row whose draw falls within that bound of
// a border is done again in 64 bits (150 labels: one row in a thousand).  Sums are added in a fixed order: the same
// call gives the same labels.
//
// The threshold is found without sorting, by bisection over the logits' bits, made to order as unsigned integers:
// of rows that the registers hold (up to 8192 labels), or of a longer row's candidates.  Those are the labels above a
// guess, made from a sample of the row: one pass over the row keeps them, and shows (by their number, or their share
// of the mass) that no other label can be kept.
//
// 640000 x 150 (float16 image, min-p) takes 71 us (31 at the copy rate; instructions bound it); 1024 x 30011 (float32, top-k, top-p,
// min-p) 74 (19; the chains of bisections and the passes' 1.7 waves); 2048 x 65536 (bfloat16, top-p) 326 (41; instructions of two
// passes, 56 thousand a row, then the draws).
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstdlib>
#include <type_traits>

#include "vi_heads.h"
#include "vi_heads_math.cuh"
#include "vi_heads_tma.cuh"
#include "vi_internal.h"

namespace vi {
namespace heads {
namespace {

constexpr uint32_t kAll = 0xffffffffu;
constexpr uint32_t kManyTies = 0x7fffffffu;

// Bits that order as the value does; -0 as 0.  A 16-bit type's values, as floats, have low bits that are all alike: they
// are left out, which saves as many steps of a bisection.
template <typename T>
struct Order {
  static constexpr int kShift = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16, kBits = 32 - kShift;
  static __device__ __forceinline__ uint32_t of(float z) {
    const uint32_t b = __float_as_uint(z + 0.0f);
    return (b & 0x80000000u ? ~b : b | 0x80000000u) >> kShift;
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float(k >> (kBits - 1) ? k << kShift & 0x7fffffffu : ~(k << kShift | ((1u << kShift) - 1)));
  }
};

// 2^x for x <= 0, to 1e-14 of it (0 below 2^-1000, and where x is no number: an infinite distance to the largest at an infinite
// temperature): 2^x = 2^k e^(f ln 2) with k whole and |f| <= 1/2, by the exponential's series to the 12th power.
__device__ __forceinline__ double pow2_64(double x) {
  constexpr double l = 0.693147180559945309417232121458;
  constexpr double c[13] = {1.0,
                            l,
                            l * l / 2,
                            l * l * l / 6,
                            l * l * l * l / 24,
                            l * l * l * l * l / 120,
                            l * l * l * l * l * l / 720,
                            l * l * l * l * l * l * l / 5040,
                            l * l * l * l * l * l * l * l / 40320,
                            l * l * l * l * l * l * l * l * l / 362880,
                            l * l * l * l * l * l * l * l * l * l / 3628800,
                            l * l * l * l * l * l * l * l * l * l * l / 39916800,
                            l * l * l * l * l * l * l * l * l * l * l * l / 479001600};
  const double y = fmax(x, -1000.0), m = y + 0x1.8p52, f = y - (m - 0x1.8p52);
  double p = c[12];
#pragma unroll
  for (int i = 11; i >= 0; i--) p = fma(p, f, c[i]);
  return x >= -1000.0 ? __hiloint2double(__double2hiint(p) + (__double2loint(m) << 20), __double2loint(p)) : 0.0;
}

constexpr double kLog2e64 = 1.44269504088896340735992468100;
// A row's settings.
struct Setting {
  double t, p, m, u;
  int64_t k;
  double scale;  // log2(e) / t
};
__device__ __forceinline__ Setting setting_of(const SampleArgs& a, int64_t row) {
  Setting s;
  s.t = a.temperature ? (double)a.temperature[row] : a.temperature_all;
  s.p = a.top_p ? (double)a.top_p[row] : a.top_p_all;
  s.m = a.min_p ? (double)a.min_p[row] : a.min_p_all;
  if (s.m > 1.0) s.m = 1.0;  // a row's own: the largest is always kept
  s.k = a.top_k ? a.top_k[row] : a.top_k_all;
  s.u = fmax((double)a.u[row], 0.0);  // under 0, or a NaN: the first one kept
  s.scale = a.temperature ? kLog2e64 / s.t : a.scale_all;
  return s;
}
__device__ __forceinline__ double log2_min_p(const SampleArgs& a, const Setting& s) { return a.min_p ? log2(s.m) : a.log2_min_p_all; }
struct Weight {
  float best;
  double scale;  // log2(e) / T
  __device__ __forceinline__ Weight(float best, double scale) : best(best), scale(scale) {}
  __device__ __forceinline__ double of(float z) const {
    return z == best ? 1.0 : z == -INFINITY ? 0.0 : pow2_64(((double)z - (double)best) * scale);
  }
};

constexpr int kUnsure = -2;

// ---- a team of warps that holds a row, or a row's candidates ----
struct TeamShared {
  double d[2][16];
  uint32_t u[2][16];
};
template <int WARPS>
struct Team {
  TeamShared& sh;
  int warp, lane, turn = 0;  // two buffers in turn: a barrier each exchange
  __device__ __forceinline__ void sync() const {
    if constexpr (WARPS > 1) __syncthreads();
  }
  __device__ __forceinline__ uint32_t sum(uint32_t v) {
    v = __reduce_add_sync(kAll, v);
    if constexpr (WARPS > 1) {
      if (lane == 0) sh.u[turn][warp] = v;
      __syncthreads();
      v = lane < WARPS ? sh.u[turn][lane] : 0;
      v = __reduce_add_sync(kAll, v);
      turn ^= 1;
    }
    return v;
  }
  __device__ __forceinline__ uint32_t most(uint32_t v) {
    v = __reduce_max_sync(kAll, v);
    if constexpr (WARPS > 1) {
      if (lane == 0) sh.u[turn][warp] = v;
      __syncthreads();
      v = lane < WARPS ? sh.u[turn][lane] : 0;
      v = __reduce_max_sync(kAll, v);
      turn ^= 1;
    }
    return v;
  }
  __device__ __forceinline__ float sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    if constexpr (WARPS > 1) {
      if (lane == 0) sh.u[turn][warp] = __float_as_uint(v);
      __syncthreads();
      v = lane < WARPS ? __uint_as_float(sh.u[turn][lane]) : 0.0f;
#pragma unroll
      for (int o = WARPS / 2; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
      v = __shfl_sync(kAll, v, 0);
      turn ^= 1;
    }
    return v;
  }
  __device__ __forceinline__ double sum(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    if constexpr (WARPS > 1) {
      if (lane == 0) sh.d[turn][warp] = v;
      __syncthreads();
      v = lane < WARPS ? sh.d[turn][lane] : 0.0;
#pragma unroll
      for (int o = WARPS / 2; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
      v = __shfl_sync(kAll, v, 0);
      turn ^= 1;
    }
    return v;
  }
  // The place at which the running sum of the held w, in index order, exceeds u times their sum.  mine: the sum of the lane's; last:
  // its last place with weight, and one, in case u is 1 or more.  margin: kUnsure where a running sum is as near to
  // u times the sum as that share of it, or where `doubt`.
  template <int E, typename F>
  __device__ __forceinline__ int place(const F (&w)[E], double mine, double u, uint32_t last, float margin = 0.0f, bool doubt = false) {
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(kAll, mine, o);
    double before, total;
    ahead(mine, before, total);
    const double want = u * total, slack = total * margin;
    uint32_t hit = 0;
    // one warp's values hold it; its neighbours at the borders are looked at for the margin's sake
    if (before - slack <= want && before + mine + slack >= want && mine > 0.0) {
      double run = before;
      if (margin > 0.0f) doubt |= fabs(run - want) <= slack;
#pragma unroll
      for (int e = 0; e < E; e++) {
        F v = w[e];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const F t = __shfl_up_sync(kAll, v, d);
          if (lane >= d) v += t;
        }
        const double r = run + (double)v;
        if (w[e] > (F)0) {
          if (margin > 0.0f) doubt |= fabs(r - want) <= slack;
          if (r > want) hit = max(hit, ~(uint32_t)((warp * E + e) * 32 + lane));
          last = max(last, (uint32_t)((warp * E + e) * 32 + lane) + 1);
        }
        run += (double)__shfl_sync(kAll, v, 31);
      }
      // by its sum the warp holds the draw, though its running sums, added in another order, stay under it
      if (before <= want && before + mine > want && !__any_sync(kAll, hit)) hit = __reduce_max_sync(kAll, last) ? ~(__reduce_max_sync(kAll, last) - 1) : 0;
    }
    if (margin > 0.0f) {
      if constexpr (WARPS > 1) doubt = __syncthreads_or(doubt);
      else doubt = __any_sync(kAll, doubt);
      if (doubt) return kUnsure;
    }
    hit = most(hit);
    if (hit) return (int)~hit;
    return margin > 0.0f ? kUnsure : (int)most(last) - 1;
  }
  // what the warps in front of this one hold, and all
  __device__ __forceinline__ void ahead(uint32_t v, uint32_t& before) {
    before = 0;
    if constexpr (WARPS > 1) {
      if (lane == 0) sh.u[turn][warp] = v;
      __syncthreads();
      for (int i = 0; i < warp; i++) before += sh.u[turn][i];
      turn ^= 1;
    }
  }
  __device__ __forceinline__ void ahead(double v, double& before, double& all) {
    before = 0.0;
    all = v;
    if constexpr (WARPS > 1) {
      if (lane == 0) sh.d[turn][warp] = v;
      __syncthreads();
      all = 0.0;
      for (int i = 0; i < WARPS; i++) {
        if (i == warp) before = all;
        all += sh.d[turn][i];
      }
      turn ^= 1;
    }
  }
};

// The draw among held values, by the definition, in 64 bits.  A lane's value e stands for place (warp * E + e) * 32 + lane,
// which is index order.  `best` is the largest and finite or +inf; empty places hold -inf.  all: the mass that top-p's share is
// of, if it is known to `slack` (mass that is not held counts), else negative.  Returns the place; kUnsure where
// another mass within the slack would move the threshold, or where more than is held is asked for.
template <typename T, int E, int WARPS>
__device__ __forceinline__ int draw(Team<WARPS>& team, const float (&z)[E], float best, const Setting& s, int64_t labels,
                                    double all = -1.0, double slack = 0.0) {
  using O = Order<T>;
  const Weight weight(best, s.scale);
  const bool greedy = !(s.t > 0.0);
  const int lane = team.lane;
  uint32_t o[E];
#pragma unroll
  for (int e = 0; e < E; e++) o[e] = O::of(z[e]);
  // kept: order above `low`, and the first `ties` of those equal to it
  uint32_t low = greedy ? O::of(best) : 0, ties = greedy ? 1 : kManyTies;
  // bisections begin at the first bit in which what is held differs
  uint32_t least = kAll;
  if (!greedy && (s.p < 1.0 || (s.k > 0 && s.k < labels))) {
#pragma unroll
    for (int e = 0; e < E; e++) least = z[e] > -INFINITY ? min(least, o[e]) : least;
    least = ~team.most(~least);
  }
  const uint32_t differ = least ^ O::of(best);
  const int start = differ ? 31 - __clz(differ) : -1;
  const uint32_t common = start < 0 ? least : least >> start >> 1 << start << 1;
  if (!greedy && s.k > 0 && s.k < labels) {
    low = common;
#pragma unroll 1
    for (int bit = start; bit >= 0; bit--) {
      const uint32_t c = low | 1u << bit;
      uint32_t n = 0;
#pragma unroll
      for (int e = 0; e < E; e++) n += o[e] >= c;
      if (team.sum(n) >= s.k) low = c;
    }
    uint32_t n = 0;
#pragma unroll
    for (int e = 0; e < E; e++) n += o[e] > low;
    ties = (uint32_t)(s.k - team.sum(n));
  }
  double w[E];
#pragma unroll
  for (int e = 0; e < E; e++) w[e] = greedy ? (o[e] == low ? 1.0 : 0.0) : weight.of(z[e]);
  if (!greedy && s.p < 1.0) {
    const auto mass = [&](uint32_t from) {  // of what is above low, from `from` on
      double v = 0.0;
#pragma unroll
      for (int e = 0; e < E; e++) v += o[e] >= from && o[e] > low ? w[e] : 0.0;
      return team.sum(v);
    };
    uint32_t n = 0;
#pragma unroll
    for (int e = 0; e < E; e++) n += o[e] == low;
    n = min(team.sum(n), ties);
    const double at_low = n ? n * (low ? weight.of(O::value(low)) : 0.0) : 0.0;
    const bool all_known = all >= 0.0;
    if (!all_known) all = mass(0) + at_low;
    const double want = fmax(s.p * all, 1e-300);
    slack *= s.p;
    if (all_known && !(mass(0) + at_low - want > slack)) return kUnsure;
    // in float32, and again in 64 bits where that gives another threshold than 64 bits would
    uint32_t cut = common;
    {
      float f[E];
#pragma unroll
      for (int e = 0; e < E; e++) f[e] = o[e] > low ? (float)w[e] : 0.0f;
      const float about = (float)want;
#pragma unroll 1
      for (int bit = start; bit >= 0; bit--) {
        const uint32_t c = cut | 1u << bit;
        float v = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) v += o[e] >= c ? f[e] : 0.0f;
        if (c <= low || team.sum(v) >= about) cut = c;
      }
      cut = max(cut, low);
    }
    double above = mass(cut + 1);
    if (!((cut == low || mass(cut) >= want) && above < want)) {
      cut = common;
#pragma unroll 1
      for (int bit = start; bit >= 0; bit--) {
        const uint32_t c = cut | 1u << bit;
        if (c <= low || mass(c) >= want) cut = c;
      }
      cut = max(cut, low);
      above = mass(cut + 1);
    }
    const double one = cut ? weight.of(O::value(cut)) : 0.0;
    uint32_t have = 0;
#pragma unroll
    for (int e = 0; e < E; e++) have += o[e] == cut;
    have = team.sum(have);
    if (cut == low) have = min(have, ties);
    const double need = one > 0.0 ? ceil((want - above) / one) : (double)have;
    ties = (uint32_t)fmin(fmax(need, 1.0), (double)have);
    low = cut;
    if (slack > 0.0 && !(want - above - (ties - 1.0) * one > slack && above + ties * one - want > slack)) return kUnsure;
  }
  // kept weights; those equal to low by their number in index order
  uint32_t equal = 0;
#pragma unroll
  for (int e = 0; e < E; e++) equal += __popc(__ballot_sync(kAll, o[e] == low));
  uint32_t seen;
  team.ahead(equal, seen);
  const uint32_t first = O::of(best);
  double mine = 0.0;
  uint32_t last = 0;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const uint32_t b = __ballot_sync(kAll, o[e] == low);
    const bool in = o[e] > low || (o[e] == low && seen + __popc(b & ((1u << lane) - 1)) < ties);
    seen += __popc(b);
    w[e] = in && (!(w[e] < s.m) || o[e] == first) ? w[e] : 0.0;
    mine += w[e];
    if (w[e] > 0.0) last = (team.warp * E + e) * 32 + lane + 1;
  }
  return team.template place<E, double>(w, mine, s.u, last);
}

// The same where neither top-k nor top-p is asked for, in float32; kUnsure where the draw, or a label at min_p, is within
// the error of a border.  Sums of chains of E + 5 additions; the warps' in 64 bits.
template <int E, int WARPS>
__device__ __forceinline__ int draw_fast(Team<WARPS>& team, const float (&z)[E], float best, const Setting& s, float margin) {
  const float scale = (float)s.scale, least = (float)s.m;
  float w[E];
  double mine = 0.0;
  bool doubt = !(s.u < 1.0);
  float part = 0.0f;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const float x = exp2_fast((z[e] - best) * scale);
    doubt |= fabsf(x - least) <= 3e-5f * least && s.m > 0.0 && z[e] != best;
    w[e] = !(x < least) || z[e] == best ? x : 0.0f;
    part += w[e];
  }
  mine = part;
  return team.template place<E, float>(w, mine, s.u, 0, margin, doubt);
}

// Whether float32's weights serve: exponents within its reach (2^17 / 2^24 of one: the rounding that all weights share).
__device__ __forceinline__ bool plain_scale(const Setting& s, float best) {
  return s.t > 1e-30 && s.t < 1e30 && fabs((double)best) * s.scale < 0x1p17;
}

// Loads a row into registers and draws.
template <typename T, int E, int WARPS>
__device__ __forceinline__ int64_t row_label(Team<WARPS>& team, const SampleArgs& a, int64_t row, float margin) {
  using O = Order<T>;
  const T* p = (const T*)a.z.p + row * a.z.rs;
  float z[E];
  uint32_t top = 0;
  bool nan = false;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int v = (team.warp * E + e) * 32 + team.lane;
    z[e] = v < a.V ? to_f(p[v * a.z.cs]) : -INFINITY;
  }
  const Setting s = setting_of(a, row);
#pragma unroll
  for (int e = 0; e < E; e++) {
    nan |= z[e] != z[e];
    top = max(top, O::of(z[e]));
  }
  top = team.most(nan || s.t != s.t ? kAll : top);  // no value's order is kAll
  if (top == kAll) return -1;
  const float best = O::value(top);
  if (best == -INFINITY) return -1;
  if (margin > 0.0f && !(s.k > 0 && s.k < a.V) && !(s.p < 1.0) && plain_scale(s, best)) {
    const int v = draw_fast<E, WARPS>(team, z, best, s, margin);
    if (v >= 0) return v;
  }
  return draw<T, E, WARPS>(team, z, best, s, a.V);
}

// Rows of up to 32 E WARPS labels: WARPS warps a row.
template <typename T, int E, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 256 : 32 * WARPS) sample_rows_kernel(const __grid_constant__ SampleArgs a) {
  __shared__ TeamShared sh;
  Team<WARPS> team{sh, WARPS == 1 ? 0 : (int)threadIdx.x / 32, (int)threadIdx.x % 32};
  const int teams = WARPS == 1 ? 8 : 1;
  for (int64_t row = (int64_t)blockIdx.x * teams + (WARPS == 1 ? threadIdx.x / 32 : 0); row < a.M; row += (int64_t)gridDim.x * teams) {
    const int64_t v = row_label<T, E, WARPS>(team, a, row, a.margin);
    if (team.lane == 0 && team.warp == 0) a.label[row] = v;
    team.sync();
  }
}

// ---- images: neighbouring rows lie next to each other ----
// A thread a pixel, or two of 16-bit logits, where neither top-k nor top-p is asked for: no exchange between lanes.  The first pass
// finds the largest, the second the sums of 16 pieces of the row, the third walks through the piece that holds the draw.
// The first reads memory, the others mostly the caches.
constexpr int kPieces = 16, kImageThreads = 128;
// A row by a warp in 64 bits, without top-k, top-p and temperature 0: 32 labels at a time, once for the sum and once for the
// draw.  at(v): the logit of label v.
template <typename F>
__device__ __forceinline__ int row_again(int V, const Setting& s, float best, F at) {
  const int lane = threadIdx.x % 32;
  const Weight weight(best, s.scale);
  double run = 0.0, want = 0.0;
  int last = -1;
#pragma unroll 1
  for (int pass = 0; pass < 2; pass++) {
    if (pass) want = s.u * run;
    run = 0.0;
#pragma unroll 1
    for (int first = 0; first < V; first += 32) {
      const float z = first + lane < V ? at(first + lane) : -INFINITY;
      double w = weight.of(z);
      if (w < s.m && z != best) w = 0.0;
      double scan = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double t = __shfl_up_sync(kAll, scan, d);
        if (lane >= d) scan += t;
      }
      const uint32_t kept = __ballot_sync(kAll, w > 0.0), hit = __ballot_sync(kAll, pass && w > 0.0 && run + scan > want);
      if (hit) return first + __ffs(hit) - 1;
      if (kept) last = first + 31 - __clz(kept);
      run += __shfl_sync(kAll, scan, 31);
    }
  }
  return last;  // u of 1 and more
}
template <typename T>
__device__ __noinline__ int64_t image_row_again(const SampleArgs& a, int64_t row) {
  const T* p = (const T*)a.z.p + row * a.z.rs;
  float best = -INFINITY;
  for (int v = threadIdx.x % 32; v < a.V; v += 32) best = fmaxf(best, to_f(p[v * a.z.cs]));
#pragma unroll
  for (int o = 16; o; o >>= 1) best = fmaxf(best, __shfl_xor_sync(kAll, best, o));
  return row_again(a.V, setting_of(a, row), best, [&](int v) { return to_f(p[v * a.z.cs]); });
}
template <typename T, int PX>
struct Pixels {
  float v[PX];
  __device__ __forceinline__ explicit Pixels(const T* p) {
    if constexpr (PX == 1) {
      v[0] = to_f(*p);
    } else {
      const uint32_t w = *(const uint32_t*)p;
      const float2 f = std::is_same<T, __half>::value ? __half22float2(*(const __half2*)&w) : __bfloat1622float2(*(const __nv_bfloat162*)&w);
      v[0] = f.x, v[1] = f.y;
    }
  }
};
template <typename T, int PX>
__global__ void __launch_bounds__(kImageThreads) sample_image_kernel(const __grid_constant__ SampleArgs a) {
  __shared__ float pieces[kPieces][PX][kImageThreads];
  const int len = (a.V + kPieces - 1) / kPieces;
  const int64_t step = (int64_t)gridDim.x * kImageThreads * PX;
  for (int64_t base = (int64_t)blockIdx.x * kImageThreads * PX; base < a.M; base += step) {
    const int64_t row = base + threadIdx.x * PX;
    const bool here = row < a.M;
    uint32_t again = 0;  // pixels that float32 does not decide
    if (here) {
      const T* p = (const T*)a.z.p + row * a.z.rs;
      float best[PX], scale[PX], least[PX], reach[PX];  // reach: how near to least float32 does not decide
      bool first[PX];  // temperature 0
#pragma unroll
      for (int j = 0; j < PX; j++) best[j] = -INFINITY;
#pragma unroll 8
      for (int v = 0; v < a.V; v++) {
        const Pixels<T, PX> z(p + v * a.z.cs);
#pragma unroll
        for (int j = 0; j < PX; j++) best[j] = max_nan(best[j], z.v[j]);
      }
      Setting s[PX];
      bool draws = false, firsts = false;
#pragma unroll
      for (int j = 0; j < PX; j++) {
        s[j] = setting_of(a, row + j);
        first[j] = !(s[j].t > 0.0) && s[j].t == s[j].t;
        if (best[j] != best[j] || s[j].t != s[j].t || best[j] == -INFINITY) {
          a.label[row + j] = -1;
          s[j].u = -1.0;  // done
        } else if (first[j]) {
          firsts = true;
        } else if (!plain_scale(s[j], best[j])) {
          again |= 1u << j;
          s[j].u = -1.0;
        } else {
          draws = true;
        }
        scale[j] = (float)s[j].scale;
        least[j] = (float)s[j].m;
        // The largest's weight, which is 1 exactly, is not in doubt.  Weights next to it are off by 2^-22 alone, as their
        // exponents are next to 0.  A min_p of 1 keeps the largest only: a scale that leaves no other weight at 1.
        reach[j] = 3e-5f * least[j];
        if (1.0f - least[j] > 1e-6f) reach[j] = fminf(reach[j], 1.0f - least[j]);
        if (s[j].m >= 1.0) scale[j] = FLT_MAX, reach[j] = 0.0f;
      }
      if (firsts) {
        int at[PX];
#pragma unroll
        for (int j = 0; j < PX; j++) at[j] = a.V;
#pragma unroll 8
        for (int v = a.V - 1; v >= 0; v--) {
          const Pixels<T, PX> z(p + v * a.z.cs);
#pragma unroll
          for (int j = 0; j < PX; j++) at[j] = z.v[j] == best[j] ? v : at[j];
        }
#pragma unroll
        for (int j = 0; j < PX; j++)
          if (first[j] && s[j].u >= 0.0) a.label[row + j] = at[j];
      }
      if (draws) {
        float run[PX] = {};
        bool doubt[PX] = {};
        const auto weight = [&](float z, int j) {
          const float x = exp2_fast((z - best[j]) * scale[j]);
          doubt[j] |= fabsf(x - least[j]) < reach[j];
          return x < least[j] ? 0.0f : x;
        };
        for (int c = 0; c < kPieces; c++) {
          const int v1 = min(a.V, (c + 1) * len);
          float sum[PX] = {};
#pragma unroll 8
          for (int v = c * len; v < v1; v++) {
            const Pixels<T, PX> z(p + v * a.z.cs);
#pragma unroll
            for (int j = 0; j < PX; j++) sum[j] += weight(z.v[j], j);
          }
#pragma unroll
          for (int j = 0; j < PX; j++) {
            run[j] += sum[j];
            pieces[c][j][threadIdx.x] = run[j];
          }
        }
#pragma unroll
        for (int j = 0; j < PX; j++) {
          if (first[j] || s[j].u < 0.0) continue;
          const float total = run[j], want = (float)s[j].u * total, slack = total * a.margin;
          int c = 0;
          while (c < kPieces - 1 && pieces[c][j][threadIdx.x] <= want) c++;
          float r = c ? pieces[c - 1][j][threadIdx.x] : 0.0f, sum = 0.0f;
          const float start = r;
          int at = -1;
          bool near = fabsf(r - want) <= slack;
          for (int v = c * len; v < min(a.V, (c + 1) * len); v++) {
            sum += weight(to_f(p[v * a.z.cs + j]), j);
            r = start + sum;
            near |= fabsf(r - want) <= slack;
            if (at < 0 && r > want) at = v;
          }
          if (near || doubt[j] || at < 0 || !(s[j].u < 1.0)) again |= 1u << j;
          else a.label[row + j] = at;
        }
      }
    }
    // what is left, a warp a row
    __syncwarp();
#pragma unroll
    for (int j = 0; j < PX; j++) {
      uint32_t todo = __ballot_sync(kAll, again >> j & 1);
      while (todo) {
        const int l = __ffs(todo) - 1;
        todo &= todo - 1;
        const int64_t r = __shfl_sync(kAll, row, l) + j, v = image_row_again<T>(a, r);
        if (threadIdx.x % 32 == 0) a.label[r] = v;
      }
    }
  }
}

__device__ __forceinline__ uint32_t max_nan2(uint32_t a, uint32_t b, __half) {
  const __half2 r = __hmax2_nan(*(const __half2*)&a, *(const __half2*)&b);
  return *(const uint32_t*)&r;
}
__device__ __forceinline__ uint32_t max_nan2(uint32_t a, uint32_t b, __nv_bfloat16) {
  const __nv_bfloat162 r = __hmax2_nan(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
  return *(const uint32_t*)&r;
}
// All bits of each half of `a` that is at least b's.
__device__ __forceinline__ uint32_t at_least2(uint32_t a, uint32_t b, __half) { return __hge2_mask(*(const __half2*)&a, *(const __half2*)&b); }
__device__ __forceinline__ uint32_t at_least2(uint32_t a, uint32_t b, __nv_bfloat16) {
  return __hge2_mask(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
}
template <typename T>
__device__ __forceinline__ uint32_t pair_bits(T a, T b) {
  return (uint32_t) * (const unsigned short*)&a | (uint32_t) * (const unsigned short*)&b << 16;
}

// The same from shared memory, where bulk copies reach the image (16-byte strides) and its labels are at most 256: a block
// takes 256 bytes of each label's pixels, 64 threads with a pixel or a pair of 16-bit ones each.  The copy needs no
// registers and no address arithmetic, and each pass reads shared memory at constant offsets.
// Weights beside the largest's: exp2(z scale - best scale), whose constant's rounding is a factor of all alike.
constexpr int kTileThreads = 64, kTileLabels = 256;
template <typename T>
__global__ void __launch_bounds__(kTileThreads) sample_tiles_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ SampleArgs a) {
  constexpr int PX = 4 / (int)sizeof(T), kLen = 16;
  constexpr uint32_t none = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  extern __shared__ __align__(128) uint32_t words[];  // [labels, whole pieces][threads]
  const int tid = threadIdx.x, pieces = (a.V + kLen - 1) / kLen;
  uint32_t* const own = words + tid;
  float* const runs = (float*)(words + pieces * kLen * kTileThreads) + tid;  // [pieces][PX][threads]
  __shared__ uint64_t bar_word;
  __shared__ int dead_word;
  volatile int* dead = &dead_word;
  const uint32_t bar = smem_u32(&bar_word);
  const auto value = [](uint32_t w, int j) -> float {
    if constexpr (PX == 1) return __uint_as_float(w);
    else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)(j ? w >> 16 : w & 0xffffu)));
    else return __uint_as_float(j ? w & 0xffff0000u : w << 16);
  };
  for (int v = a.V; v < pieces * kLen; v++) own[v * kTileThreads] = none;
  if (tid == 0) {
    mbar_init(bar, 1);
    dead_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  uint32_t phase = 0;
  const int64_t tiles = (a.M + kTileThreads * PX - 1) / (kTileThreads * PX);
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, phase ^= 1) {
    if (tid == 0 && !a.withhold) {
      mbar_expect(bar, a.V * kTileThreads * 4);
      tma_load<false>(smem_u32(words), &map, bar, (int)(tile * kTileThreads * PX), 0, 0);
    }
    bool on = mbar_wait(bar, phase, dead, a.wait_limit);
    if (a.lapse && tid == 37) on = false, *dead = 1;
    if (!__syncthreads_and(on)) break;  // the block leaves together: what follows exchanges between lanes, and has a barrier
    const int64_t row = (tile * kTileThreads + tid) * PX;
    uint32_t again = 0;  // pixels that float32 does not decide
    float best[PX];
    {
      uint32_t m[2] = {none, none};
      for (int c = 0; c < pieces; c++) {
#pragma unroll
        for (int i = 0; i < kLen; i++) {
          const uint32_t w = own[(c * kLen + i) * kTileThreads];
          if constexpr (PX == 1) m[i & 1] = __float_as_uint(max_nan(__uint_as_float(m[i & 1]), __uint_as_float(w)));
          else m[i & 1] = max_nan2(m[i & 1], w, T());
        }
      }
#pragma unroll
      for (int j = 0; j < PX; j++) best[j] = max_nan(value(m[0], j), value(m[1], j));
    }
    Setting s[PX];
    bool draws[PX], near[PX], cut = false, any = false;
    T least[PX];  // min-p keeps the logits from a value on: the type's first value there
    float scale[PX], shift[PX];
#pragma unroll
    for (int j = 0; j < PX; j++) {
      draws[j] = false;
      least[j] = from_f<T>(-INFINITY);
      scale[j] = shift[j] = 0.0f;
      if (row + j >= a.M) continue;
      s[j] = setting_of(a, row + j);
      near[j] = !(s[j].u < 1.0);
      if (best[j] != best[j] || s[j].t != s[j].t || best[j] == -INFINITY) {
        a.label[row + j] = -1;
      } else if (!(s[j].t > 0.0)) {
        int at = 0;
        for (int c = pieces - 1; c >= 0; c--) {
#pragma unroll
          for (int i = kLen - 1; i >= 0; i--) at = value(own[(c * kLen + i) * kTileThreads], j) == best[j] ? c * kLen + i : at;
        }
        a.label[row + j] = at;
      } else if (!plain_scale(s[j], best[j])) {
        again |= 1u << j;
      } else {
        draws[j] = any = true;
        scale[j] = (float)s[j].scale;
        shift[j] = -best[j] * scale[j];
        if (s[j].m >= 1.0) {
          least[j] = from_f<T>(best[j]);
          cut = true;
        } else if (s[j].m > 0.0) {
          const double at = (double)best[j] + (a.min_p || a.temperature ? log2_min_p(a, s[j]) / s[j].scale : a.cut_all);
          double round;
          if constexpr (sizeof(T) == 4) least[j] = __double2float_ru(at), round = (double)(float)at;
          else if constexpr (std::is_same<T, __half>::value) least[j] = __float2half_ru(__double2float_ru(at)), round = (double)__half2float(__double2half(at));
          else least[j] = __float2bfloat16_ru(__double2float_ru(at)), round = (double)__bfloat162float(__double2bfloat16(at));
          near[j] |= fabs(round - at) <= 1e-12 * (fabs(at) + fabs((double)best[j]));
          cut = true;
        }
      }
    }
    uint32_t from;
    if constexpr (PX == 1) from = __float_as_uint(least[0]);
    else from = pair_bits(least[0], least[1]);
    // the word of label v without what min-p drops
    const auto kept = [&](auto cuts, uint32_t w) {
      if constexpr (!decltype(cuts)::value) return w;
      else if constexpr (PX == 1) return __uint_as_float(w) >= __uint_as_float(from) ? w : none;
      else {
        const uint32_t in = at_least2(w, from, T());
        return (w & in) | (none & ~in);
      }
    };
    const auto draw_pixels = [&](auto cuts) {
      float run[PX] = {};
      for (int c = 0; c < pieces; c++) {
        float q[PX][2] = {};
#pragma unroll
        for (int i = 0; i < kLen; i++) {
          const uint32_t w = kept(cuts, own[(c * kLen + i) * kTileThreads]);
#pragma unroll
          for (int j = 0; j < PX; j++) q[j][i & 1] += exp2_fast(fmaf(value(w, j), scale[j], shift[j]));
        }
#pragma unroll
        for (int j = 0; j < PX; j++) runs[(c * PX + j) * kTileThreads] = run[j] += q[j][0] + q[j][1];
      }
#pragma unroll
      for (int j = 0; j < PX; j++) {
        if (!draws[j]) continue;
        const float want = (float)s[j].u * run[j], slack = run[j] * a.margin;
        int c = 0;
        float start = 0.0f;
        for (int i = 0; i < pieces - 1; i++) {
          const float r = runs[(i * PX + j) * kTileThreads];
          const bool behind = r <= want;
          c += behind;
          start = behind ? r : start;
        }
        bool close = near[j] | (fabsf(start - want) <= slack);
        int at = -1;
        float r = 0.0f;
        const uint32_t* piece = own + c * kLen * kTileThreads;
#pragma unroll
        for (int i = 0; i < kLen; i++) {
          r += exp2_fast(fmaf(value(kept(cuts, piece[i * kTileThreads]), j), scale[j], shift[j]));
          close |= fabsf(start + r - want) <= slack;
          at = at < 0 && start + r > want ? c * kLen + i : at;
        }
        if (close || at < 0) again |= 1u << j;
        else a.label[row + j] = at;
      }
    };
    if (any) {
      if (cut) draw_pixels(std::true_type());
      else draw_pixels(std::false_type());
    }
    // what is left, a warp a row
    __syncwarp();
#pragma unroll
    for (int j = 0; j < PX; j++) {
      uint32_t todo = __ballot_sync(kAll, again >> j & 1);
      while (todo) {
        const int l = __ffs(todo) - 1;
        todo &= todo - 1;
        const int64_t r = __shfl_sync(kAll, row, l) + j;
        const uint32_t* column = words + (tid & 32) + l;
        const int v = row_again(a.V, setting_of(a, r), __shfl_sync(kAll, best[j], l), [&](int v) { return value(column[v * kTileThreads], j); });
        if (tid % 32 == 0) a.label[r] = v;
      }
    }
    __syncthreads();
  }
  if (tid == 0 && *dead) {  // the copy in flight ends before the block does
    if (!a.withhold) mbar_drain(bar, phase, a.wait_limit);
    atomicOr(a.status, VI_DEVICE_HEAD_TIMEOUT);
  }
}

// ---- long rows: a block a row ----
constexpr int kRowLabels = 8192;               // that a block's registers hold
constexpr int kHeld = 16;
constexpr int kListWarp = 32 * kHeld;          // candidates a warp keeps
constexpr int kSample = 32;                    // labels a lane looks at for the guess
constexpr int kSums = 64;                      // sums of steps a warp keeps
constexpr int kBins = 256;
constexpr int kFew = 256;                      // candidates that one warp draws from
template <int W>
struct LongShared {
  TeamShared team;
  union {
    float sums[W][kSums];
    double mass[W][kSums];
  };
  uint32_t equal[W][kSums];
  uint32_t bins[kBins];
  int few[kFew];
  float guess;
  int answer;
};
// What the passes over a row leave for the draw.
enum { kDone, kFromList, kWhole };
struct RowNote {
  double all;       // mass beside exp2 of ref scale, as rounded to float32
  float best, ref;
  int state;
  int n[16];        // candidates of each warp
  int pad[3];
};
__host__ __device__ constexpr int64_t list_bytes(int warps) { return (int64_t)warps * kListWarp * 4; }
__device__ __forceinline__ int* list_of(const SampleArgs& a, int64_t row) { return (int*)((char*)a.scratch + a.list_at + row * a.list_bytes); }

// How a row is read: any stride, or contiguous, in 16-byte vectors.
enum { kStrided, kVectors };

// A row whose labels are counted from the 16-byte boundary at or before its first one (kVectors): label v has place v + shift.
template <typename T, int MODE>
struct Row {
  const T* p;  // of place 0, which is not read where shift is not 0
  int64_t cs;
  int shift, end;
  __device__ __forceinline__ Row(const SampleArgs& a, int64_t row) {
    p = (const T*)a.z.p + row * a.z.rs;
    cs = a.z.cs;
    shift = MODE == kVectors ? (int)((uintptr_t)p % 16 / sizeof(T)) : 0;
    p -= shift;
    end = a.V + shift;
  }
  __device__ __forceinline__ float at(int place) const { return to_f(p[MODE == kVectors ? (int64_t)place : place * cs]); }
};
// Steps of 256 places of each of W warps.
template <int W, typename T>
__host__ __device__ constexpr int64_t part_of(int64_t V) { return (V + 16 / (int)sizeof(T) + W * 256 - 1) / (W * 256) * 256; }

// What a lane holds of 256 places from `first` on: 8 in a row (kVectors), or every 32nd; -inf where there is no label.
template <typename T, int MODE>
struct Step {
  static constexpr int kPer = 16 / (int)sizeof(T);
  union {
    uint4 q[8 / kPer];
    T t[8];
  };
  __device__ __forceinline__ Step() {}
  __device__ __forceinline__ float z(int e) const { return to_f(t[e]); }
  static __device__ __forceinline__ int place(int first, int lane, int e) { return MODE == kVectors ? first + lane * 8 + e : first + e * 32 + lane; }
  __device__ __forceinline__ void load(const Row<T, MODE>& r, int first, int lane, int end) {
    if constexpr (MODE == kVectors) {
      if (first + 256 <= end && first >= kPer) return load_whole(r, first, lane);
#pragma unroll
      for (int i = 0; i < 8 / kPer; i++) {
        const int v = first + lane * 8 + i * kPer;
        if (v >= r.shift && v + kPer <= end) {
          q[i] = *(const uint4*)(r.p + v);
        } else {
#pragma unroll
          for (int e = 0; e < kPer; e++) t[i * kPer + e] = v + e >= r.shift && v + e < end ? r.p[v + e] : from_f<T>(-INFINITY);
        }
      }
    } else {
      const T* at = r.p + (first + lane) * r.cs;
      const int64_t step = 32 * r.cs;
#pragma unroll
      for (int e = 0; e < 8; e++) t[e] = first + e * 32 + lane < end ? at[e * step] : from_f<T>(-INFINITY);
    }
  }
  // The same where all 256 places hold labels.
  __device__ __forceinline__ void load_whole(const Row<T, MODE>& r, int first, int lane) {
#pragma unroll
    for (int i = 0; i < 8 / kPer; i++) q[i] = ((const uint4*)(r.p + first + lane * 8))[i];
  }
  // The largest, or a NaN if there is one.
  __device__ __forceinline__ float most(float m) const {
    if constexpr (sizeof(T) == 4 || MODE != kVectors) {
#pragma unroll
      for (int e = 0; e < 8; e++) m = max_nan(m, z(e));
      return m;
    } else {
      uint32_t w = max_nan2(max_nan2(q[0].x, q[0].y, T()), max_nan2(q[0].z, q[0].w, T()), T());
      const T a = ((const T*)&w)[0], b = ((const T*)&w)[1];
      return max_nan(m, max_nan(to_f(a), to_f(b)));
    }
  }
  // Bit e: whether value e is at least `from`.
  __device__ __forceinline__ uint32_t at_least(float from, uint32_t from2) const {
    uint32_t in = 0;
    if constexpr (sizeof(T) == 4 || MODE != kVectors) {
#pragma unroll
      for (int e = 0; e < 8; e++) in |= z(e) >= from ? 1u << e : 0u;
    } else {
      const uint32_t a = at_least2(q[0].x, from2, T()), b = at_least2(q[0].y, from2, T()), c = at_least2(q[0].z, from2, T()),
                     d = at_least2(q[0].w, from2, T());
      if (a | b | c | d)
        in = (a & 1) | (a >> 30 & 2) | (b & 4) | (b >> 28 & 8) | (c & 16) | (c >> 26 & 32) | (d & 64) | (d >> 24 & 128);
    }
    return in;
  }
};

// f of every label of a row and of some -inf, in any order: several loads in flight.
template <int W, typename T, int MODE, typename F>
__device__ __forceinline__ void each_of_row(const Row<T, MODE>& row, int warp, int lane, F f) {
  constexpr int kDeep = sizeof(T) == 4 ? 2 : 4;
  for (int first = warp * 256; first < row.end; first += kDeep * W * 256) {
    Step<T, MODE> x[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; i++) x[i].load(row, first + i * W * 256, lane, row.end);
#pragma unroll
    for (int i = 0; i < kDeep; i++) {
#pragma unroll
      for (int e = 0; e < 8; e++) f(x[i].z(e));
    }
  }
}

// The whole row by the definition in 64 bits, read again for every step of the bisections: where the guess was
// wrong, or candidates are too many to be held; and where float32 leaves a plain draw in doubt.
template <int W, typename T, int MODE>
__device__ __noinline__ int whole_row(Team<W>& team, LongShared<W>& sh, const Row<T, MODE>& row, int V, float best, const Setting& s) {
  using O = Order<T>;
  const Weight weight(best, s.scale);
  const int warp = team.warp, lane = team.lane;
  const bool greedy = !(s.t > 0.0);
  uint32_t low = greedy ? O::of(best) : 0, ties = greedy ? 1 : kManyTies;
  const auto each = [&](auto f) { each_of_row<W, T, MODE>(row, warp, lane, f); };
  const auto count = [&](auto f) {
    uint32_t n = 0;
    each([&](float z) { n += f(O::of(z)); });
    return team.sum(n);
  };
  const auto mass = [&](uint32_t from) {  // of what is above low, from `from` on
    double m = 0.0;
    each([&](float z) {
      const uint32_t o = O::of(z);
      const double w = weight.of(z);
      m += o >= from && o > low ? w : 0.0;
    });
    return team.sum(m);
  };
  if (!greedy && s.k > 0 && s.k < V) {
    for (int bit = O::kBits - 1; bit >= 0; bit--) {
      const uint32_t c = low | 1u << bit;
      if (count([&](uint32_t o) { return o >= c; }) >= s.k) low = c;
    }
    ties = (uint32_t)(s.k - count([&](uint32_t o) { return o > low; }));
  }
  if (!greedy && s.p < 1.0) {
    const uint32_t end = O::of(best), n_low = low ? min(count([&](uint32_t o) { return o == low; }), ties) : 0;
    const double at_low = n_low ? n_low * weight.of(O::value(low)) : 0.0;
    uint32_t cut = 0, have = 0;
    double want = 0.0, above = 0.0;
    bool found = false;
    // the threshold's own label count, the mass above it and the whole, in one pass of 64 bits: does the threshold stand?
    const auto stands = [&] {
      double whole = 0.0, front = 0.0;
      uint32_t n = 0;
      each([&](float z) {
        const uint32_t o = O::of(z);
        const double w = o > low ? weight.of(z) : 0.0;
        whole += w;
        front += o > cut ? w : 0.0;
        n += o == cut;
      });
      want = fmax(s.p * (team.sum(whole) + at_low), 1e-300);
      above = team.sum(front);
      have = team.sum(n);
      if (cut == low) have = min(have, ties);
      return above < want && (cut == low || above + have * weight.of(O::value(cut)) >= want);
    };
    if (plain_scale(s, best)) {  // in float32 first
      const float scale = (float)s.scale, shift = -best * scale;
      const auto mass32 = [&](uint32_t from) {
        float m = 0.0f;
        each([&](float z) {
          const uint32_t o = O::of(z);
          m += o >= from && o > low ? exp2_fast(fmaf(z, scale, shift)) : 0.0f;
        });
        return team.sum(m);
      };
      const float about = (float)s.p * (mass32(0) + (float)at_low);
      for (int bit = O::kBits - 1; bit >= 0; bit--) {
        const uint32_t c = cut | 1u << bit;
        if (c <= end && (c <= low || mass32(c) >= about)) cut = c;
      }
      cut = max(cut, low);
      found = stands();
    }
    if (!found) {
      cut = 0;
      stands();  // for `want`
      for (int bit = O::kBits - 1; bit >= 0; bit--) {
        const uint32_t c = cut | 1u << bit;
        if (c <= end && (c <= low || mass(c) >= want)) cut = c;
      }
      cut = max(cut, low);
      stands();
    }
    const double one = cut ? weight.of(O::value(cut)) : 0.0, need = one > 0.0 ? ceil((want - above) / one) : (double)have;
    ties = (uint32_t)fmin(fmax(need, 1.0), (double)have);
    low = cut;
  }
  // in index order: a warp a part of the row.  Of each group of its steps the mass above the threshold, and how many labels
  // are equal to it
  const int part = (int)part_of<W, T>(V), v0 = min(row.end, warp * part), v1 = min(row.end, v0 + part);
  const int steps = part / 256, group = (steps + kSums - 1) / kSums;
  const auto enough = [&](double w, float z) { return greedy || !(w < s.m) || z == best; };
  const float z_low = low ? O::value(low) : -INFINITY;
  double w_low = weight.of(z_low);
  if (!enough(w_low, z_low)) w_low = 0.0;
  const bool limited = low > 0;
  for (int g = lane; g < kSums; g += 32) sh.mass[warp][g] = 0.0, sh.equal[warp][g] = 0;
  __syncwarp();
  Step<T, MODE> next;
  next.load(row, v0, lane, v1);
  for (int i0 = 0; i0 < steps && v0 + i0 * 256 < v1; i0 += group) {
    double m = 0.0;
    uint32_t n = 0;
    for (int i = i0; i < min(steps, i0 + group) && v0 + i * 256 < v1; i++) {
      const Step<T, MODE> x = next;
      next.load(row, v0 + (i + 1) * 256, lane, v1);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float z = x.z(e);
        const uint32_t o = O::of(z);
        const double w = weight.of(z);
        m += o > low && enough(w, z) ? w : 0.0;
        n += o == low;
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m += __shfl_xor_sync(kAll, m, o);
    n = __reduce_add_sync(kAll, n);
    if (lane == 0) sh.mass[warp][i0 / group] = m, sh.equal[warp][i0 / group] = limited ? n : 0;
  }
  __syncwarp();
  // groups 2 lane and 2 lane + 1: equal ones in front of them, then running masses
  static_assert(kSums == 64, "two groups a lane");
  const uint32_t n0 = sh.equal[warp][2 * lane], n1 = sh.equal[warp][2 * lane + 1];
  uint32_t scan = n0 + n1;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t t = __shfl_up_sync(kAll, scan, d);
    if (lane >= d) scan += t;
  }
  uint32_t ahead;
  team.ahead(__shfl_sync(kAll, scan, 31), ahead);
  const uint32_t e0 = ahead + scan - n0 - n1, e1 = e0 + n0;
  const auto some = [&](uint32_t from, uint32_t n) { return (double)(min(ties, from + n) - min(ties, from)) * w_low; };
  const double m0 = sh.mass[warp][2 * lane] + some(e0, n0), m1 = sh.mass[warp][2 * lane + 1] + some(e1, n1);
  double run = m0 + m1;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double t = __shfl_up_sync(kAll, run, d);
    if (lane >= d) run += t;
  }
  const double mine = __shfl_sync(kAll, run, 31);
  double before, total;
  team.ahead(mine, before, total);
  const double want = s.u < 1.0 ? s.u * total : INFINITY;
  // the warp whose part holds the draw (u of 1 and more: every warp, for its last label)
  uint32_t hit = 0, last = 0;
  if (mine > 0.0 && ((before <= want && before + mine > want) || !(s.u < 1.0))) {
    // in front of the lane's groups: sums of what lies there alone, so that in front of the first label with weight there is 0
    const double others = __shfl_up_sync(kAll, run, 1), f0 = before + (lane ? others : 0.0), f1 = f0 + m0;
    const uint32_t holds = __ballot_sync(kAll, (f1 > want && m0 > 0.0) || (f1 + m1 > want && m1 > 0.0));
    const uint32_t some_mass = __ballot_sync(kAll, m0 + m1 > 0.0);
    const int l = holds ? __ffs(holds) - 1 : 31 - __clz(some_mass);
    for (int half = 0; half < 2 && !hit; half++) {
      const int g = 2 * l + half;
      double r = __shfl_sync(kAll, half ? f1 : f0, l);
      uint32_t seen = __shfl_sync(kAll, half ? e1 : e0, l);
      for (int i = g * group; i < min(steps, (g + 1) * group) && v0 + i * 256 < v1 && !hit; i++) {
        Step<T, MODE> x;
        const int first = v0 + i * 256;
        x.load(row, first, lane, v1);
        double w[8], sum = 0.0, front = 0.0;
        if constexpr (MODE == kVectors) {  // a lane's labels lie in a row
          uint32_t n = 0;
#pragma unroll
          for (int e = 0; e < 8; e++) n += limited && O::of(x.z(e)) == low;
          uint32_t rank = n;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const uint32_t t = __shfl_up_sync(kAll, rank, d);
            if (lane >= d) rank += t;
          }
          const uint32_t all = __shfl_sync(kAll, rank, 31);
          rank += seen - n;
          seen += all;
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float z = x.z(e);
            const uint32_t o = O::of(z);
            const double q = weight.of(z);
            w[e] = (o > low && enough(q, z)) ? q : limited && o == low && rank < ties ? w_low : 0.0;
            rank += limited && o == low;
            sum += w[e];
          }
          front = sum;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const double t = __shfl_up_sync(kAll, front, d);
            if (lane >= d) front += t;
          }
          const double all_sum = __shfl_sync(kAll, front, 31);
          front = __shfl_up_sync(kAll, front, 1);
          double q = r + (lane ? front : 0.0);
#pragma unroll
          for (int e = 0; e < 8; e++) {
            q += w[e];
            if (w[e] > 0.0) {
              const uint32_t v = first + lane * 8 + e;
              last = max(last, v + 1);
              if (q > want) hit = max(hit, ~v);
            }
          }
          r += all_sum;
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float z = x.z(e);
            const uint32_t o = O::of(z), b = __ballot_sync(kAll, limited && o == low);
            const double q = weight.of(z);
            w[e] = (o > low && enough(q, z)) ? q : (b >> lane & 1) && seen + __popc(b & ((1u << lane) - 1)) < ties ? w_low : 0.0;
            seen += __popc(b);
            sum = w[e];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
              const double t = __shfl_up_sync(kAll, sum, d);
              if (lane >= d) sum += t;
            }
            if (w[e] > 0.0) {
              const uint32_t v = first + e * 32 + lane;
              last = max(last, v + 1);
              if (r + sum > want) hit = max(hit, ~v);
            }
            r += __shfl_sync(kAll, sum, 31);
          }
        }
        hit = __reduce_max_sync(kAll, hit);
      }
    }
    last = __reduce_max_sync(kAll, last);
    // by their sums the groups hold the draw, though running sums added in another order stay under it
    if (!hit && s.u < 1.0 && last) hit = ~(last - 1);
  }
  hit = team.most(hit);
  if (hit) return (int)~hit - row.shift;
  return (int)team.most(last) - 1 - row.shift;
}

template <int W, typename T, int MODE>
__global__ void __launch_bounds__(32 * W, W == 8 ? 4 : 2) sample_long_kernel(const __grid_constant__ SampleArgs a) {
  using O = Order<T>;
  __shared__ LongShared<W> sh;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, V = a.V;
  Team<W> team{sh.team, warp, lane};
  // a warp's part of the row: whole steps of 256
  const int part = (int)part_of<W, T>(V);
  const int steps = part / 256, group = (steps + kSums - 1) / kSums;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const Row<T, MODE> r(a, row);
    const Setting s = setting_of(a, row);
    RowNote& note = ((RowNote*)a.scratch)[row];
    const int v0 = min(r.end, warp * part), v1 = min(r.end, v0 + part);
    int* const candidates = list_of(a, row) + warp * kListWarp;
    const bool greedy = !(s.t > 0.0), top_k = !greedy && s.k > 0 && s.k < V, top_p = !greedy && !top_k && s.p < 1.0;
    const bool list = greedy || top_k || top_p || s.m > 0.0;
    const float scale = (float)s.scale;

    // the sample: two steps of each warp
    float ref = -INFINITY, low = INFINITY;
    const auto each_sample = [&](auto f) {
#pragma unroll 1
      for (int h = 0; h < kSample / 16; h++) {
        Step<T, MODE> x[2];
#pragma unroll
        for (int i = 0; i < 2; i++) x[i].load(r, v0 + (2 * h + i) * max(1, steps / (kSample / 8)) * 256, lane, v1);
#pragma unroll
        for (int i = 0; i < 16; i++) f(x[i / 8].z(i % 8));
      }
    };
    each_sample([&](float z) {
      ref = fmaxf(ref, z);
      if (z > -INFINITY) low = fminf(low, z);
    });
    ref = O::value(max(team.most(O::of(ref)), O::of(-INFINITY)));
    const bool workable = plain_scale(s, ref) || (greedy && fabsf(ref) < INFINITY);

    const float ref_scaled = __fmul_rn(ref, scale);  // its rounding is a factor of all weights alike, up to 0.3% (plain_scale)

    // one pass over the row, for sums of the weights beside 2^(ref scale), or for the labels from `guess` on
    float best = -INFINITY;
    int n = 0;
    double sum = 0.0;
    const auto pass = [&](auto wants_list, auto wants_best, auto wants_groups, float guess) {
      constexpr bool kList = decltype(wants_list)::value, kBest = decltype(wants_best)::value, kGroups = decltype(wants_groups)::value;
      // the type's last value that is not above the guess
      T under = from_f<T>(guess);
      if constexpr (std::is_same<T, __half>::value) under = __float2half_rd(guess);
      if constexpr (std::is_same<T, __nv_bfloat16>::value) under = __float2bfloat16_rd(guess);
      [[maybe_unused]] const uint32_t guess2 = sizeof(T) == 4 ? 0 : pair_bits(under, under);
      constexpr int kBatch = sizeof(T) == 4 ? 2 : 4;  // steps whose loads are in flight together
      float group_sum = 0.0f;
      int left = group, g = 0;
      for (int first0 = v0; first0 < v1; first0 += kBatch * 256) {
        Step<T, MODE> batch[kBatch];
        if (MODE == kVectors && first0 >= Step<T, MODE>::kPer && first0 + kBatch * 256 <= v1) {
#pragma unroll
          for (int j = 0; j < kBatch; j++) batch[j].load_whole(r, first0 + j * 256, lane);
        } else {
#pragma unroll
          for (int j = 0; j < kBatch; j++) batch[j].load(r, first0 + j * 256, lane, v1);
        }
#pragma unroll
        for (int j = 0; j < kBatch; j++) {  // steps behind the end hold -inf
          const int first = first0 + j * 256;
          const Step<T, MODE>& x = batch[j];
          if (kBest) best = x.most(best);
          if constexpr (!kList) {
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = exp2_fast(fmaf(x.z(e), scale, -ref_scaled));
            const float v = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
            if constexpr (kGroups) {
              group_sum += v;
              if (--left == 0 || first + 256 >= v1) {
#pragma unroll
                for (int o = 16; o; o >>= 1) group_sum += __shfl_xor_sync(kAll, group_sum, o);
                if (lane == 0 && g < kSums) sh.sums[warp][g] = group_sum;
                if (lane == 0) sum += group_sum;
                g++;
                group_sum = 0.0f;
                left = group;
              }
            } else {
              sum += v;
            }
          } else if constexpr (MODE == kVectors) {
            uint32_t in = x.at_least(guess, guess2);
            const uint32_t lanes = __ballot_sync(kAll, in);
            if (!lanes) continue;
            if (!__any_sync(kAll, in & (in - 1))) {
              const int to = n + __popc(lanes & ((1u << lane) - 1));
              n += __popc(lanes);
              if (in && to < kListWarp) candidates[to] = first + lane * 8 + __ffs(in) - 1;
              continue;
            }
            const int mine = __popc(in);
            int scan = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
              const int t = __shfl_up_sync(kAll, scan, d);
              if (lane >= d) scan += t;
            }
            int to = n + scan - mine;
            n += __shfl_sync(kAll, scan, 31);
            for (; in && to < kListWarp; in &= in - 1) candidates[to++] = first + lane * 8 + __ffs(in) - 1;
          } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const bool in = x.z(e) >= guess;
              const uint32_t b = __ballot_sync(kAll, in);
              if (!b) continue;
              const int to = n + __popc(b & ((1u << lane) - 1));
              n += __popc(b);
              if (to < kListWarp && in) candidates[to] = first + e * 32 + lane;
            }
          }
        }
      }
      if (!kList) {
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
      }
    };
    double all = -1.0, slack = 0.0, before = 0.0;  // all: the row's mass, known to the slack
    if (!workable) {                               // infinite, or nothing seen yet
      each_of_row<W, T, MODE>(r, warp, lane, [&](float z) {
        best = max_nan(best, z);
      });
    } else if (!list || top_p) {
      if (list) pass(std::false_type(), std::true_type(), std::false_type(), INFINITY);
      else pass(std::false_type(), std::true_type(), std::true_type(), INFINITY);
      team.ahead(sum, before, all);
    }
    // The type's lowest finite value, and the least guess: a place behind the row's ends holds -inf, as does a label that cannot
    // be kept, and neither is a candidate (a list of places that hold no label would be read past the row).
    constexpr float kLowest = sizeof(T) == 4 ? -FLT_MAX : std::is_same<T, __half>::value ? -65504.0f : -0x1.fep127f;
    float tail = 0.75f;  // top-p: of the share that is not kept, what may lie under the guess
    int tries = 2;
    while (workable && list) {
      // the guess: from where on candidates are kept
      float guess = ref;
      if (top_k || top_p) {
        low = -O::value(max(team.most(O::of(-low)), O::of(-INFINITY)));
        const float range = top_k ? ref - low : fminf(ref - low, 40.0f / scale), width = range * (1.0f / kBins);
        for (int i = threadIdx.x; i < kBins; i += (32 * W)) sh.bins[i] = 0;
        __syncthreads();
        const float to_bin = width > 0.0f ? 1.0f / width : 0.0f;
        each_sample([&](float z) {
          if (z > -INFINITY) atomicAdd(&sh.bins[(int)fminf((ref - z) * to_bin, (float)(kBins - 1))], 1u);
        });
        __syncthreads();
        if (warp == 0) {
          const float share = fminf(1.0f, (float)(32 * W * kSample) / (float)V);
          // top-k: the rank in the sample that the row's k-th is hardly ever behind.  top-p: as much of the tail as leaves some
          // of what is not kept, beside the whole mass; the tail's small weights are sampled well
          const float mean = (float)s.k * share, want = top_k ? mean + 4.0f * sqrtf(mean) + 2.0f : tail * (1.0f - (float)fmax(s.p, 0.0)) * (float)all * share;
          float c[8], mine = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int b = lane * 8 + i;
            mine += c[i] = (float)sh.bins[b] * (top_k ? 1.0f : exp2_fast(-(b + 0.5f) * width * scale));
          }
          float run = mine;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const float t = __shfl_up_sync(kAll, run, d);
            if (lane >= d) run += t;
          }
          const float total = __shfl_sync(kAll, run, 31);
          run -= mine;
          int bin = kBins;  // the first bin that, with those in front of it, is enough
#pragma unroll
          for (int i = 7; i >= 0; i--) {
            float front = run;
#pragma unroll
            for (int j = 0; j <= i; j++) front += c[j];
            if (top_k ? front >= want : total - front <= want) bin = lane * 8 + i;
          }
          bin = __reduce_min_sync(kAll, bin);
          if (lane == 0) sh.guess = bin >= kBins - 1 ? -INFINITY : ref - (bin + 1) * width;
        }
        __syncthreads();
        guess = sh.guess;
      } else if (!greedy) {
        guess = ref + (float)(log2_min_p(a, s) / s.scale) * (1.0f + 1e-5f) - 1e-6f * fabsf(ref);
      }
      guess = fmaxf(guess, kLowest);
      n = 0;
      if (top_p) pass(std::true_type(), std::false_type(), std::false_type(), guess);
      else pass(std::true_type(), std::true_type(), std::false_type(), guess);
      if (!top_p || --tries == 0 || guess == kLowest) break;
      // more of the tail, if what is held is not enough
      __syncwarp();
      double m = 0.0;
      for (int i = lane; i < min(n, kListWarp); i += 32) m += exp2_fast(fmaf(r.at(candidates[i]), scale, -ref_scaled));
      if (team.sum(m) > s.p * all * (1.0 + 1e-5)) break;
      tail = 0.3f;
    }
    const uint32_t top = team.most(best != best || s.t != s.t ? kAll : O::of(best));
    const uint32_t longest = team.most((uint32_t)n);
    int state = kDone, label = -1;
    if (top != kAll && O::value(top) > -INFINITY) {
      best = O::value(top);
      state = kWhole;
      if (workable && list) {
        if (longest <= kListWarp && fabsf(best) < INFINITY) state = kFromList;
      } else if (workable && !list && (best - ref) * scale < 8.0f) {
        // both sums, up to the draw and u times the whole, are u times the whole or so; that part's mean exponent is at most
        // log2 V - log2 u
        const double want = s.u * all;
        slack = (want + 1e-6 * all) * (a.margin + (fmax(0.0, (double)(best - ref) * s.scale) - 0.5 * log2f(fmaxf((float)s.u, 1e-6f))) * a.margin_far);
        if (threadIdx.x == 0) sh.answer = kUnsure;
        __syncthreads();
        if (want > slack && all - want > slack && before <= want && before + sum > want) {
          // this warp's part holds the draw: its group, then its label
          const int groups = (steps + group - 1) / group;
          int g = 0;
          double run = before;
          while (g < groups - 1 && run + sh.sums[warp][g] <= want) run += sh.sums[warp][g++];
          int found = -1;
          bool near = fabs(run - want) <= slack;
          for (int i = g * group; i < min(steps, (g + 1) * group) && found < 0; i++) {
            Step<T, MODE> x;
            const int first = v0 + i * 256;
            x.load(r, first, lane, v1);
            // running sums in index order
            uint32_t hit = 0;
            if constexpr (MODE == kVectors) {
              float w[8], mine = 0.0f;
#pragma unroll
              for (int e = 0; e < 8; e++) mine += w[e] = exp2_fast(fmaf(x.z(e), scale, -ref_scaled));
              float scan = mine;
#pragma unroll
              for (int d = 1; d < 32; d <<= 1) {
                const float t = __shfl_up_sync(kAll, scan, d);
                if (lane >= d) scan += t;
              }
              double q = run + (double)(scan - mine);
#pragma unroll
              for (int e = 0; e < 8; e++) {
                q += w[e];
                near |= fabs(q - want) <= slack && w[e] > 0.0f;
                if (!hit && q > want) hit = ~(uint32_t)(lane * 8 + e);
              }
              run += (double)__shfl_sync(kAll, scan, 31);
            } else {
#pragma unroll
              for (int e = 0; e < 8; e++) {
                const float w = exp2_fast(fmaf(x.z(e), scale, -ref_scaled));
                float scan = w;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                  const float t = __shfl_up_sync(kAll, scan, d);
                  if (lane >= d) scan += t;
                }
                const double q = run + (double)scan;
                near |= fabs(q - want) <= slack && w > 0.0f;
                if (!hit && q > want) hit = ~(uint32_t)(e * 32 + lane);
                run += (double)__shfl_sync(kAll, scan, 31);
              }
            }
            hit = __reduce_max_sync(kAll, hit);
            if (hit) found = first + (int)~hit;
          }
          near = __any_sync(kAll, near);
          if (lane == 0 && found >= 0 && !near) sh.answer = found - r.shift;
        }
        __syncthreads();
        label = sh.answer;
        if (label != kUnsure) state = kDone;
      }
    }
    if (threadIdx.x == 0) {
      a.label[row] = label;
      note.state = state, note.best = best, note.ref = ref, note.all = all;
    }
    if (lane == 0) note.n[warp] = n;
    __syncthreads();
  }
}

// What the passes left open: the draw from a row's candidates, or from the whole row.  Apart from the passes, so that
// the draws of many rows, whose steps wait for one another, run side by side.  W: warps of the passes.
template <int W, typename T, int MODE>
__global__ void __launch_bounds__(32 * W, W == 8 ? 4 : 1) sample_held_kernel(const __grid_constant__ SampleArgs a) {
  __shared__ LongShared<W> sh;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  Team<W> team{sh.team, warp, lane};
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const RowNote& note = ((const RowNote*)a.scratch)[row];
    if (note.state == kDone) continue;
    const Row<T, MODE> r(a, row);
    const int* const candidates = list_of(a, row);
    const Setting s = setting_of(a, row);
    const bool greedy = !(s.t > 0.0), top_k = !greedy && s.k > 0 && s.k < a.V, top_p = !greedy && !top_k && s.p < 1.0;
    const float best = note.best;
    int label = kUnsure;
    if (note.state == kFromList) {
      int before = 0, held = 0, longest = 0;
#pragma unroll
      for (int i = 0; i < W; i++) {
        if (i == warp) before = held;
        held += note.n[i];
        longest = max(longest, note.n[i]);
      }
      double all = -1.0, slack = 0.0;  // all: the row's mass, known to the slack
      if (top_p) {
        // the passes' weights are beside 2^ref_scaled, as rounded there; here they are beside the largest's
        const float scale = (float)s.scale, ref_scaled = __fmul_rn(note.ref, scale);
        const double far = fmax(0.0, (double)(best - note.ref) * s.scale), up = exp2((double)ref_scaled - (double)best * (double)scale);
        all = note.all * up;
        slack = 0.5 * all * (a.margin + far * a.margin_far);
        if (!(far < 8.0)) all = INFINITY;  // the sum in float32 counts on a sample that comes near the largest
      }
      for (int again = 0; again < 2 && (!top_k || held >= s.k); again++) {
        if (held <= kFew) {  // one warp, which exchanges without barriers
          for (int i = lane; i < note.n[warp]; i += 32) sh.few[before + i] = candidates[warp * kListWarp + i];
          __syncthreads();
          if (warp == 0) {
            constexpr int E = kFew / 32;
            float z[E];
#pragma unroll
            for (int e = 0; e < E; e++) z[e] = e * 32 + lane < held ? r.at(sh.few[e * 32 + lane]) : -INFINITY;
            Team<1> one{sh.team, 0, lane};
            const int at = draw<T, E, 1>(one, z, best, s, a.V, all, slack);
            if (lane == 0) sh.answer = at < 0 ? at : sh.few[at] - r.shift;
          }
          __syncthreads();
          label = sh.answer;
        } else {
          const auto from_list = [&](auto places) {
            constexpr int E = decltype(places)::value;
            const int n = note.n[warp];
            float z[E];
#pragma unroll
            for (int e = 0; e < E; e++) z[e] = e * 32 + lane < n ? r.at(candidates[warp * kListWarp + e * 32 + lane]) : -INFINITY;
            const int at = draw<T, E, W>(team, z, best, s, a.V, all, slack);
            label = at < 0 ? at : candidates[at / (32 * E) * kListWarp + at % (32 * E)] - r.shift;
          };
          if (longest <= 32 * kHeld / 2) from_list(std::integral_constant<int, kHeld / 2>());
          else from_list(std::integral_constant<int, kHeld>());
        }
        if (label != kUnsure || !(slack > 0.0)) break;
        const Weight weight(best, s.scale);  // the mass again, in 64 bits
        double m = 0.0;
        each_of_row<W, T, MODE>(r, warp, lane, [&](float z) { m += weight.of(z); });
        all = team.sum(m);
        slack = 0.0;
      }
    }
    if (label == kUnsure) label = whole_row<W, T, MODE>(team, sh, r, a.V, best, s);
    if (threadIdx.x == 0) a.label[row] = label;
    __syncthreads();
  }
}

// More than 48 KB of shared memory for a kernel, once a device.
template <auto kernel>
cudaError_t allow_shared(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (rc == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return rc;
}

int long_warps(int64_t M, int sms) { return M <= sms ? 16 : 8; }

template <typename T>
cudaError_t launch(const SampleArgs& a, int sms, cudaStream_t s) {
  SampleArgs b = a;
  b.scale_all = kLog2e64 / a.temperature_all;
  b.cut_all = a.min_p_all > 0.0 ? log2(a.min_p_all) / b.scale_all : 0.0;
  b.log2_min_p_all = a.min_p_all > 0.0 ? log2(a.min_p_all) : 0.0;
  int bits = 1;
  while ((1ll << bits) < a.V) bits++;
  // twice the error, relative to the whole sum, of a running sum in float32 and of u times the sum.  exp2 is off by 2^-22 of a weight; its
  // argument by three half steps, 3 ln 2 = 2.1 times 2^-24 |t| of the weight, where |t| counts with the weights: at most as
  // log2 V (the entropy), and twice the distance to the largest where that was not known; additions by 2^-24 each.
  const auto margin = [&](double chain, double extra) {
    return (float)(2.0 * (0x1p-22 + 2.1 * 0x1p-24 * (bits + extra) + (chain + 4) * 0x1p-24));
  };
  const auto run = [&](auto* kernel, int64_t units, int threads, int per_sm) {
    kernel<<<(unsigned)std::min<int64_t>(units, (int64_t)sms * per_sm), threads, 0, s>>>(b);
    return cudaPeekAtLastError();
  };
  const bool image = a.z.rs == 1 && a.z.cs != 1 && a.M > 1;
  if (image && a.V <= 1024 && !a.top_k && !a.top_p && (a.top_k_all <= 0 || a.top_k_all >= a.V) && a.top_p_all >= 1.0) {
    b.margin = margin((a.V + kPieces - 1) / kPieces + kPieces, 0);
    constexpr int PX = 4 / (int)sizeof(T);
    if (a.V <= kTileLabels && a.z.cs * (int64_t)sizeof(T) % 16 == 0 && (uintptr_t)a.z.p % 16 == 0 && a.z.cs >= a.M) {
      CUtensorMap map;
      EncodeFn fn = encode_fn();
      const cuuint64_t dims[3] = {(cuuint64_t)a.M, (cuuint64_t)a.V, 1}, strides[2] = {(cuuint64_t)a.z.cs * sizeof(T), (cuuint64_t)a.z.cs * sizeof(T)};
      const cuuint32_t box[3] = {(cuuint32_t)(kTileThreads * PX), (cuuint32_t)a.V, 1}, unit[3] = {1, 1, 1};
      b.status = status_word();
      const char* test = getenv("VI_HEADS_TEST_TIMEOUT");
      b.withhold = test && test[0] == '1';
      b.lapse = test && test[0] == '2';
      b.wait_limit = b.withhold || b.lapse ? 1 << 20 : kWaitLimit;
      if (fn && b.status &&
          fn(&map, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(a.z.p), dims, strides, box,
             unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS) {
        const int pieces = (a.V + 15) / 16;
        const int smem = pieces * (16 + PX) * kTileThreads * 4;
        b.margin = margin(8 + 2 + 16 + 16, 0);
        cudaError_t rc = cudaSuccess;
        if (smem > 48 * 1024) rc = allow_shared<sample_tiles_kernel<T>>(kTileLabels / 16 * (16 + PX) * kTileThreads * 4);
        if (rc != cudaSuccess) return rc;
        const int64_t tiles = (a.M + kTileThreads * PX - 1) / (kTileThreads * PX);
        const int per_sm = std::min(16, 220 * 1024 / (smem + 1100));
        sample_tiles_kernel<T><<<(unsigned)std::min<int64_t>(tiles, (int64_t)sms * per_sm), kTileThreads, smem, s>>>(map, b);
        return cudaPeekAtLastError();
      }
    }
    if constexpr (sizeof(T) == 2)
      if (a.M % 2 == 0 && a.z.cs % 2 == 0 && (uintptr_t)a.z.p % 4 == 0)
        return run(sample_image_kernel<T, 2>, (a.M + 2 * kImageThreads - 1) / (2 * kImageThreads), kImageThreads, 64);
    return run(sample_image_kernel<T, 1>, (a.M + kImageThreads - 1) / kImageThreads, kImageThreads, 64);
  }
  if (a.V <= 256) {
    b.margin = margin(8 + 5, 0);
    return run(sample_rows_kernel<T, 8, 1>, (a.M + 7) / 8, 256, 64);
  }
  b.margin = margin(16 + 5 + 8, 0);
  if (a.V <= 1024) return run(sample_rows_kernel<T, 16, 2>, a.M, 64, 64);
  if (a.V <= 4096) return run(sample_rows_kernel<T, 16, 8>, a.M, 256, 16);
  if (a.V <= kRowLabels) return run(sample_rows_kernel<T, 16, 16>, a.M, 512, 8);
  // few rows: more warps for each
  const auto rows = [&](auto warps) {
    constexpr int W = decltype(warps)::value;
    const int64_t steps = part_of<W, T>(a.V) / 256, group = (steps + kSums - 1) / kSums;
    b.margin = margin((double)group + 3 + 5 + 3, 0);
    b.margin_far = (float)(2.0 * 2.0 * 2.1 * 0x1p-24);
    b.list_at = a.M * (int64_t)sizeof(RowNote);
    b.list_bytes = list_bytes(W);
    const auto both = [&](auto mode) {
      constexpr int MODE = decltype(mode)::value;
      const cudaError_t rc = run(sample_long_kernel<W, T, MODE>, a.M, 32 * W, W == 8 ? 4 : 2);
      return rc == cudaSuccess ? run(sample_held_kernel<W, T, MODE>, a.M, 32 * W, W == 8 ? 16 : 2) : rc;
    };
    return a.z.cs == 1 ? both(std::integral_constant<int, kVectors>()) : both(std::integral_constant<int, kStrided>());
  };
  return long_warps(a.M, sms) == 16 ? rows(std::integral_constant<int, 16>()) : rows(std::integral_constant<int, 8>());
}

}  // namespace

uint64_t sample_scratch(int64_t M, int64_t V, int sms) {
  return V <= kRowLabels ? 0 : (uint64_t)M * (sizeof(RowNote) + list_bytes(long_warps(M, sms)));
}
cudaError_t launch_sample(int dtype, const SampleArgs& a, int sms, cudaStream_t s) {
  return dtype == VI_F32 ? launch<float>(a, sms, s) : dtype == VI_F16 ? launch<__half>(a, sms, s) : launch<__nv_bfloat16>(a, sms, s);
}

}  // namespace heads
}  // namespace vi
