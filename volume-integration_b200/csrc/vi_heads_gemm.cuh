// The heads' matrix product on the tensor cores, acc(m, n) = sum_k A(m, k) B(n, k),
// with its epilogues.
//
// Persistent blocks.  One warp copies 64-wide blocks of k of both operands into a ring
// of shared-memory stages (cp.async.bulk.tensor, 128-byte swizzle), one issues
// tcgen05.mma on them (128 x BN x 16, or 256 x 256 x 16 by a pair of blocks, float32 accumulators in tensor memory), 8 or 16
// take finished accumulators out of tensor memory and run the epilogue.  Two accumulators alternate, so the epilogue of one tile
// overlaps the product of the next.  Either operand may have k or its rows
// contiguous: both are layouts the tensor core reads, so a backward product
// transposes nothing.
//
// float32 operands come as three bfloat16 planes, x = x0 + x1 + x2.  Of the nine
// products of planes the six with i + j <= 2 are summed; the others are below 2^-24
// of |x||w|.  x0 w0 has an accumulator of its own and the five small products share
// another, added to it in the epilogue: the tensor core cuts an addend's bits below the
// accumulator's, and small ones cut 5 times as often cost ten times the error (5001 x 515 ->
// 257: 3.3e-6 in one accumulator, 3e-7 in two).
//
// A sum longer than a chain (chain_blocks) is made of several accumulations, added up in tensor memory by the
// epilogue's warps.  A float32 product's error is then 7.5e-7 of it at any K (in one accumulation 1.6e-6 at 1536 terms, 3.9e-5 at
// 32768; terms of one sign 1.4e-6, 1.6e-4); 16384 x 4096 -> 1024 takes 730 us (707), the statistics of 4096 x 1024,
// V = 8192, 380 (360).
//
// 8-bit integers (kEpiInt8) take the same bytes through the same ring: a block of k is 128 of them, a product 32, and the
// sums are exact in 32-bit integers.
//
// Every wait is bounded; one that runs out ends the block's work, drains what it
// has in flight, and is latched in a status word (VI_DEVICE_HEAD_TIMEOUT).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdio>
#include <cstdlib>
#include <type_traits>

#include "vi_heads.h"
#include "vi_heads_math.cuh"
#include "vi_heads_tma.cuh"
#include "vi_internal.h"

namespace vi {
namespace heads {
namespace {

constexpr int kBM = 128, kBK = 64;
// Terms of a block of k: 128 bytes of a row.
__host__ __device__ constexpr int block_terms(int epi) { return epi == kEpiInt8 ? 128 : kBK; }

// Narrow tiles belong to products that memory bounds (few columns, short sums): two
// blocks per SM, so that one's epilogue runs while the other waits for memory.  A
// 256-wide tile takes all tensor memory (two accumulators) and its SMs for itself.
// PL planes of both operands share a stage, so that the six products of float32's are made of
// each copied block once.
template <typename T, int BN, int EPI, int PL>
struct Shape {
  static_assert(PL == 1 || BN <= 128, "three planes of a 256-wide tile leave no second stage");
  // 256-wide tiles are 256 rows high and made by two blocks on neighbouring SMs (cta_group::2): each copies
  // its 128 rows of A and half of B, which the other's tensor core reads too
  static constexpr bool kPair = pair_tile(EPI, BN);
  static constexpr int kBlocks = BN == 256 || PL == 3 ? 1 : 2;
  // Epilogue warps.  The softmax on a 256-wide tile has 16: with 8 its latency, not its
  // instructions, bound it (K = 256: gradient 289 us with 8, 230 with 16; statistics 207, 159).
  // So do the 8-bit products, whose sums are made twice as fast (32768 x 1024 -> 4096: 185 us with 8).
  static constexpr int kWarps = BN == 256 && (EPI == kEpiLse || EPI == kEpiGrad || EPI == kEpiInt8) ? 16 : 8;
  static constexpr int kParts = kWarps / 4;  // warps that share a tile's columns, 32 at a time
  static constexpr int kThreads = (kWarps + 2) * 32;
  static constexpr int kTileA = kBM * kBK * 2, kTileB = BN / (kPair ? 2 : 1) * kBK * 2;  // bytes of a plane
  static constexpr int kStage = PL * (kTileA + kTileB);
  static constexpr int kStages = PL == 3   ? 2
                                 : BN == 256 ? (EPI == kEpiInt8 ? (sizeof(T) == 4 ? 4 : 5) : kPair ? 6 : 4)
                                 : BN == 128 ? (kBlocks == 2 ? 2 : 5)
                                             : (kBlocks == 2 ? 3 : 7);
  static constexpr int kStageWarp = EPI == kEpiLse ? 0 : 32 * 32 * (int)sizeof(T);  // an epilogue warp's staging
  // beside the stages each epilogue warp has its staging and 32 float32 of bias (kEpiInt8: and of scales)
  static constexpr int kSlot = EPI == kEpiInt8 ? 256 : 128;
  static constexpr int kBars = kStages * kStage + kWarps * (kStageWarp + kSlot);
  static constexpr int kSmem = kBars + (2 * kStages + 5) * 8 + 8;
  static_assert(kBlocks * (kSmem + 1024) <= 228 * 1024, "shared memory of an SM");
};

// n / d for 0 <= n < 2^31 by a multiplication: mul = ceil(2^(31 + s) / d), s = ceil(log2 d).
// The rounding of mul adds less than n / 2^31 / d to the quotient, which changes no floor.
struct FastDiv {
  uint32_t d, mul, shift;
  static FastDiv of(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) s++;
    return FastDiv{d, d == 1 ? 0u : (uint32_t)(((1ull << (31 + s)) + d - 1) / d), s ? s - 1 : 0};
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return d == 1 ? n : __umulhi(n, mul) >> shift; }
};

struct Args {
  int M, N;
  int m_tiles, n_tiles;  // n_tiles: column tiles
  int kblocks;           // 64-wide blocks of the whole sum
  int kps, splits;
  int chain;             // blocks of k that one accumulation takes (chain_blocks); 0: all of a piece's
  int span, spans;
  uint32_t idesc;        // instruction descriptor
  uint32_t a_lbo, b_lbo; // bytes >> 4
  uint32_t a_step, b_step;  // bytes >> 4 from one 16-wide slice of k to the next
  int a_k_major, b_k_major;
  int items;
  FastDiv per_split, per_group;  // items of one piece of the sum; of 16 row tiles
  FastDiv last_rows;             // row tiles of the last group
  int64_t wait_limit;    // cycles
  int withhold;          // testing hook: the first load is never issued
  uint32_t* status;      // gets VI_DEVICE_HEAD_TIMEOUT when a wait ran out
  Epilogue e;
};

// Address of the same shared-memory location in block `rank` of the cluster.
__device__ __forceinline__ uint32_t at_rank(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
// Relaxed: what the arrival announces is that tensor memory has been read (wait::ld, then the fence), and a
// release at cluster scope would wait for the stores to global memory too.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// Shared memory by its 32-bit address: a generic pointer would cost 64-bit arithmetic per access.
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint32_t lds_cell(uint32_t a, uint32_t) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint16_t lds_cell(uint32_t a, uint16_t) {
  uint16_t v;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts_cell(uint32_t a, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void sts_cell(uint32_t a, uint16_t v) {
  asm volatile("st.shared.b16 [%0], %1;" ::"r"(a), "h"(v) : "memory");
}

// Shared-memory matrix descriptor: address, leading and stride byte offsets (>> 4),
// version 1, 128-byte swizzle.  Stride: from one group of 8 rows (k contiguous) or of 8 k
// (rows contiguous) to the next, 1024 bytes.  Leading (rows contiguous): from one
// 64-row column of the tile to the next.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)lbo << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
template <bool PAIR>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (PAIR) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
    return;
  }
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 8-bit integers, 32 terms, sums in 32-bit integers.
template <bool PAIR>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (PAIR) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
    return;
  }
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives at the barrier (of both blocks of a pair) when the products issued so far have ended.
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (PAIR) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
    return;
  }
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 32 columns of this warp's 32 lanes of tensor memory.
__device__ __forceinline__ void tmem_load32(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
      "%24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_load8(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_store8(uint32_t addr, const float* v) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const float* v) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// Work item -> row tile, column tile (or span of them), piece of the sum.  Groups of 16 row
// tiles run through all columns before the next group, so the blocks that run
// together share operand tiles in L2.
struct Item {
  int mt, nt, nt_end, kb0, kb1, split, span;
};
template <int EPI>
__device__ __forceinline__ Item item_of(const Args& a, int i) {
  Item t;
  t.split = 0;
  if (EPI == kEpiPartial) {
    t.split = (int)a.per_split.div(i);
    i -= t.split * (int)a.per_split.d;
  }
  if (EPI != kEpiLse && a.n_tiles == 1) {
    t.mt = i;
    t.span = t.nt = 0;
    t.nt_end = 1;
    t.kb0 = t.split * a.kps;
    t.kb1 = min(a.kblocks, t.kb0 + a.kps);
    return t;
  }
  const int group = (int)a.per_group.div(i), r = i - group * (int)a.per_group.d;
  if (group * 16 + 16 <= a.m_tiles) {
    t.mt = group * 16 + (r & 15);
    t.span = r >> 4;
  } else {
    t.span = (int)a.last_rows.div(r);
    t.mt = group * 16 + r - t.span * (int)a.last_rows.d;
  }
  t.nt = EPI == kEpiLse ? t.span * a.span : t.span;
  t.nt_end = EPI == kEpiLse ? min(a.n_tiles, t.nt + a.span) : t.nt + 1;
  t.kb0 = t.split * a.kps;
  t.kb1 = min(a.kblocks, t.kb0 + a.kps);
  return t;
}

// ---- epilogue pieces ----
// Each works on 32 rows (one per lane) x 32 columns in registers.

// The stored type of act' beside T.
template <typename T>
using SlopeCell = typename std::conditional<sizeof(T) == 4, float, uint16_t>::type;

// 32 elements, one row of a warp's 32 x 32 tile.
template <typename Z>
union Row {
  static constexpr int kPieces = 2 * sizeof(Z);  // of 16 bytes
  using Bits = typename std::conditional<sizeof(Z) == 4, uint32_t, uint16_t>::type;
  uint4 q[kPieces];
  uint32_t w[8 * sizeof(Z)];
  Bits b[32];
  Z z[32];
  __device__ __forceinline__ Row() {}
};

// Values 2j and 2j + 1 of a row, rounded to T.
__device__ __forceinline__ void set_pair(Row<float>& r, int j, float2 v) {
  r.z[2 * j] = v.x;
  r.z[2 * j + 1] = v.y;
}
template <typename T>
__device__ __forceinline__ void set_pair(Row<T>& r, int j, float2 v) {
  r.w[j] = pack2(v, T());
}
template <typename T>
__device__ __forceinline__ float2 get_pair(const Row<T>& r, int j) {
  return make_float2(to_f(r.z[2 * j]), to_f(r.z[2 * j + 1]));
}

// A lane's places in its warp's staging, 32 lines of 32 elements.  The 16-byte pieces of a
// line are exchanged by the line's number, so that lanes writing a line each and lanes
// reading along lines both touch every bank once.
template <typename Z>
struct Stage {
  static constexpr int kLanes = Row<Z>::kPieces, kStep = 32 / kLanes, kPer = 16 / (int)sizeof(Z);  // lanes a line, lines a step
  static constexpr uint32_t kLine = 32 * sizeof(Z);
  static __device__ __forceinline__ uint32_t key(int line) { return (uint32_t)(sizeof(Z) == 4 ? line & 7 : (line >> 1) & 3) << 4; }
  // piece i of the lane's own line
  static __device__ __forceinline__ uint32_t own(uint32_t st, int lane, int i) {
    return st + lane * kLine + ((uint32_t)(i << 4) ^ key(lane));
  }
  // element j of a line
  static __device__ __forceinline__ uint32_t cell(uint32_t st, int line, int j) {
    return st + line * kLine + ((uint32_t)(j / kPer << 4) ^ key(line)) + j % kPer * (int)sizeof(Z);
  }
  // the lane's piece of its line of step i
  static __device__ __forceinline__ uint32_t along(uint32_t st, int lane, int i) {
    const int line = lane / kLanes + i * kStep;
    return st + line * kLine + ((uint32_t)((lane % kLanes) << 4) ^ key(line));
  }
};

// An image's tile: the column of the lane's line in step i.  16-bit elements are staged
// in pairs of columns, 4 bytes a row, so that a lane's 8 rows of a pair are two 16-byte
// pieces; odd pairs have them exchanged, so that 8 lanes touch every bank once.
template <typename Z>
__device__ __forceinline__ int image_column(int line, int i) {
  return sizeof(Z) == 4 ? line + i * 4 : 2 * (line + (i >> 1) * 8) + (i & 1);
}
__device__ __forceinline__ uint32_t image_line(int lane, int i) { return (lane / 4 + i * 8) * 128 + (lane % 4) * 32; }
__device__ __forceinline__ uint32_t image_half(int lane) { return (lane & 4) << 2; }

enum Access { kNone, kVector, kImage, kScalar };
// How a matrix is reached: columns contiguous on 16-byte rows, rows contiguous on 16-byte
// columns (an image), or any strides.
template <typename Z>
__device__ __forceinline__ int access_of(const View& v) {
  if (!v.p) return kNone;
  constexpr int per = 16 / (int)sizeof(Z);
  if ((uintptr_t)v.p & 15) return kScalar;
  return v.cs == 1 && v.rs % per == 0 ? kVector : v.rs == 1 && v.cs % per == 0 ? kImage : kScalar;
}

// A 32 x 32 tile of a matrix: its first element's row and column, and how many of its rows and
// columns exist (at least one each).
struct Place {
  int m0, n0;
  int rows, cols;
};

// Ragged ends and any strides: into the staging, and out of it.  A row at a time where columns are
// contiguous and many, else a column at a time, eight loads in flight.  Calls, not inlined: in the
// epilogue's code they cost the common case its registers (frame 203 us, 220).
template <typename Z>
__device__ __noinline__ void load_ragged(const typename Row<Z>::Bits* q, int64_t rs, int64_t cs, uint32_t st, int lane, int rows,
                                         int cols) {
  using Bits = typename Row<Z>::Bits;
  using G = Stage<Z>;
  const bool by_rows = cs == 1 && cols > 16;
  const int lines = by_rows ? rows : cols, along = by_rows ? cols : rows;
  const int64_t step = by_rows ? rs : cs;
  if (lane >= along) return;
  q += lane * (by_rows ? cs : rs);
#pragma unroll 1
  for (int l = 0; l < lines; l += 8) {
    Bits b[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (l + i < lines) b[i] = q[(l + i) * step];
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (l + i < lines) sts_cell(by_rows ? G::cell(st, l + i, lane) : G::cell(st, lane, l + i), b[i]);
  }
}
template <typename Z>
__device__ __noinline__ void store_ragged(typename Row<Z>::Bits* q, int64_t rs, int64_t cs, uint32_t st, int lane, int rows, int cols) {
  using Bits = typename Row<Z>::Bits;
  using G = Stage<Z>;
  const bool by_rows = cs == 1 && cols > 16;
  const int lines = by_rows ? rows : cols, along = by_rows ? cols : rows;
  const int64_t step = by_rows ? rs : cs;
  if (lane >= along) return;
  q += lane * (by_rows ? cs : rs);
#pragma unroll 4
  for (int l = 0; l < lines; l++, q += step) *q = lds_cell(by_rows ? G::cell(st, l, lane) : G::cell(st, lane, l), Bits());
}

// Loads a tile of v, 16 bytes a lane: along rows (kVector), along columns (kImage), or else
// element by element into the staging; own_row hands them to their rows' lanes.  Returns the way.
template <typename Z>
__device__ __forceinline__ int load_tile(Row<Z>& r, const View& v, int access, uint32_t st, int lane, const Place& t) {
  using G = Stage<Z>;
  const Z* p = (const Z*)v.p;
  const int line = lane / G::kLanes, piece = lane % G::kLanes;
  if (access == kVector && t.cols >= 32) {
    const Z* q = p + (int64_t)(t.m0 + line) * v.rs + t.n0 + piece * G::kPer;
    const int64_t step = G::kStep * v.rs;
#pragma unroll
    for (int i = 0; i < G::kLanes; i++, q += step)
      if (line + i * G::kStep < t.rows) r.q[i] = *(const uint4*)q;
    return kVector;
  }
  if (access == kImage && t.rows >= 32) {
    const Z* q = p + (int64_t)t.n0 * v.cs + t.m0 + piece * G::kPer;
#pragma unroll
    for (int i = 0; i < G::kLanes; i++) {
      const int c = image_column<Z>(line, i);
      if (c < t.cols) r.q[i] = *(const uint4*)(q + c * v.cs);
    }
    return kImage;
  }
  __syncwarp();
  load_ragged<Z>((const typename Row<Z>::Bits*)p + (int64_t)t.m0 * v.rs + (int64_t)t.n0 * v.cs, v.rs, v.cs, st, lane, t.rows, t.cols);
  return kScalar;
}
// What load_tile left along lines, to a row each, through the staging.
template <typename Z>
__device__ __forceinline__ void own_row(Row<Z>& r, int way, uint32_t st, int lane) {
  using G = Stage<Z>;
  __syncwarp();
  if (way != kImage) {
    if (way == kVector) {
#pragma unroll
      for (int i = 0; i < G::kLanes; i++) sts128(G::along(st, lane, i), r.q[i]);
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < G::kLanes; i++) r.q[i] = lds128(G::own(st, lane, i));
  } else if constexpr (sizeof(Z) == 4) {  // staged as columns of 32 rows; neighbouring lanes read neighbouring elements
#pragma unroll
    for (int i = 0; i < G::kLanes; i++) sts128(st + lane * 16 + i * 512, r.q[i]);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 32; j++) r.b[j] = lds_cell(st + lane * 4 + j * 128, 0u);
  } else {  // staged as pairs of columns of 32 rows
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const uint4 a = r.q[2 * i], b = r.q[2 * i + 1];
      const uint32_t at = st + image_line(lane, i);
      sts128(at + image_half(lane), make_uint4(__byte_perm(a.x, b.x, 0x5410), __byte_perm(a.x, b.x, 0x7632),
                                               __byte_perm(a.y, b.y, 0x5410), __byte_perm(a.y, b.y, 0x7632)));
      sts128(at + (image_half(lane) ^ 16), make_uint4(__byte_perm(a.z, b.z, 0x5410), __byte_perm(a.z, b.z, 0x7632),
                                                      __byte_perm(a.w, b.w, 0x5410), __byte_perm(a.w, b.w, 0x7632)));
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; j++) r.w[j] = lds_cell(st + j * 128 + ((lane * 4) ^ ((j & 1) << 4)), 0u);
  }
}

// Writes each lane's row to a tile of v, one of whose strides is 1.  The cell `fix` of the
// lane's row (none if negative; matrices with contiguous columns only) gets the value `with`.
template <typename Z>
__device__ __forceinline__ void store_tile(const Row<Z>& r, const View& v, int access, uint32_t st, int lane,
                                           const Place& t, int fix = -1, typename Row<Z>::Bits with = 0) {
  using G = Stage<Z>;
  Z* p = (Z*)v.p;
  const int line = lane / G::kLanes, piece = lane % G::kLanes;
  __syncwarp();
  if (access == kImage && t.rows >= 32) {
    Z* q = p + (int64_t)t.n0 * v.cs + t.m0 + piece * G::kPer;
    if constexpr (sizeof(Z) == 4) {
#pragma unroll
      for (int j = 0; j < 32; j++) sts_cell(st + lane * 4 + j * 128, r.w[j]);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < G::kLanes; i++) {
        const int c = image_column<Z>(line, i);
        if (c < t.cols) *(uint4*)(q + c * v.cs) = lds128(st + lane * 16 + i * 512);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; j++) sts_cell(st + j * 128 + ((lane * 4) ^ ((j & 1) << 4)), r.w[j]);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const uint32_t at = st + image_line(lane, i);
        const uint4 a = lds128(at + image_half(lane)), b = lds128(at + (image_half(lane) ^ 16));
        const int c = image_column<Z>(line, 2 * i);
        if (c < t.cols)
          *(uint4*)(q + c * v.cs) = make_uint4(__byte_perm(a.x, a.y, 0x5410), __byte_perm(a.z, a.w, 0x5410),
                                               __byte_perm(b.x, b.y, 0x5410), __byte_perm(b.z, b.w, 0x5410));
        if (c + 1 < t.cols)
          *(uint4*)(q + (c + 1) * v.cs) = make_uint4(__byte_perm(a.x, a.y, 0x7632), __byte_perm(a.z, a.w, 0x7632),
                                                     __byte_perm(b.x, b.y, 0x7632), __byte_perm(b.z, b.w, 0x7632));
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < G::kLanes; i++) sts128(G::own(st, lane, i), r.q[i]);
  if (fix >= 0) sts_cell(G::cell(st, lane, fix), with);
  __syncwarp();
  typename Row<Z>::Bits* q = (typename Row<Z>::Bits*)p + (int64_t)t.m0 * v.rs + (int64_t)t.n0 * v.cs;
  if (access == kVector && t.cols >= 32) {
    q += line * v.rs + piece * G::kPer;
    const int64_t step = G::kStep * v.rs;
#pragma unroll
    for (int i = 0; i < G::kLanes; i++, q += step)
      if (line + i * G::kStep < t.rows) *(uint4*)q = lds128(G::along(st, lane, i));
  } else {
    store_ragged<Z>(q, v.rs, v.cs, st, lane, t.rows, t.cols);
  }
}

__device__ __forceinline__ uint16_t bits_of(__half v) { return __half_as_ushort(v); }
__device__ __forceinline__ uint16_t bits_of(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }

__device__ __forceinline__ float2 unpack2(uint32_t w, __half) { return __half22float2(*(const __half2*)&w); }
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) { return __bfloat1622float2(*(const __nv_bfloat162*)&w); }

// Sum over the 32 rows of one column of the tile that store_tile has left in the staging: a lane adds 4 rows of
// 8 columns, then lanes hand halves of their columns to each other.  Which column: `column`.
template <typename T>
__device__ __forceinline__ float staged_column_sum(uint32_t st, int lane, int& column) {
  using G = Stage<T>;
  float2 s[4] = {pair(0.0f), pair(0.0f), pair(0.0f), pair(0.0f)};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint4 q = lds128(G::along(st, lane, i));
    s[0] = __fadd2_rn(s[0], unpack2(q.x, T()));
    s[1] = __fadd2_rn(s[1], unpack2(q.y, T()));
    s[2] = __fadd2_rn(s[2], unpack2(q.z, T()));
    s[3] = __fadd2_rn(s[3], unpack2(q.w, T()));
  }
  float t[8] = {s[0].x, s[0].y, s[1].x, s[1].y, s[2].x, s[2].y, s[3].x, s[3].y};
  column = (lane % 4) * 8;
#pragma unroll
  for (int h = 4; h; h /= 2) {
    const bool up = lane & (4 * h);
    if (up) column += h;
#pragma unroll
    for (int j = 0; j < h; j++) {
      const float give = up ? t[j] : t[j + h], keep = up ? t[j + h] : t[j];
      t[j] = keep + __shfl_xor_sync(0xffffffffu, give, 4 * h);
    }
  }
  return t[0];
}

// A long sum's accumulations are added up here, rounded: 32 columns of this warp's lanes from `acc` to `total` (the
// first, to them), COLS at a time.
template <int COLS>
__device__ __forceinline__ void fold_chain(uint32_t total, uint32_t acc, bool first) {
  static_assert(COLS == 8 || COLS == 16, "columns");
#pragma unroll
  for (int c = 0; c < 32; c += COLS) {
    float2 v[COLS / 2], u[COLS / 2];
    if constexpr (COLS == 16) {
      tmem_load16(acc + c, (float*)v);
      if (!first) tmem_load16(total + c, (float*)u);
    } else {
      tmem_load8(acc + c, (float*)v);
      if (!first) tmem_load8(total + c, (float*)u);
    }
    tmem_wait_load();
    if (!first) {
#pragma unroll
      for (int j = 0; j < COLS / 2; j++) v[j] = __fadd2_rn(v[j], u[j]);
    }
    if constexpr (COLS == 16) tmem_store16(total + c, (float*)v);
    else tmem_store8(total + c, (float*)v);
  }
  tmem_wait_store();
}
// Where two blocks share an SM, a call of few registers.
__device__ __noinline__ void fold_chain_call(uint32_t total, uint32_t acc, bool first) { fold_chain<8>(total, acc, first); }

// v += COLS values of a bias slot.
template <int COLS>
__device__ __forceinline__ void add_bias(uint32_t slot, float2* v) {
#pragma unroll
  for (int i = 0; i < COLS / 4; i++) {
    const uint4 q = lds128(slot + i * 16);
    v[2 * i] = __fadd2_rn(v[2 * i], make_float2(__uint_as_float(q.x), __uint_as_float(q.y)));
    v[2 * i + 1] = __fadd2_rn(v[2 * i + 1], make_float2(__uint_as_float(q.z), __uint_as_float(q.w)));
  }
}

// 16 sums in integers times the row's scale and a slot of columns' scales.
__device__ __forceinline__ void scale_sums(uint32_t slot, float row, float2* v) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint4 q = lds128(slot + i * 16);
    const float2 s0 = __fmul2_rn(make_float2(__uint_as_float(q.x), __uint_as_float(q.y)), pair(row));
    const float2 s1 = __fmul2_rn(make_float2(__uint_as_float(q.z), __uint_as_float(q.w)), pair(row));
    const float2 a = make_float2((float)__float_as_int(v[2 * i].x), (float)__float_as_int(v[2 * i].y));
    const float2 b = make_float2((float)__float_as_int(v[2 * i + 1].x), (float)__float_as_int(v[2 * i + 1].y));
    v[2 * i] = __fmul2_rn(a, s0);
    v[2 * i + 1] = __fmul2_rn(b, s1);
  }
}

// CHAIN: sums may be longer than a chain.
template <typename T, int BN, int EPI, int PL, int ACT, bool CHAIN>
__global__ void __launch_bounds__(Shape<T, BN, EPI, PL>::kThreads, Shape<T, BN, EPI, PL>::kBlocks)
    gemm_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ Args a) {
  using S = Shape<T, BN, EPI, PL>;
  constexpr int kStages = S::kStages, kStage = S::kStage, kEpiWarps = S::kWarps;
  constexpr int kAcc = PL == 3 ? 2 * BN : BN;   // tensor memory columns of an accumulator
  constexpr uint32_t kCols = 2 * kAcc;          // two of them alternate
  extern __shared__ __align__(1024) char smem[];
  uint64_t* bars = (uint64_t*)(smem + S::kBars);
  uint32_t* tmem_slot = (uint32_t*)(bars + 2 * kStages + 5);
  volatile int* dead = (int*)(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t full = smem_u32(bars), empty = full + 8 * kStages, tfull = empty + 8 * kStages, tempty = tfull + 16,
                 drain = tempty + 16;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; i++) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(tfull + 8 * i, 1);
      mbar_init(tempty + 8 * i, S::kPair ? 2 * kEpiWarps : kEpiWarps);
    }
    mbar_init(drain, 1);
    *dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kEpiWarps + 1) {
    if constexpr (S::kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  // a pair's blocks: rank 0 issues the products of both; its barriers count both blocks' copies and epilogues
  uint32_t rank = 0;
  if constexpr (S::kPair) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int first_item = S::kPair ? blockIdx.x / 2 : blockIdx.x, item_step = S::kPair ? gridDim.x / 2 : gridDim.x;
  fence_before();
  __syncwarp();
  if constexpr (S::kPair) cluster_sync();
  else __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == kEpiWarps) {
    // ---- loads ----
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int64_t issued = 0;
      bool on = true;
#pragma unroll 1
      for (int i = first_item; i < a.items && on; i += item_step) {
        const Item t = item_of<EPI>(a, i);
#pragma unroll 1
        for (int nt = t.nt; nt < t.nt_end && on; nt++) {
          const int row = S::kPair ? (2 * t.mt + (int)rank) * kBM : t.mt * kBM;
          const int column = S::kPair ? nt * BN + (int)rank * (BN / 2) : nt * BN;
#pragma unroll 1
          for (int kb = t.kb0; kb < t.kb1; kb++) {
            if (!mbar_wait(empty + 8 * stage, phase ^ 1, dead, a.wait_limit)) {
              on = false;
              break;
            }
            uint32_t bar = full + 8 * stage;
            if constexpr (S::kPair) bar = at_rank(bar, 0);
            uint32_t at = smem_u32(smem + stage * kStage);
            if (a.withhold && issued == 0) {  // this stage is never filled: its consumer's wait runs out
              issued++;
            } else {
              if (rank == 0) mbar_expect(full + 8 * stage, S::kPair ? 2 * kStage : kStage);
#pragma unroll
              for (int pl = 0; pl < PL; pl++) {
                if (a.a_k_major) {
                  tma_load<S::kPair>(at, &map_a, bar, kb * block_terms(EPI), row, pl);
                } else {
#pragma unroll
                  for (int j = 0; j < kBM / 64; j++)
                    tma_load<S::kPair>(at + j * 8192, &map_a, bar, row + j * 64, kb * block_terms(EPI), pl);
                }
                at += S::kTileA;
              }
#pragma unroll
              for (int pl = 0; pl < PL; pl++) {
                if (a.b_k_major) {
                  tma_load<S::kPair>(at, &map_b, bar, kb * block_terms(EPI), column, pl);
                } else {
#pragma unroll
                  for (int j = 0; j < BN / 64 / (S::kPair ? 2 : 1); j++)
                    tma_load<S::kPair>(at + j * 8192, &map_b, bar, column + j * 64, kb * block_terms(EPI), pl);
                }
                at += S::kTileB;
              }
              issued++;
            }
            if (++stage == kStages) stage = 0, phase ^= 1;
          }
        }
      }
      // every arrival that the products still owe this block's barriers (a pair's second block gets them from
      // the first) comes before the block leaves: the last release of every stage
#pragma unroll 1
      for (int j = 0; j < kStages && j < issued && on; j++) {
        const int64_t f = issued - 1 - j;
        on = mbar_wait(empty + 8 * (uint32_t)(f % kStages), (uint32_t)(f / kStages) & 1, dead, a.wait_limit);
      }
      if (*dead && rank == 0) {  // wait for the copies in flight (a pair's: both blocks'): the last fill of every stage
        for (int j = 0; j < kStages && j < issued; j++) {
          const int64_t f = issued - 1 - j;  // fill number: stage f % kStages, phase (f / kStages) & 1
          if (a.withhold && f == 0) continue;
          mbar_drain(full + 8 * (uint32_t)(f % kStages), (uint32_t)(f / kStages) & 1, a.wait_limit);
        }
      }
    }
  } else if (warp == kEpiWarps + 1) {
    // ---- products ----
    if (lane == 0 && rank == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool on = true;
#pragma unroll 1
      for (int i = first_item; i < a.items && on; i += item_step) {
        const Item t = item_of<EPI>(a, i);
        const int steps = t.kb1 - t.kb0;
#pragma unroll 1
        for (int nt = t.nt; nt < t.nt_end && on; nt++) {
          const int chain = CHAIN && a.chain ? a.chain : steps;
#pragma unroll 1
          for (int s0 = 0; s0 < steps; s0 += chain) {
            if (!mbar_wait(tempty + 8 * acc, acc_phase ^ 1, dead, a.wait_limit)) {
              on = false;
              break;
            }
            fence_after();
            const uint32_t d = tmem + acc * kAcc;
            const int s1 = min(steps, s0 + chain);
#pragma unroll 1
            for (int s = s0; s < s1; s++) {
              if (!mbar_wait(full + 8 * stage, phase, dead, a.wait_limit)) {
                on = false;
                break;
              }
              fence_after();
              const uint32_t sa = smem_u32(smem + stage * kStage), sb = sa + PL * S::kTileA;
              // planes of the six products, smallest first: (2,0) (1,1) (0,2) (1,0) (0,1) (0,0)
              constexpr int kPairs = PL == 3 ? 6 : 1;
#pragma unroll
              for (int p = 0; p < kPairs; p++) {
                const int pa = PL == 1 ? 0 : p == 0 ? 2 : p == 1 || p == 3 ? 1 : 0;
                const int pb = PL == 1 ? 0 : p == 2 ? 2 : p == 1 || p == 4 ? 1 : 0;
                const uint64_t da = smem_desc(sa + pa * S::kTileA, a.a_lbo), db = smem_desc(sb + pb * S::kTileB, a.b_lbo);
#pragma unroll
                for (int k = 0; k < kBK / 16; k++) {
                  if constexpr (EPI == kEpiInt8)
                    mma_i8<S::kPair>(d, da + k * a.a_step, db + k * a.b_step, a.idesc, s > s0 || k > 0);
                  else
                    mma_f16<S::kPair>(PL == 3 && p < 5 ? d + BN : d, da + k * a.a_step, db + k * a.b_step, a.idesc,
                                      s > s0 || (p > 0 && p < 5) || k > 0);
                }
              }
              mma_commit<S::kPair>(empty + 8 * stage);
              if (++stage == kStages) stage = 0, phase ^= 1;
            }
            if (!on) break;
            mma_commit<S::kPair>(tfull + 8 * acc);
            if ((CHAIN && a.chain) || ++acc == 2) acc = 0, acc_phase ^= 1;
          }
        }
      }
      if (*dead) {
        mma_commit<S::kPair>(drain);
        mbar_drain(drain, 0, a.wait_limit);
      }
    }
  } else {
    // ---- epilogue ----
    const int quad = warp % 4, part = warp / 4;
    const uint32_t st = smem_u32(smem + kStages * kStage) + warp * S::kStageWarp;
    const uint32_t bias_slot = smem_u32(smem + kStages * kStage) + kEpiWarps * S::kStageWarp + warp * S::kSlot;
    constexpr bool kAct = EPI == kEpiAct || EPI == kEpiInt8;
    int bias_at = -1;  // column the slot holds
    const Epilogue& e = a.e;
    const int out_access = access_of<T>(e.out), res_access = access_of<T>(e.res);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool on = true;
#pragma unroll 1
    for (int i = first_item; i < a.items && on; i += item_step) {
      const Item t = item_of<EPI>(a, i);
      const int m0 = (S::kPair ? 2 * t.mt + (int)rank : t.mt) * kBM + quad * 32, m = m0 + lane;
      const int rows = min(32, a.M - m0);
      auto place = [&](int n0) { return Place{m0, n0, rows, min(32, a.N - n0)}; };
      float top = -INFINITY, sum = 0.0f;
      int target = -1;  // its column, if it is one of these
      float lsum = 0.0f, coef = 0.0f, alpha = 1.0f, gtarget = 0.0f;
      if ((EPI == kEpiLse || EPI == kEpiGrad) && m < a.M) {
        const int64_t c = e.target[m] - (EPI == kEpiGrad ? e.col0 : 0);
        if (c >= 0 && c < a.N) target = (int)c;
      }
      if (EPI == kEpiGrad && m < a.M) {
        top = e.lse[m], lsum = e.lse[a.M + m], coef = e.coef[m];
        // the target's gradient from the forward's logit, once a row
        gtarget = coef == 0.0f ? 0.0f : coef * (exp2_fast(fmaf(e.lse[2 * (int64_t)a.M + m] - top, kLog2e, -lsum)) - 1.0f);
      }
      if (EPI == kEpiStore && e.alpha) alpha = *e.alpha;
      float row_bias = 0.0f;
      if (kAct && e.bias_rows && m < a.M) row_bias = to_f(((const T*)e.bias)[m]);
      float row_scale = 0.0f;
      if (EPI == kEpiInt8 && m < a.M) row_scale = e.row_scale[m];
#pragma unroll 1
      for (int nt = t.nt; nt < t.nt_end; nt++) {
        // what the epilogue adds is asked for before the product is waited for
        constexpr bool kAdds = kAct || EPI == kEpiPartial;
        const int first = part * 32;
        const int col = nt * BN;
        View add{nullptr, 0, 0};
        if (kAct) add = e.res;
        if (EPI == kEpiPartial && e.add) add = View{e.part + (int64_t)t.split * a.M * a.N, a.N, 1};
        bool waited = false;
        auto wait_product = [&] {
          if (!mbar_wait(tfull + 8 * acc, acc_phase, dead, a.wait_limit)) on = false;
          on = __all_sync(0xffffffffu, on);
          fence_after();
          waited = true;
        };
        if (CHAIN && a.chain) {
          // a sum longer than a chain: each accumulation, in the first accumulator, is added to the second, which no
          // product writes; the product waits for that once a chain
#pragma unroll 1
          for (int s0 = t.kb0; s0 < t.kb1; s0 += a.chain) {
            wait_product();
            if (!on) break;
#pragma unroll 1
            for (int c = first; c < kAcc && m0 < a.M; c += 32 * S::kParts) {
              if (col + c % BN >= a.N) continue;
              const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + c;
              if constexpr (S::kBlocks == 2) fold_chain_call(from + kAcc, from, s0 == t.kb0);
              else fold_chain<16>(from + kAcc, from, s0 == t.kb0);
            }
            fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (S::kPair) mbar_arrive_cluster(at_rank(tempty, 0));
              else mbar_arrive(tempty);
            }
            acc_phase ^= 1;
          }
          if (!on) break;
        }
#pragma unroll 1
        for (int c = first; c < BN && col + c < a.N && m0 < a.M; c += 32 * S::kParts) {
          const int n0 = col + c;
          const Place here = place(n0);
          Row<T> extra;
          int way = kNone;
          if (kAdds && add.p) way = load_tile<T>(extra, add, kAct ? res_access : access_of<T>(add), st, lane, here);
          if (!waited) wait_product();
          if (!on) break;
          const uint32_t src = tmem + ((uint32_t)(quad * 32) << 16) + (CHAIN && a.chain ? kAcc : acc * kAcc) + c;
          if (EPI != kEpiPartial && EPI != kEpiStore) {
            if ((EPI == kEpiInt8 || (e.bias && !e.bias_rows)) && bias_at != n0) {  // a lane a column, then every lane all of them
              __syncwarp();
              if (EPI != kEpiInt8 || (e.bias && !e.bias_rows))
                sts_cell(bias_slot + lane * 4, __float_as_uint(lane < here.cols ? to_f(((const T*)e.bias)[n0 + lane]) : 0.0f));
              if (EPI == kEpiInt8) sts_cell(bias_slot + 128 + lane * 4, __float_as_uint(lane < here.cols ? e.col_scale[n0 + lane] : 0.0f));
              bias_at = n0;
            }
          }
          __syncwarp();
          if constexpr (kAct || EPI == kEpiStore || EPI == kEpiPartial) {
            if (kAdds && add.p) own_row<T>(extra, way, st, lane);
            Row<T> y;
            auto columns = [&](auto with_slope, Row<SlopeCell<T>>& d) {
              constexpr bool kSlope = decltype(with_slope)::value;
#pragma unroll
              for (int h = 0; h < 2; h++) {  // 16 columns at a time: with 32 the activations spill
                float2 v[8];
                tmem_load16(src + h * 16, (float*)v);
                if constexpr (PL == 3) {
                  float2 u[8];
                  tmem_load16(src + BN + h * 16, (float*)u);
                  tmem_wait_load();
#pragma unroll
                  for (int j = 0; j < 8; j++) v[j] = __fadd2_rn(v[j], u[j]);
                } else {
                  tmem_wait_load();
                }
                if constexpr (EPI == kEpiInt8) scale_sums(bias_slot + 128 + h * 64, row_scale, v);
                if constexpr (kAct) {
                  if (e.bias_rows) {
#pragma unroll
                    for (int j = 0; j < 8; j++) v[j] = __fadd2_rn(v[j], pair(row_bias));
                  } else if (e.bias) {
                    add_bias<16>(bias_slot + h * 64, v);
                  }
#pragma unroll
                  for (int j = 0; j < 8; j++) {
                    float2 w, s;
                    activate<ACT, sizeof(T) == 4, kSlope>(v[j], w, s);
                    v[j] = ACT == VI_ACT_RELU ? relu_signed_zero<T>(w) : w;
                    if constexpr (kSlope) {
                      if constexpr (sizeof(T) == 4) set_pair(d, h * 8 + j, s);
                      else d.w[h * 8 + j] = Slope<T>::pack(s);
                    }
                  }
                }
                if (kAdds && add.p) {
#pragma unroll
                  for (int j = 0; j < 8; j++) v[j] = __fadd2_rn(v[j], get_pair(extra, h * 8 + j));
                }
#pragma unroll
                for (int j = 0; j < 8; j++)
                  set_pair(y, h * 8 + j, EPI == kEpiStore ? __fmul2_rn(v[j], pair(alpha)) : v[j]);
                // the half is finished before the next one starts, or their registers add up
#pragma unroll
                for (int j = 0; j < 4 * (int)sizeof(T); j++) {
                  asm volatile("" : "+r"(y.w[h * 4 * sizeof(T) + j]));
                  if constexpr (kSlope) asm volatile("" : "+r"(d.w[h * 4 * sizeof(T) + j]));
                }
              }
            };
            Row<SlopeCell<T>> d;
            if (EPI != kEpiInt8 && ACT != VI_ACT_NONE && e.dact) {
              columns(std::true_type(), d);
              store_tile(d, View{e.dact, e.out.rs, e.out.cs}, (uintptr_t)e.dact & 15 ? kScalar : out_access, st, lane, here);
            } else {
              columns(std::false_type(), d);
            }
            const View out = EPI == kEpiPartial ? View{e.part + (int64_t)t.split * a.M * a.N, a.N, 1} : e.out;
            store_tile(y, out, EPI == kEpiPartial ? access_of<T>(out) : out_access, st, lane, here);
          } else if constexpr (EPI == kEpiLse) {
            float2 v[16];
            tmem_load32(src, (float*)v);
            if constexpr (PL == 3) {
              float2 u[16];
              tmem_load32(src + BN, (float*)u);
              tmem_wait_load();
#pragma unroll
              for (int j = 0; j < 16; j++) v[j] = __fadd2_rn(v[j], u[j]);
            } else {
              tmem_wait_load();
            }
            if (e.bias) add_bias<32>(bias_slot, v);
            float* z = (float*)v;
            const int tc = target - n0;
            if (__any_sync(0xffffffffu, tc >= 0 && tc < 32)) {  // the target's logit, by halves
              float u[16];
#pragma unroll
              for (int j = 0; j < 16; j++) u[j] = tc & 16 ? z[j + 16] : z[j];
#pragma unroll
              for (int h = 8; h; h /= 2)
#pragma unroll
                for (int j = 0; j < h; j++) u[j] = tc & h ? u[j + h] : u[j];
              if (tc >= 0 && tc < 32) e.ztarget[m] = u[0];
            }
            if (n0 + 32 > a.N) {
#pragma unroll
              for (int j = 0; j < 32; j++)
                if (n0 + j >= a.N) z[j] = -INFINITY;
            }
            float u[8];  // several chains: one of 32 dependent steps would be waited for
#pragma unroll
            for (int j = 0; j < 8; j++) u[j] = fmaxf(fmaxf(z[j], z[j + 8]), fmaxf(z[j + 16], z[j + 24]));
            const float best = fmaxf(fmaxf(fmaxf(fmaxf(u[0], u[1]), fmaxf(u[2], u[3])), top),
                                     fmaxf(fmaxf(u[4], u[5]), fmaxf(u[6], u[7])));
            // a row of -inf so far: leave the sum at zero, without -inf - -inf
            const float ref = best == -INFINITY ? 0.0f : best;
            float2 s2[4] = {pair(0.0f), pair(0.0f), pair(0.0f), pair(0.0f)};
#pragma unroll
            for (int j = 0; j < 16; j++) {
              // the difference first: a logit of the type's lowest value times log2(e) would overflow
              const float2 x = __fmul2_rn(__fadd2_rn(v[j], pair(-ref)), pair(kLog2e));
              s2[j % 4] = __fadd2_rn(s2[j % 4], make_float2(exp2_fast(x.x), exp2_fast(x.y)));
            }
            const float2 all = __fadd2_rn(__fadd2_rn(s2[0], s2[1]), __fadd2_rn(s2[2], s2[3]));
            sum = sum * exp2_fast((top - ref) * kLog2e) + (all.x + all.y);
            top = best;
          } else if constexpr (EPI == kEpiGrad) {
            float2 v[16];
            tmem_load32(src, (float*)v);
            if constexpr (PL == 3) {
              float2 u[16];
              tmem_load32(src + BN, (float*)u);
              tmem_wait_load();
#pragma unroll
              for (int j = 0; j < 16; j++) v[j] = __fadd2_rn(v[j], u[j]);
            } else {
              tmem_wait_load();
            }
            if (e.bias) add_bias<32>(bias_slot, v);
            float* z = (float*)v;
#pragma unroll
            for (int j = 0; j < 16; j++) {
              const float2 x = __ffma2_rn(__fadd2_rn(v[j], pair(-top)), pair(kLog2e), pair(-lsum));
              v[j] = make_float2(exp2_fast(x.x), exp2_fast(x.y));
            }
            const int fix = target >= n0 && target < n0 + 32 ? target - n0 : -1;
#pragma unroll
            for (int j = 0; j < 16; j++) v[j] = __fmul2_rn(v[j], pair(coef));
            if (__any_sync(0xffffffffu, coef == 0.0f)) {  // an ignored row's logits may be anything
#pragma unroll
              for (int j = 0; j < 32; j++) z[j] = coef == 0.0f ? 0.0f : z[j];
            }
            if constexpr (sizeof(T) == 4) {
#pragma unroll
              for (int pl = 0; pl < 3; pl++) {
                Row<__nv_bfloat16> g;
#pragma unroll
                for (int j = 0; j < 32; j++) {
                  __nv_bfloat16 s3[3];
                  split3(z[j], s3);
                  g.z[j] = s3[pl];
                }
                const View out{(__nv_bfloat16*)e.grad + pl * e.grad_plane, e.grad_ld, 1};
                __nv_bfloat16 t3[3];
                split3(gtarget, t3);
                store_tile(g, out, kVector, st, lane, here, fix, __bfloat16_as_ushort(t3[pl]));
              }
            } else {
              Row<T> g;
#pragma unroll
              for (int j = 0; j < 16; j++) set_pair(g, j, v[j]);
              store_tile(g, View{e.grad, e.grad_ld, 1}, kVector, st, lane, here, fix, bits_of(from_f<T>(gtarget)));
              if (e.column_part) {
                __syncwarp();
                int column;
                const float sum = staged_column_sum<T>(st, lane, column);
                if (column < here.cols) e.column_part[(int64_t)(m0 / 32) * a.N + n0 + column] = sum;
              }
            }
          }
        }
        if (!waited) wait_product();
        if (!on) break;
        if (CHAIN && a.chain) continue;  // the accumulators were handed back as they were added
        fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (S::kPair) mbar_arrive_cluster(at_rank(tempty + 8 * acc, 0));
          else mbar_arrive(tempty + 8 * acc);
        }
        if (++acc == 2) acc = 0, acc_phase ^= 1;
      }
      if (EPI == kEpiLse && on && m < a.M) {
        e.pmax[(int64_t)(S::kParts * t.span + part) * a.M + m] = top;
        e.psum[(int64_t)(S::kParts * t.span + part) * a.M + m] = sum;
      }
    }
  }
  __syncwarp();
  // a pair ends together: its blocks arrive at each other's barriers.  Where both gave up, the first one's
  // last arrival at the second is that of its drain
  if constexpr (S::kPair) {
    __syncthreads();
    if (threadIdx.x == 0 && rank == 1 && *dead) mbar_drain(drain, 0, a.wait_limit);
    __syncwarp();
    cluster_sync();
  } else {
    __syncthreads();
  }
  if (warp == kEpiWarps + 1) {
    if constexpr (S::kPair)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
  }
  if (threadIdx.x == 0 && *dead) atomicOr(a.status, VI_DEVICE_HEAD_TIMEOUT);
}

// ---- host ----
constexpr int kInt8 = -1;  // operands of 8-bit integers, k contiguous

// The operand as [plane][outer][inner] with boxes of `box_rows` rows x 128 bytes of k.
bool encode(CUtensorMap* map, const Operand& o, int planes, int dtype, int box_rows) {
  const bool bytes = dtype == kInt8;
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t inner = (cuuint64_t)(o.k_major ? o.k : o.rows), outer = (cuuint64_t)(o.k_major ? o.rows : o.k);
  const cuuint64_t dims[3] = {inner, outer, (cuuint64_t)planes};
  const cuuint64_t size = bytes ? 1 : 2;
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * size, (cuuint64_t)(planes > 1 ? o.plane : o.ld) * size};
  const cuuint32_t box[3] = {bytes ? 128u : 64u, (cuuint32_t)(o.k_major ? box_rows : kBK), 1};
  const cuuint32_t unit[3] = {1, 1, 1};
  return fn(map, bytes             ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                 : dtype == VI_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                   : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.p), dims,
            strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// type: of the operands in the instruction descriptor (float16 0, bfloat16 1; signed 8-bit integers 1); sums are
// float32 (1) or 32-bit integers (2).  Returns a vi_status.
int fill_args(Args& a, const Operand& A, const Operand& B, const Plan& p, int epi, uint32_t type) {
  a = Args{};
  const bool pair = pair_tile(epi, p.bn);
  a.M = (int)A.rows;
  a.N = (int)B.rows;
  const int64_t rows = pair ? 2 * kBM : kBM;  // of a tile
  a.m_tiles = (int)((A.rows + rows - 1) / rows);
  a.n_tiles = (int)((B.rows + p.bn - 1) / p.bn);
  a.kblocks = (int)((A.k + block_terms(epi) - 1) / block_terms(epi));
  a.kps = p.kps;
  a.splits = p.splits;
  a.span = p.span;
  a.spans = p.spans;
  a.a_k_major = A.k_major;
  a.b_k_major = B.k_major;
  // k contiguous: 16 k are 32 bytes of a swizzled row.  Rows contiguous: 16 k are two groups of 1024 bytes.
  a.a_lbo = A.k_major ? 1 : 8192 >> 4;
  a.b_lbo = B.k_major ? 1 : 8192 >> 4;
  a.a_step = A.k_major ? 32 >> 4 : 2048 >> 4;
  a.b_step = B.k_major ? 32 >> 4 : 2048 >> 4;
  a.idesc = ((epi == kEpiInt8 ? 2u : 1u) << 4) | (type << 7) | (type << 10) | ((A.k_major ? 0u : 1u) << 15) | ((B.k_major ? 0u : 1u) << 16) |
            ((uint32_t)(p.bn >> 3) << 17) | ((uint32_t)(rows >> 4) << 24);
  const int64_t cols = epi == kEpiLse ? p.spans : a.n_tiles, items = (int64_t)a.m_tiles * cols * p.splits;
  if (items > INT32_MAX - 65536 || 16 * cols > INT32_MAX)
    return set_error(VI_ERR_UNSUPPORTED, "heads: more than 2^31 tiles");
  a.items = (int)items;
  a.per_split = FastDiv::of((uint32_t)(a.m_tiles * cols));
  a.per_group = FastDiv::of((uint32_t)(16 * cols));
  a.last_rows = FastDiv::of((uint32_t)(a.m_tiles % 16 ? a.m_tiles % 16 : 16));
  const char* test = getenv("VI_HEADS_TEST_TIMEOUT");
  a.withhold = test && test[0] == '1';
  a.wait_limit = a.withhold ? 1 << 20 : kWaitLimit;
  a.status = status_word();
  return a.status ? VI_OK : set_error(VI_ERR_CUDA, "heads: the status word has no address");
}

template <typename T, int BN, int EPI, int PL, int ACT, bool CHAIN>
cudaError_t run(const CUtensorMap& ma, const CUtensorMap& mb, const Args& a, int sms, cudaStream_t s) {
  using S = Shape<T, BN, EPI, PL>;
  auto* k = gemm_tc_kernel<T, BN, EPI, PL, ACT, CHAIN>;
  // once per device: the call costs as much as a launch
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (!(done.load(std::memory_order_relaxed) & bit)) {
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  }
  if constexpr (S::kPair) {
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(2 * (unsigned)std::min<int64_t>(a.items, std::max(1, sms / 2)));
    c.blockDim = dim3(S::kThreads);
    c.dynamicSmemBytes = S::kSmem;
    c.stream = s;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    c.attrs = &attr;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, k, ma, mb, a);
  } else {
    k<<<(unsigned)std::min<int64_t>(a.items, (int64_t)sms * S::kBlocks), S::kThreads, S::kSmem, s>>>(ma, mb, a);
    return cudaPeekAtLastError();
  }
}
}  // namespace
}  // namespace heads
}  // namespace vi
