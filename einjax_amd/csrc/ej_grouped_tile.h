// Tile kernels of the products grouped by expert: BM x BN results per
// workgroup, WR x WC waves, a ring of NS stages in LDS.
#pragma once

#include "ej_grouped.h"

#include <type_traits>

namespace ej {

template <int N>
__device__ inline void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Waits until the oldest stage in flight has landed; `later` stages of LPS
// loads each were issued after it (at most NS - 2).
template <int NS, int LPS>
__device__ inline void wait_oldest(int later) {
  static_assert((NS == 2 || NS == 3) && (NS - 2) * LPS < 64, "ring depth");
  if constexpr (NS == 3) {
    if (later >= 1) { wait_vm<LPS>(); return; }
  }
  wait_vm<0>();
}

// Position of logical block lb in a grid of rbs x cbs blocks: bands of `band`
// row blocks, walked column by column, so that the blocks which run together
// on an XCD share both operands' tiles in its L2.
__device__ inline void band_pos(uint32_t lb, uint32_t rbs, uint32_t cbs, uint32_t band, int *rb,
                                int *cb) {
  const uint32_t per = band * cbs, i = lb / per, r = lb - i * per;
  const uint32_t h = rbs - i * band < band ? rbs - i * band : band;
  *rb = static_cast<int>(i * band + r % h);
  *cb = static_cast<int>(r / h);
}

template <class Op, int BM, int BN, int WR, int WC, bool AKC, bool BKC, bool DIRECT, int NS>
struct TileShape {
  static constexpr int kWaves = WR * WC;
  static constexpr int kThreads = kWaves * 64;
  static constexpr int WM = BM / WR, WN = BN / WC;
  static constexpr int FM = WM / 16, FN = WN / 16;
  using TA = Tile<Op, BM, AKC>;
  using TB = Tile<Op, BN, BKC>;
  using FA = Fragments<Op, TA, AKC, FM>;
  using FB = Fragments<Op, TB, BKC, FN>;
  using LA = Loader<Op, BM, AKC, kWaves, DIRECT>;
  using LB = Loader<Op, BN, BKC, kWaves, DIRECT>;
  static constexpr int kSlot = TA::kBytes + TB::kBytes;
  static constexpr int kLds = NS == 0 ? 3 * TA::kBytes + 2 * TB::kBytes : NS * kSlot;
  static constexpr int kLoads = LA::kLoads + LB::kLoads;
};

// acc[i][j] += A fragment i times B fragment j over the stage `slot` bytes
// into the ring.  The B fragment gives the accumulator's register rows, so a lane
// ends with four consecutive columns of one row of the result.
template <class Op, class S>
__device__ inline void stage_mma(typename Op::acc (&acc)[S::FM][S::FN], const typename S::FA &fa,
                                 const typename S::FB &fb, uint32_t slot) {
#pragma unroll
  for (int slab = 0; slab < 2; ++slab) {
    i32v4_t a[S::FM], b[S::FN];
#pragma unroll
    for (int i = 0; i < S::FM; ++i) a[i] = fa.read(slot, i, slab);
#pragma unroll
    for (int j = 0; j < S::FN; ++j) b[j] = fb.read(slot, j, slab);
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
      for (int j = 0; j < S::FN; ++j) mma<Op>(acc[i][j], b[j], a[i]);
  }
}

// The same with the fragments of one 64-byte slab read while the matrix
// instructions of the slab before run, on a ring of three stages of A and two
// of B:
//   slab 0 of stage st:  read slab 1's fragments; load A of stage st + 2 into
//                        the slot of stage st - 1
//   every wave has read stage st and stage st + 1 has landed: one barrier
//   slab 1 of stage st:  read slab 0's fragments of stage st + 1; load B of
//                        stage st + 2 into the slot of stage st
// So loads are under way all the time: the L1 keeps only some hundred requests
// of 128 bytes in flight, for 500 cycles or more each, which is what bounds
// the large blocks, and a burst of a whole stage would leave it idle in
// between.  Loads and LDS reads are spread over the matrix instructions.  One
// group of 16384 x 4096 x 2048 in bf16, 256 x 256: 198 us (1386 TFLOP/s);
// 8192 cubed, W [n][k]: 755 us (1456 TFLOP/s; the library's product 728).
// Measured no better: loads at higher wave priority, padded rows instead of
// the swizzle, stages of half the depth in a longer ring.
template <class Op, class S, class Load>
__device__ inline void run_pipelined(typename Op::acc (&acc)[S::FM][S::FN], unsigned char *ring,
                                     int stages, const typename S::FA &pa,
                                     const typename S::FB &pb, Load load_stage) {
  i32v4_t fa[2][S::FM], fb[2][S::FN];
  constexpr int kA = S::TA::kBytes, kB = S::TB::kBytes;
  constexpr int kFrags = S::FN + S::FM;
  constexpr int kReads = S::FM * S::TA::kReads + S::FN * S::TB::kReads;
  // fragment r of the FN + FM of a slab
  auto read = [&](int f, uint32_t a, uint32_t b, int slab, int r) {
    if (r < S::FN) fb[f][r] = pb.read(b, r, slab);
    else fa[f][r - S::FN] = pa.read(a, r - S::FN, slab);
  };
  // matrix instructions of fragments f, while slab `slab` of the stage at a, b
  // is read and `n` loads are issued
  auto slab = [&](int f, uint32_t a, uint32_t b, int slab, auto kN, auto load) {
    constexpr int n = decltype(kN)::value, cells = S::FM * S::FN;
    // a part for each load where it has enough matrix instructions
    constexpr int parts = cells / n >= 8 ? n : 1;
#pragma unroll
    for (int p = 0; p < parts; ++p) {
      constexpr int kFragsOf = (kFrags + parts - 1) / parts, kLoadsOf = n / parts;
#pragma unroll
      for (int q = 0; q < kFragsOf || q < kLoadsOf; ++q) {
        if (q < kLoadsOf) load(p * kLoadsOf + q);
        const int r = p * kFrags / parts + q;
        if (r < (p + 1) * kFrags / parts) read(1 - f, a, b, slab, r);
      }
#pragma unroll
      for (int c = p * cells / parts; c < (p + 1) * cells / parts; ++c)
        mma<Op>(acc[c / S::FN][c % S::FN], fb[f][c % S::FN], fa[f][c / S::FN]);
      constexpr int kMma = cells * (kElem<Op> == 4 ? 4 : 1);
      constexpr int kEach = kMma / kReads > 1 ? 2 : 1;
#pragma unroll
      for (int r = 0; r < kReads / parts; ++r) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
        __builtin_amdgcn_sched_group_barrier(0x8, kEach, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using NA = std::integral_constant<int, S::LA::kLoads>;
  using NB = std::integral_constant<int, S::LB::kLoads>;
  if (stages == 0) return;
  // stages past the end are zeros, loaded from one cached line
  int st = 0;
  uint32_t a_now = 0, a_next = kA, a_put = 2 * kA, b_now = 3 * kA, b_next = 3 * kA + kB;
#pragma unroll
  for (int v = 0; v < S::LA::kLoads; ++v) load_stage(v, 0, ring + a_now, true);
#pragma unroll
  for (int v = 0; v < S::LB::kLoads; ++v)
    load_stage(S::LA::kLoads + v, 0, ring + b_now - kA, true);
#pragma unroll
  for (int v = 0; v < S::LA::kLoads; ++v) load_stage(v, 1, ring + a_next, true);
#pragma unroll
  for (int v = 0; v < S::LB::kLoads; ++v)
    load_stage(S::LA::kLoads + v, 1, ring + b_next - kA, true);
  wait_vm<S::kLoads>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int r = 0; r < kFrags; ++r) read(0, a_now, b_now - kA, 0, r);
  auto step = [&](auto kWhole) {
    constexpr bool part = !decltype(kWhole)::value;
    slab(0, a_now, b_now - kA, 1, NA(),
         [&](int v) { load_stage(v, st + 2, ring + a_put, part); });
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(S::LA::kLoads) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    slab(1, a_next, b_next - kA, 0, NB(), [&](int v) {
      load_stage(S::LA::kLoads + v, st + 2, ring + b_now - kA, part);
    });
    const uint32_t a = a_now, b = b_now;
    a_now = a_next;
    a_next = a_put;
    a_put = a;
    b_now = b_next;
    b_next = b;
    ++st;
  };
  while (st + 3 < stages) step(std::true_type());
  while (st < stages) step(std::false_type());
  // no load may still be writing LDS when the workgroup ends
  wait_vm<0>();
}

// The ring: load_stage(st, slot pointer) starts the loads of stage st,
// store_stage(slot pointer) finishes them where they go through registers.
template <class Op, class S, bool DIRECT, int NS, class Load, class Store>
__device__ inline void run_stages(typename Op::acc (&acc)[S::FM][S::FN], unsigned char *ring,
                                  int stages, int row0, int col0, int lane, Load load_stage,
                                  Store store_stage) {
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<size_t>((lds_u8 *)ring));
  typename S::FA fa;
  typename S::FB fb;
  fa.init(base, row0, lane);
  fb.init(base + S::TA::kBytes, col0, lane);
  auto load_all = [&](int st, unsigned char *slot) {
#pragma unroll
    for (int v = 0; v < S::kLoads; ++v) load_stage(v, st, slot, true);
  };
  if constexpr (DIRECT && NS == 0) {
    run_pipelined<Op, S>(acc, ring, stages, fa, fb, load_stage);
  } else if constexpr (DIRECT) {
    int put = 0, get = 0;
    for (int st = 0; st < NS - 1 && st < stages; ++st) {
      load_all(st, ring + put * S::kSlot);
      put = put + 1 == NS ? 0 : put + 1;
    }
    for (int st = 0; st < stages; ++st) {
      const int left = stages - 1 - st;
      wait_oldest<NS, S::kLoads>(left < NS - 2 ? left : NS - 2);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (st + NS - 1 < stages) {
        load_all(st + NS - 1, ring + put * S::kSlot);
        put = put + 1 == NS ? 0 : put + 1;
      }
      stage_mma<Op, S>(acc, fa, fb, get * S::kSlot);
      // read before the barrier after which other waves load into this slot
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      get = get + 1 == NS ? 0 : get + 1;
    }
  } else {
    if (stages > 0) {
      load_all(0, ring);
      store_stage(ring);
    }
    for (int st = 0; st < stages; ++st) {
      __syncthreads();
      if (st + 1 < stages) load_all(st + 1, ring);
      stage_mma<Op, S>(acc, fa, fb, (st & 1) * S::kSlot);
      if (st + 1 < stages) store_stage(ring + ((st + 1) & 1) * S::kSlot);
    }
  }
}

// The results of a wave: row(i, &at) gives the element offset of fragment row
// i's results and whether there is such a row, value(i, j, c) its result c of
// four in fragment column j.
template <class S, class Row, class Value>
__device__ inline void put_results(const GroupedArgs &g, int col0, int lane, Row row,
                                   Value value) {
  if (S::FN % 2 == 0 && g.out != EJ_F32) {
#pragma unroll
    for (int i = 0; i < S::FM; ++i) {
      int64_t at;
      const bool there = row(i, &at);
#pragma unroll
      for (int j = 0; j + 1 < S::FN; j += 2) {
        float v[2][4];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c / 4][c % 4] = value(i, j + c / 4, c % 4);
        put8(g.c, g.out, at, col0 + j * 16, g.n, lane, there, v);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < S::FM; ++i) {
    int64_t at;
    if (!row(i, &at)) continue;
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
      const int col = col0 + j * 16 + (lane >> 4) * 4;
      if (col >= g.n) continue;
      float v[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = value(i, j, c);
      put4(g.c, g.out, at, col, g.n, v);
    }
  }
}

// C rows of one row block of a group times the BN columns from n0.
template <class Op, int BM, int BN, int WR, int WC, bool BKC, bool DIRECT, int NS>
__device__ inline void rows_block(GroupedArgs g, const RowBlock &r, int n0, unsigned char *ring) {
  using S = TileShape<Op, BM, BN, WR, WC, true, BKC, DIRECT, NS>;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row0 = wave / WC * S::WM, col0 = wave % WC * S::WN;
  int st0, st1;
  part_of((g.k + kStep<Op> - 1) / kStep<Op>, blockIdx.y, g.splits, &st0, &st1);
  const int64_t k0 = static_cast<int64_t>(st0) * kStep<Op>;
  const int ks = g.k - static_cast<int>(k0);  // k left from the part's start

  typename S::LA la;
  typename S::LB lb;
  la.init_k(wave, lane, g.k, [&](int i) {
    const int s = r.lo + i < r.hi ? r.lo + i : r.hi - 1;
    return g.a + (slot_row(g.a_rows, g.n_a, s) * g.lda + k0) * kElem<Op>;
  });
  const char *bg = g.b + r.group * g.b_group * kElem<Op>;
  int64_t b_step;
  if constexpr (BKC) {
    lb.init_k(wave, lane, g.k, [&](int i) {
      const int n = n0 + i < g.n ? n0 + i : g.n - 1;
      return bg + (n * g.ldb + k0) * kElem<Op>;
    });
    b_step = kRowB;
  } else {
    lb.init_m(wave, lane, bg + k0 * g.ldb * kElem<Op>, g.ldb, n0, g.n);
    b_step = kStep<Op> * g.ldb * kElem<Op>;
  }

  typename Op::acc acc[S::FM][S::FN];
#pragma unroll
  for (int i = 0; i < S::FM; ++i)
#pragma unroll
    for (int j = 0; j < S::FN; ++j) acc[i][j] = typename Op::acc{0, 0, 0, 0};
  run_stages<Op, S, DIRECT, NS>(
      acc, ring, st1 - st0, row0, col0, lane,
      [&](int v, int st, unsigned char *slot, bool part) {
        const int left = ks - st * kStep<Op>;
        if (v < S::LA::kLoads)
          la.load(v, slot, wave, left, kRowB, part);
        else
          lb.load(v - S::LA::kLoads, slot + S::TA::kBytes, wave, left, b_step, part);
      },
      [&](unsigned char *slot) {
        la.store(slot, wave, lane);
        lb.store(slot + S::TA::kBytes, wave, lane);
      });

  if (g.splits > 1) {
    g.c = g.partial + blockIdx.y * g.slots * g.n;
    g.ldc = g.n;
    g.out = EJ_F32;
  }
  float as[S::FM], bs[S::FN][4];  // 8 bits: scales of the rows and columns
  if constexpr (Op::kInt) {
#pragma unroll
    for (int i = 0; i < S::FM; ++i) {
      const int s = r.lo + row0 + i * 16 + (lane & 15);
      as[i] = g.a_scale[slot_row(g.a_rows, g.n_a, s < r.hi ? s : r.hi - 1)];
    }
#pragma unroll
    for (int j = 0; j < S::FN; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int col = n0 + col0 + j * 16 + (lane >> 4) * 4 + c;
        bs[j][c] = g.b_scale[static_cast<int64_t>(r.group) * g.n + (col < g.n ? col : g.n - 1)];
      }
  }
  put_results<S>(
      g, n0 + col0, lane,
      [&](int i, int64_t *at) {
        const int s = r.lo + row0 + i * 16 + (lane & 15);
        *at = s * g.ldc;
        return s < r.hi;
      },
      [&](int i, int j, int c) {
        const float v = static_cast<float>(acc[i][j][c]);
        if constexpr (Op::kInt) return scaled(v, as[i], bs[j][c]);
        else return v;
      });
}

// A workgroup for each row block of a group and block of columns.  Bound by the
// loads into LDS (operands of two bytes, see run_pipelined) or by the matrix
// instructions (fp32).  4096 rows in 8 groups, k = 1024, n = 2048 in fp32, 64 x
// 64: 154 us (111 TFLOP/s, of 128 that a large fp32 product reaches).  Rows off
// 16 bytes (3022 rows in 12 groups, k = 771, n = 1283, f16), 128 x 128 through
// registers: 33 us, 21 us at aligned extents; the rest are another column of
// tiles and stage of k, and the unaligned loads, two lines for most of them.
// Aligned loads with the bytes shifted into place afterwards took as long.
template <class Op, int BM, int BN, int WR, int WC, bool BKC, bool DIRECT, int NS>
__global__ __launch_bounds__(WR *WC * 64) void grouped_rows_kernel(GroupedArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using S = TileShape<Op, BM, BN, WR, WC, true, BKC, DIRECT, NS>;
  __shared__ __align__(1024) unsigned char ring[S::kLds];
  const uint32_t grid = g.row_blocks * g.col_blocks;
  if (blockIdx.x >= grid) {
    if (blockIdx.y == 0) zero_dead_rows(g, blockIdx.x - grid, gridDim.x - grid);
    return;
  }
  const uint32_t rbs = live_row_blocks(g, BM), live = rbs * g.col_blocks;
  if (blockIdx.x >= live) return;
  int rb, cb;
  band_pos(xcd_logical_block(live), rbs, g.col_blocks, 1024 / BM, &rb, &cb);
  rows_block<Op, BM, BN, WR, WC, BKC, DIRECT, NS>(g, find_row_block(g, BM, rb), cb * BN, ring);
#endif
}

// Large blocks of 256 x 256 results, one workgroup to a CU, run in rounds of
// kLargeRound.  The blocks of a last round that would leave half the CUs idle
// or more are cut in two (128 x 256) or four (128 x 128), a workgroup each.
constexpr uint32_t kLargeRound = 256;
constexpr uint32_t kLargeExtra = 192;  // workgroups that cutting adds at most

// The work of a workgroup: a block, or from row, col of it one of `parts`.
struct LargeUnit {
  uint32_t block, parts;
  int row, col;
  __device__ inline bool find(uint32_t live, uint32_t run) {
    uint32_t whole = live / kLargeRound * kLargeRound;
    const uint32_t last = live - whole;
    const uint32_t cut = last <= kLargeRound / 4 ? 4 : last <= kLargeRound / 2 ? 2 : 1;
    if (cut == 1) whole = live;
    parts = 1;
    row = col = 0;
    if (blockIdx.x < whole) {
      block = xcd_logical_block(whole, run);
      return true;
    }
    const uint32_t units = (live - whole) * cut;
    if (blockIdx.x - whole >= units) return false;
    const uint32_t u = xcd_logical_of(blockIdx.x - whole, units, 0), part = u % cut;
    parts = cut;
    block = whole + u / cut;
    row = (part & 1) * 128;
    col = (part >> 1) * 128;
    return true;
  }
};

// Rows in large blocks.  One of at most 128 rows (the end of a group) takes
// half the work.  16384 rows in 16 groups, k = 4096, n = 2048 in bf16: 265 us
// (1040 TFLOP/s), uncut and with whole blocks alone 40 us more; 32768 rows, k =
// n = 4096: 945 us (1164 TFLOP/s), 50 more; 16384 rows in 8 groups in 8 bits, k
// = n = 4096: 260 us (2115 TOP/s), 45 more.  256 workgroups that walk the blocks
// and load the next while they store the last were 5% faster in one group and
// in 8 bits, 3 to 10% slower in 16 groups (dealt out beforehand, the short
// blocks leave CUs waiting, and the registers spill).
template <class Op, bool BKC>
__global__ __launch_bounds__(512) void grouped_large_kernel(GroupedArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using S = TileShape<Op, 256, 256, 2, 4, true, BKC, true, 0>;
  __shared__ __align__(1024) unsigned char ring[S::kLds];
  const uint32_t grid = g.row_blocks * g.col_blocks + kLargeExtra;
  if (blockIdx.x >= grid) {
    zero_dead_rows(g, blockIdx.x - grid, gridDim.x - grid);
    return;
  }
  const uint32_t rbs = live_row_blocks(g, 256);
  LargeUnit u;
  if (!u.find(rbs * g.col_blocks, 0)) return;
  int rb, cb;
  band_pos(u.block, rbs, g.col_blocks, 4, &rb, &cb);
  RowBlock r = find_row_block(g, 256, rb);
  r.lo += u.row;
  const int n0 = cb * 256 + u.col;
  if (r.lo >= r.hi || n0 >= g.n) return;
  if (u.parts == 4)
    rows_block<Op, 128, 128, 2, 4, BKC, true, 0>(g, r, n0, ring);
  else if (u.parts == 2 || r.hi - r.lo <= 128)
    rows_block<Op, 128, 256, 2, 4, BKC, true, 0>(g, r, n0, ring);
  else
    rows_block<Op, 256, 256, 2, 4, BKC, true, 0>(g, r, n0, ring);
#endif
}

// D_e block: the BM columns of P from m0 (rows of the result) by the BN
// columns of Q from n0, over the slots of a group; one without slots writes
// zeros.  GATHER: 1 if P's rows go through an index, 2 if Q's do.
template <class Op, int BM, int BN, int WR, int WC, bool DIRECT, int NS, int GATHER>
__device__ inline void wgrad_block(GroupedArgs g, int group, int m0, int n0, unsigned char *ring) {
  using S = TileShape<Op, BM, BN, WR, WC, false, false, DIRECT, NS>;
  int lo, hi;
  group_range(g, group, &lo, &hi);
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row0 = wave / WC * S::WM, col0 = wave % WC * S::WN;

  typename S::LA la;
  typename S::LB lb;
  int st0, st1;
  part_of((hi - lo + kStep<Op> - 1) / kStep<Op>, blockIdx.y, g.splits, &st0, &st1);
  if (g.splits > 1) {
    lo += st0 * kStep<Op>;
    g.c = g.partial + blockIdx.y * (static_cast<int64_t>(g.n_groups) * g.m * g.n);
    g.c_group = static_cast<int64_t>(g.m) * g.n;
    g.ldc = g.n;
    g.out = EJ_F32;
  }
  la.init_m(wave, lane, g.a + (GATHER == 1 ? 0 : lo * g.lda * kElem<Op>), g.lda, m0, g.m);
  lb.init_m(wave, lane, g.b + (GATHER == 2 ? 0 : lo * g.ldb * kElem<Op>), g.ldb, n0, g.n);
  // the gathered operand's rows of a stage, lane by lane, read a stage ahead
  const int32_t *rows = GATHER == 1 ? g.a_rows : g.b_rows;
  const int64_t n_rows = GATHER == 1 ? g.n_a : g.n_b;
  auto rows_of = [&](int st) {
    const int64_t s = lo + static_cast<int64_t>(st) * kStep<Op> + lane;
    return static_cast<int>(slot_row(rows, n_rows, static_cast<int>(s < hi ? s : hi - 1)));
  };
  int row_now = 0, row_next = 0;
  if (GATHER && st1 > st0) row_next = rows_of(0);

  typename Op::acc acc[S::FM][S::FN];
#pragma unroll
  for (int i = 0; i < S::FM; ++i)
#pragma unroll
    for (int j = 0; j < S::FN; ++j) acc[i][j] = typename Op::acc{0, 0, 0, 0};
  run_stages<Op, S, DIRECT, NS>(
      acc, ring, st1 - st0, row0, col0, lane,
      [&](int v, int st, unsigned char *slot, bool part) {
        const int left = hi - lo - st * kStep<Op>;
        // all sources of the gathered operand at its first load: the lane
        // moves wait for every LDS read before them
        if (v < S::LA::kLoads) {
          if constexpr (GATHER == 1) {
            if (v == 0) {
              row_now = row_next;
              row_next = rows_of(st + 1);
              la.seek(g.a, g.lda, row_now);
            }
          }
          la.load(v, slot, wave, left, kStep<Op> * g.lda * kElem<Op>, part);
        } else {
          const int u = v - S::LA::kLoads;
          if constexpr (GATHER == 2) {
            if (u == 0) {
              row_now = row_next;
              row_next = rows_of(st + 1);
              lb.seek(g.b, g.ldb, row_now);
            }
          }
          lb.load(u, slot + S::TA::kBytes, wave, left, kStep<Op> * g.ldb * kElem<Op>, part);
        }
      },
      [&](unsigned char *slot) {
        la.store(slot, wave, lane);
        lb.store(slot + S::TA::kBytes, wave, lane);
      });

  put_results<S>(
      g, n0 + col0, lane,
      [&](int i, int64_t *at) {
        const int row = m0 + row0 + i * 16 + (lane & 15);
        *at = group * g.c_group + static_cast<int64_t>(row) * g.ldc;
        return row < g.m;
      },
      [&](int i, int j, int c) { return static_cast<float>(acc[i][j][c]); });
}

// row_blocks x col_blocks covers one group's D; the grid holds n_groups of
// them.
template <class Op, int BM, int BN, int WR, int WC, bool DIRECT, int NS, int GATHER>
__global__ __launch_bounds__(WR *WC * 64) void grouped_wgrad_kernel(GroupedArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using S = TileShape<Op, BM, BN, WR, WC, false, false, DIRECT, NS>;
  __shared__ __align__(1024) unsigned char ring[S::kLds];
  const uint32_t per = g.row_blocks * g.col_blocks;
  // runs of blocks dealt to the XCDs in turn: as one part each, the XCD of the
  // longest group ends last (16384 rows in 16 groups of unequal length, 2048 x
  // 4096 bf16, 256 x 256: 363 us so, 305 dealt; groups of equal length 285 and
  // 287)
  const uint32_t block = xcd_logical_block(gridDim.x, kXcdRun), group = block / per;
  int rb, cb;
  band_pos(block - group * per, g.row_blocks, g.col_blocks, 1024 / BM, &rb, &cb);
  wgrad_block<Op, BM, BN, WR, WC, DIRECT, NS, GATHER>(g, group, rb * BM, cb * BN, ring);
#endif
}

// The same in blocks of 256 x 256, cut as grouped_large_kernel's.  16384 rows
// in 16 groups, 2048 x 4096 bf16: 272 us (1010 TFLOP/s), 306 with P gathered
// (128 x 128: 350 and 442, 64 x 64: 522 and 721).  The bounds check of a row's
// index, in rows_of, follows its load, and waiting for that is waiting for every
// load in flight: each stage empties the ring that the others keep full.
template <class Op, int GATHER>
__global__ __launch_bounds__(512) void grouped_wgrad_large_kernel(GroupedArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using S = TileShape<Op, 256, 256, 2, 4, false, false, true, 0>;
  __shared__ __align__(1024) unsigned char ring[S::kLds];
  const uint32_t per = g.row_blocks * g.col_blocks;
  LargeUnit u;
  if (!u.find(per * g.n_groups, kXcdRun)) return;
  const uint32_t group = u.block / per;
  int rb, cb;
  band_pos(u.block - group * per, g.row_blocks, g.col_blocks, 4, &rb, &cb);
  const int m0 = rb * 256 + u.row, n0 = cb * 256 + u.col;
  if (m0 >= g.m || n0 >= g.n) return;
  if (u.parts == 4)
    wgrad_block<Op, 128, 128, 2, 4, true, 0, GATHER>(g, group, m0, n0, ring);
  else if (u.parts == 2 || g.m - m0 <= 128)
    wgrad_block<Op, 128, 256, 2, 4, true, 0, GATHER>(g, group, m0, n0, ring);
  else
    wgrad_block<Op, 256, 256, 2, 4, true, 0, GATHER>(g, group, m0, n0, ring);
#endif
}

// Few rows for each group: the time is that of reading the weights once.  A
// workgroup takes 16 rows by BN columns; its waves split k stage by stage
// (so that together they read long pieces of each weight row), each on a ring
// of its own without barriers, and add up their parts in LDS at the end, in
// the order of the waves.  32 slots of 16 groups, W [n][k] of 2048 x 4096 in
// bf16: 41 us for the 218 MB of the groups that have slots (5.4 TB/s); 4 rows x
// 4096 x 8192 in 8 bits 8.1 us (4.1 TB/s).
template <class Op, int BN, int NW, bool BKC, int NS>
struct SkinnyShape {
  static constexpr int BM = 16, FM = 1, FN = BN / 16;
  using TA = Tile<Op, BM, true>;
  using TB = Tile<Op, BN, BKC>;
  using FA = Fragments<Op, TA, true, FM>;
  using FB = Fragments<Op, TB, BKC, FN>;
  using LA = Loader<Op, BM, true, 1, true>;
  using LB = Loader<Op, BN, BKC, 1, true>;
  static constexpr int kSlot = TA::kBytes + TB::kBytes;
  static constexpr int kLoads = LA::kLoads + LB::kLoads;
  static constexpr int kRing = NS * kSlot;
  static constexpr int kPart = BM * BN * 4;  // bytes of a wave's sums
  static constexpr int kLds = NW * (kRing > kPart ? kRing : kPart);
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
};

template <class Op, int BN, int NW, bool BKC, int NS>
__global__ __launch_bounds__(NW * 64) void grouped_skinny_kernel(GroupedArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using S = SkinnyShape<Op, BN, NW, BKC, NS>;
  __shared__ __align__(1024) unsigned char lds[S::kLds];
  const uint32_t grid = g.row_blocks * g.col_blocks;
  if (blockIdx.x >= grid) {
    zero_dead_rows(g, blockIdx.x - grid, gridDim.x - grid);
    return;
  }
  const uint32_t rbs = live_row_blocks(g, S::BM), live = rbs * g.col_blocks;
  if (blockIdx.x >= live) return;
  // the row blocks of one group and column block follow each other: they read
  // the same weights
  int rb, cb;
  band_pos(xcd_logical_block(live), rbs, g.col_blocks, 4, &rb, &cb);
  const RowBlock r = find_row_block(g, S::BM, rb);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = cb * BN;
  unsigned char *ring = lds + wave * S::kRing;

  typename S::LA la;
  typename S::LB lb;
  const int stages = (g.k + kStep<Op> - 1) / kStep<Op>;
  const int mine = stages > wave ? (stages - wave + NW - 1) / NW : 0;
  const int64_t k0 = static_cast<int64_t>(wave) * kStep<Op>;
  la.init_k(0, lane, g.k, [&](int i) {
    const int s = r.lo + i < r.hi ? r.lo + i : r.hi - 1;
    return g.a + (slot_row(g.a_rows, g.n_a, s) * g.lda + k0) * kElem<Op>;
  });
  const char *bg = g.b + r.group * g.b_group * kElem<Op>;
  int64_t b_step;
  if constexpr (BKC) {
    lb.init_k(0, lane, g.k, [&](int i) {
      const int n = n0 + i < g.n ? n0 + i : g.n - 1;
      return bg + (n * g.ldb + k0) * kElem<Op>;
    });
    b_step = kRowB;
  } else {
    lb.init_m(0, lane, bg + k0 * g.ldb * kElem<Op>, g.ldb, n0, g.n);
    b_step = kStep<Op> * g.ldb * kElem<Op>;
  }
  auto load = [&](int i) {
    unsigned char *slot = ring + i % NS * S::kSlot;
    const int left = g.k - (wave + i * NW) * kStep<Op>;
#pragma unroll
    for (int v = 0; v < S::LA::kLoads; ++v) la.load(v, slot, 0, left, NW * kRowB, true);
#pragma unroll
    for (int v = 0; v < S::LB::kLoads; ++v)
      lb.load(v, slot + S::TA::kBytes, 0, left, NW * b_step, true);
  };
  typename S::FA fa;
  typename S::FB fb;
  fa.init(lds_address(ring), 0, lane);
  fb.init(lds_address(ring) + S::TA::kBytes, 0, lane);
  typename Op::acc acc[1][S::FN];
#pragma unroll
  for (int j = 0; j < S::FN; ++j) acc[0][j] = typename Op::acc{0, 0, 0, 0};
  for (int i = 0; i < NS - 1 && i < mine; ++i) load(i);
  for (int i = 0; i < mine; ++i) {
    const int later = mine - 1 - i;
    // the slot that is loaded next was read a stage ago: those reads are done
    // once their matrix instructions have been issued
    if (i + NS - 1 < mine) load(i + NS - 1);
    wait_oldest<NS + 1, S::kLoads>(later < NS - 1 ? later : NS - 1);
    stage_mma<Op, S>(acc, fa, fb, i % NS * S::kSlot);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }

  // the waves' sums, added in their order
  __syncthreads();
  float *part = reinterpret_cast<float *>(lds);
#pragma unroll
  for (int j = 0; j < S::FN; ++j)
    *reinterpret_cast<typename Op::acc *>(part + wave * (S::BM * BN) + (lane & 15) * BN + j * 16 +
                                          (lane >> 4) * 4) = acc[0][j];
  __syncthreads();
  for (int q = tid; q < S::BM * BN / 4; q += NW * 64) {
    const int row = q / (BN / 4), col = q % (BN / 4) * 4;
    const int s = r.lo + row;
    if (s >= r.hi || n0 + col >= g.n) continue;
    typename Op::acc sum = *reinterpret_cast<typename Op::acc *>(part + q * 4);
#pragma unroll
    for (int w = 1; w < NW; ++w)
      sum += *reinterpret_cast<typename Op::acc *>(part + w * (S::BM * BN) + q * 4);
    float v[4];
    float as = 1.f;
    if constexpr (Op::kInt) as = g.a_scale[slot_row(g.a_rows, g.n_a, s)];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      v[c] = static_cast<float>(sum[c]);
      const int n = n0 + col + c;
      if constexpr (Op::kInt)
        v[c] = scaled(v[c], as,
                      g.b_scale[static_cast<int64_t>(r.group) * g.n + (n < g.n ? n : g.n - 1)]);
    }
    put4(g.c, g.out, s * g.ldc, n0 + col, g.n, v);
  }
#endif
}

// Results from the sums of the parts, added in their order: element (row, col)
// of group-major rows, m to a group, goes to c_group, ldc.  Rows of no group
// (offsets given) are zero already.  Bound by its launch: 3.5 us for 16 parts
// of 128 x 128.
static __global__ __launch_bounds__(256) void grouped_join_kernel(GroupedArgs g, int64_t rows,
                                                                  int64_t m, bool skip_dead) {
  const int64_t quads = (g.n + 3) / 4, i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= rows * quads) return;
  const int64_t row = i / quads;
  const int col = static_cast<int>(i % quads) * 4;
  if (skip_dead && g.offsets && (row < g.offsets[0] || row >= g.offsets[g.n_groups])) return;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
  const float *src = g.partial + row * g.n + col;
  const int64_t part = rows * g.n;
  if (g.n % 4 == 0) {
#pragma unroll 8
    for (int p = 0; p < g.splits; ++p)
      sum += *reinterpret_cast<const f32x4_t *>(src + p * part);
  } else {
    for (int p = 0; p < g.splits; ++p)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (col + c < g.n) sum[c] += src[p * part + c];
  }
  const float v[4] = {sum[0], sum[1], sum[2], sum[3]};
  put4(g.c, g.out, row / m * g.c_group + row % m * g.ldc, col, g.n, v);
}

}  // namespace ej
