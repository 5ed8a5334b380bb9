// Tile kernels of the products grouped by expert: BM x BN results per
// workgroup, WR x WC waves, a ring of NS stages in LDS.
#pragma once

#include "ej_grouped.h"

namespace ej {

template <int N>
__device__ inline void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Waits until the oldest stage in flight has landed; `later` stages of LPS
// loads each were issued after it (at most NS - 2).
template <int NS, int LPS>
__device__ inline void wait_oldest(int later) {
  static_assert(NS >= 2 && NS <= 4 && (NS - 2) * LPS < 64, "ring depth");
  if constexpr (NS >= 4) {
    if (later >= 2) { wait_vm<2 * LPS>(); return; }
  }
  if constexpr (NS >= 3) {
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
  using LA = Loader<Op, BM, AKC, kWaves, DIRECT>;
  using LB = Loader<Op, BN, BKC, kWaves, DIRECT>;
  static constexpr int kSlot = TA::kBytes + TB::kBytes;
  static constexpr int kLds = NS * kSlot;
  static constexpr int kLoads = LA::kLoads + LB::kLoads;
};

// acc[i][j] += A fragment i times B fragment j over the stage at LDS address
// `slot`.  The B fragment gives the accumulator's register rows, so a lane
// ends with four consecutive columns of one row of the result.
template <class Op, class S>
__device__ inline void stage_mma(typename Op::acc (&acc)[S::FM][S::FN], uint32_t slot, int row0,
                                 int col0, int lane) {
#pragma unroll
  for (int slab = 0; slab < 2; ++slab) {
    i32v4_t a[S::FM], b[S::FN];
#pragma unroll
    for (int i = 0; i < S::FM; ++i) a[i] = S::TA::frag(slot, row0 + i * 16, slab, lane);
#pragma unroll
    for (int j = 0; j < S::FN; ++j)
      b[j] = S::TB::frag(slot + S::TA::kBytes, col0 + j * 16, slab, lane);
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
      for (int j = 0; j < S::FN; ++j) mma<Op>(acc[i][j], b[j], a[i]);
  }
}

// The ring: load_stage(st, slot pointer) starts the loads of stage st,
// store_stage(slot pointer) finishes them where they go through registers.
template <class Op, class S, bool DIRECT, int NS, class Load, class Store>
__device__ inline void run_stages(typename Op::acc (&acc)[S::FM][S::FN], unsigned char *ring,
                                  int stages, int row0, int col0, int lane, Load load_stage,
                                  Store store_stage) {
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<size_t>((lds_u8 *)ring));
  if constexpr (DIRECT) {
    int put = 0, get = 0;
    for (int st = 0; st < NS - 1 && st < stages; ++st) {
      load_stage(st, ring + put * S::kSlot);
      put = put + 1 == NS ? 0 : put + 1;
    }
    for (int st = 0; st < stages; ++st) {
      const int left = stages - 1 - st;
      wait_oldest<NS, S::kLoads>(left < NS - 2 ? left : NS - 2);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (st + NS - 1 < stages) {
        load_stage(st + NS - 1, ring + put * S::kSlot);
        put = put + 1 == NS ? 0 : put + 1;
      }
      stage_mma<Op, S>(acc, base + get * S::kSlot, row0, col0, lane);
      get = get + 1 == NS ? 0 : get + 1;
    }
  } else {
    if (stages > 0) {
      load_stage(0, ring);
      store_stage(ring);
    }
    for (int st = 0; st < stages; ++st) {
      __syncthreads();
      if (st + 1 < stages) load_stage(st + 1, ring);
      stage_mma<Op, S>(acc, base + (st & 1) * S::kSlot, row0, col0, lane);
      if (st + 1 < stages) store_stage(ring + ((st + 1) & 1) * S::kSlot);
    }
  }
}

// C rows of one row block of a group times one block of columns.
template <class Op, int BM, int BN, int WR, int WC, bool BKC, bool DIRECT, int NS>
__global__ __launch_bounds__(WR *WC * 64) void grouped_rows_kernel(GroupedArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using S = TileShape<Op, BM, BN, WR, WC, true, BKC, DIRECT, NS>;
  __shared__ __align__(1024) unsigned char ring[S::kLds];
  const uint32_t grid = g.row_blocks * g.col_blocks;
  if (blockIdx.x >= grid) {
    zero_dead_rows(g, blockIdx.x - grid, gridDim.x - grid);
    return;
  }
  const uint32_t rbs = live_row_blocks(g, BM), live = rbs * g.col_blocks;
  if (blockIdx.x >= live) return;
  int rb, cb;
  band_pos(xcd_logical_block(live), rbs, g.col_blocks, 1024 / BM, &rb, &cb);
  const RowBlock r = find_row_block(g, BM, rb);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row0 = wave / WC * S::WM, col0 = wave % WC * S::WN;
  const int n0 = cb * BN;

  typename S::LA la;
  typename S::LB lb;
  la.init_k(wave, lane, [&](int i) {
    const int s = r.lo + i < r.hi ? r.lo + i : r.hi - 1;
    return g.a + slot_row(g.a_rows, g.n_a, s) * g.lda * kElem<Op>;
  });
  const char *bg = g.b + r.group * g.b_group * kElem<Op>;
  int64_t b_step;
  if constexpr (BKC) {
    lb.init_k(wave, lane, [&](int i) {
      const int n = n0 + i < g.n ? n0 + i : g.n - 1;
      return bg + n * g.ldb * kElem<Op>;
    });
    b_step = kRowB;
  } else {
    lb.init_m(wave, lane, bg, g.ldb, n0, g.n);
    b_step = kStep<Op> * g.ldb * kElem<Op>;
  }

  typename Op::acc acc[S::FM][S::FN];
#pragma unroll
  for (int i = 0; i < S::FM; ++i)
#pragma unroll
    for (int j = 0; j < S::FN; ++j) acc[i][j] = typename Op::acc{0, 0, 0, 0};
  run_stages<Op, S, DIRECT, NS>(
      acc, ring, (g.k + kStep<Op> - 1) / kStep<Op>, row0, col0, lane,
      [&](int st, unsigned char *slot) {
        const int left = g.k - st * kStep<Op>;
        la.load(slot, wave, left, kRowB);
        lb.load(slot + S::TA::kBytes, wave, left, b_step);
      },
      [&](unsigned char *slot) {
        la.store(slot, wave, lane);
        lb.store(slot + S::TA::kBytes, wave, lane);
      });

  const bool vec = vec_rows(g);
#pragma unroll
  for (int i = 0; i < S::FM; ++i) {
    const int s = r.lo + row0 + i * 16 + (lane & 15);
    if (s >= r.hi) continue;
    float as = 1.f;
    if constexpr (Op::kInt) as = g.a_scale[slot_row(g.a_rows, g.n_a, s)];
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
      const int col = n0 + col0 + j * 16 + (lane >> 4) * 4;
      if (col >= g.n) continue;
      float v[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        v[c] = static_cast<float>(acc[i][j][c]);
        if constexpr (Op::kInt)
          v[c] *= as * g.b_scale[static_cast<int64_t>(r.group) * g.n +
                                 (col + c < g.n ? col + c : g.n - 1)];
      }
      put4(g.c, g.out, s * g.ldc, col, g.n, vec, v);
    }
  }
#endif
}

// D_e block: rows i of P's columns, columns j of Q's, over the slots of group
// e.  The bound row_blocks x col_blocks covers one group's D; the grid holds
// n_groups of them, and a group without slots writes zeros.
template <class Op, int BM, int BN, int WR, int WC, bool DIRECT, int NS>
__global__ __launch_bounds__(WR *WC * 64) void grouped_wgrad_kernel(GroupedArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using S = TileShape<Op, BM, BN, WR, WC, false, false, DIRECT, NS>;
  __shared__ __align__(1024) unsigned char ring[S::kLds];
  const uint32_t per = g.row_blocks * g.col_blocks;
  const uint32_t lb_ = xcd_logical_block(gridDim.x);
  const int group = lb_ / per;
  int rb, cb, lo, hi;
  band_pos(lb_ - group * per, g.row_blocks, g.col_blocks, 1024 / BM, &rb, &cb);
  group_range(g, group, &lo, &hi);
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row0 = wave / WC * S::WM, col0 = wave % WC * S::WN;

  typename S::LA la;
  typename S::LB lb;
  la.init_m(wave, lane, g.a, 0, rb * BM, g.m);
  lb.init_m(wave, lane, g.b, 0, cb * BN, g.n);
  int acol[S::LA::kLoads], bcol[S::LB::kLoads];
#pragma unroll
  for (int v = 0; v < S::LA::kLoads; ++v)
    acol[v] = static_cast<int>((la.src[v] - g.a) / kElem<Op>);
#pragma unroll
  for (int v = 0; v < S::LB::kLoads; ++v)
    bcol[v] = static_cast<int>((lb.src[v] - g.b) / kElem<Op>);

  typename Op::acc acc[S::FM][S::FN];
#pragma unroll
  for (int i = 0; i < S::FM; ++i)
#pragma unroll
    for (int j = 0; j < S::FN; ++j) acc[i][j] = typename Op::acc{0, 0, 0, 0};
  run_stages<Op, S, DIRECT, NS>(
      acc, ring, (hi - lo + kStep<Op> - 1) / kStep<Op>, row0, col0, lane,
      [&](int st, unsigned char *slot) {
        const int s0 = lo + st * kStep<Op>;
        la.seek_slots(g.a, g.lda, g.a_rows, g.n_a, s0, hi, acol);
        lb.seek_slots(g.b, g.ldb, g.b_rows, g.n_b, s0, hi, bcol);
        la.load(slot, wave, hi - s0, 0);
        lb.load(slot + S::TA::kBytes, wave, hi - s0, 0);
      },
      [&](unsigned char *slot) {
        la.store(slot, wave, lane);
        lb.store(slot + S::TA::kBytes, wave, lane);
      });

  const bool vec = vec_rows(g);
#pragma unroll
  for (int i = 0; i < S::FM; ++i) {
    const int row = rb * BM + row0 + i * 16 + (lane & 15);
    if (row >= g.m) continue;
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
      const int col = cb * BN + col0 + j * 16 + (lane >> 4) * 4;
      if (col >= g.n) continue;
      const float v[4] = {static_cast<float>(acc[i][j][0]), static_cast<float>(acc[i][j][1]),
                          static_cast<float>(acc[i][j][2]), static_cast<float>(acc[i][j][3])};
      put4(g.c, g.out, group * g.c_group + static_cast<int64_t>(row) * g.ldc, col, g.n, vec, v);
    }
  }
#endif
}

}  // namespace ej
