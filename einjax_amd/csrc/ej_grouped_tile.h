// Tile kernels of the products grouped by expert: BM x BN results per
// workgroup, WR x WC waves, a ring of NS stages in LDS.
#pragma once

#include "ej_gated.h"
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

template <class Op, int BM, int BN, int WR, int WC, bool AKC, bool BKC, int LOADS, int NS>
struct TileShape {
  using elem = typename Op::elem;
  static constexpr int kWaves = WR * WC;
  static constexpr int kThreads = kWaves * 64;
  static constexpr int kRows = BM, kCols = BN;
  static constexpr int WM = BM / WR, WN = BN / WC;
  static constexpr int FM = WM / 16, FN = WN / 16;
  using TA = Tile<Op, BM, AKC>;
  using TB = Tile<Op, BN, BKC>;
  using FA = Fragments<Op, TA, AKC, FM>;
  using FB = Fragments<Op, TB, BKC, FN>;
  using LA = Loader<Op, BM, AKC, kWaves, LOADS>;
  using LB = Loader<Op, BN, BKC, kWaves, LOADS>;
  // scales of a stage, one a thread: the tile's rows', then its columns'
  static constexpr int kScaleAt = TA::kBytes + TB::kBytes;
  static constexpr int kScales = kBlocks<Op> ? kThreads * 4 : 0;
  static_assert(!kBlocks<Op> || BM + BN <= kThreads, "a thread for each scale");
  static constexpr int kSlot = TA::kBytes + TB::kBytes + kScales;
  // NS == 0: the pipelined loops' rings
  static constexpr int kPieces = LA::kLoads;  // of 64 rows (blocks): run_blocks
  static constexpr int kLds = NS > 0           ? NS * kSlot
                              : !kBlocks<Op> ? 3 * TA::kBytes + 2 * TB::kBytes
                                             : (3 * kPieces - 1) * 8192 + 2 * TB::kBytes +
                                                   4 * kScales;
  static constexpr int kLoads = LA::kLoads + LB::kLoads + (kBlocks<Op> ? 1 : 0);
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

// This lane's places among a stage's scales: its row in the first fragment, and
// the wave's columns, which lie in one block of 128.
struct ScalePlace {
  uint32_t row, col;
  __device__ inline void init(uint32_t base, int rows, int row0, int col0, int lane) {
    row = base + (row0 + (lane & 15)) * 4;
    col = base + (rows + col0) * 4;
  }
  __device__ static inline float at(uint32_t lds) {
    return *reinterpret_cast<const __attribute__((address_space(3))) float *>(
        (lds_u8 *)(size_t)lds);
  }
};

// acc[i][j] += (A fragment i times B fragment j over one block of 128) times
// the product of their scales.
template <class Op, class S>
__device__ inline void stage_blocks(f32x4_t (&acc)[S::FM][S::FN], const typename S::FA &fa,
                                    const typename S::FB &fb, const ScalePlace &scales,
                                    uint32_t slot) {
  static_assert(128 % (S::FN * 16) == 0, "a wave's columns lie in one block");
  BlockFragment<Op> b[S::FN];
#pragma unroll
  for (int j = 0; j < S::FN; ++j) b[j].set(fb.read(slot, j, 0), fb.read(slot, j, 1));
  const float bs = ScalePlace::at(scales.col + slot);
#pragma unroll
  for (int i = 0; i < S::FM; ++i) {
    BlockFragment<Op> a;
    a.set(fa.read(slot, i, 0), fa.read(slot, i, 1));
    const float s = ScalePlace::at(scales.row + slot + i * 64) * bs;
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
      const f32x4_t t = mma_block(b[j], a);
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][j][c] = fmaf(t[c], s, acc[i][j][c]);
    }
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
template <class Op, class S, int LOADS, int NS, class Load, class Store>
__device__ inline void run_stages(typename Op::acc (&acc)[S::FM][S::FN], unsigned char *ring,
                                  int stages, int row0, int col0, int lane, Load load_stage,
                                  Store store_stage) {
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<size_t>((lds_u8 *)ring));
  typename S::FA fa;
  typename S::FB fb;
  fa.init(base, row0, lane);
  fb.init(base + S::TA::kBytes, col0, lane);
  ScalePlace scales;
  if constexpr (kBlocks<Op>) scales.init(base + S::kScaleAt, S::kRows, row0, col0, lane);
  auto stage = [&](uint32_t slot) {
    if constexpr (kBlocks<Op>) stage_blocks<Op, S>(acc, fa, fb, scales, slot);
    else stage_mma<Op, S>(acc, fa, fb, slot);
  };
  auto load_all = [&](int st, unsigned char *slot) {
#pragma unroll
    for (int v = 0; v < S::kLoads; ++v) load_stage(v, st, slot, true);
  };
  if constexpr (LOADS == kLoadDirect && NS == 0) {
    run_pipelined<Op, S>(acc, ring, stages, fa, fb, load_stage);
  } else if constexpr (LOADS == kLoadDirect) {
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
      stage(get * S::kSlot);
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
      stage((st & 1) * S::kSlot);
      if (st + 1 < stages) store_stage(ring + ((st + 1) & 1) * S::kSlot);
    }
  }
}

// The results of a wave: row(i, &at) gives the element offset of fragment row
// i's results and whether there is such a row, value(i, j, c) its result c of
// four in fragment column j.
template <class S, int FN = S::FN, class Row, class Value>
__device__ inline void put_results(const GroupedArgs &g, int col0, int lane, Row row,
                                   Value value) {
  if (FN % 2 == 0 && g.out != EJ_F32) {
#pragma unroll
    for (int i = 0; i < S::FM; ++i) {
      int64_t at;
      const bool there = row(i, &at);
#pragma unroll
      for (int j = 0; j + 1 < FN; j += 2) {
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
    for (int j = 0; j < FN; ++j) {
      const int col = col0 + j * 16 + (lane >> 4) * 4;
      if (col >= g.n) continue;
      float v[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = value(i, j, c);
      put4(g.c, g.out, at, col, g.n, v);
    }
  }
}

// The gated results of a wave: fragment columns j of the gate and j + FN / 2 of
// the other projection give columns col0 + 16 j on; row0 is the slot of the
// wave's first row.  With the contraction in parts, their sums instead.  8192 x
// 4096 x 8192 bf16 in large blocks: 392 us (1400 TFLOP/s; the product of the same
// extents alone 400 to 435), with both projections kept in fp32 438: the stores of a
// block stand behind its last products.
template <class S, class Acc>
__device__ inline void put_gated(const GroupedArgs &g, int col0, int lane, int row0, int hi,
                                 const Acc &acc) {
  constexpr int H = S::FN / 2;
  float *both = g.splits > 1 ? g.partial + blockIdx.y * g.slots * (2 * static_cast<int64_t>(g.n))
                             : g.gate_up;
  if (both) {
#pragma unroll
    for (int i = 0; i < S::FM; ++i) {
      const int s = row0 + i * 16 + (lane & 15);
      if (s >= hi) continue;
      const int64_t at = s * (2 * static_cast<int64_t>(g.n));
#pragma unroll
      for (int j = 0; j < S::FN; ++j) {
        const int col = col0 + j % H * 16 + (lane >> 4) * 4;
        if (col >= g.n) continue;
        const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        put4(both, EJ_F32, at + j / H * static_cast<int64_t>(g.n), col, g.n, v);
      }
    }
  }
  if (g.splits > 1 || !g.c) return;
  auto put = [&](auto act) {
    put_results<S, H>(
        g, col0, lane,
        [&](int i, int64_t *at) {
          const int s = row0 + i * 16 + (lane & 15);
          *at = s * g.ldc;
          return s < hi;
        },
        [&](int i, int j, int c) { return act(acc[i][j][c]) * acc[i][j + H][c]; });
  };
  by_activation<sizeof(typename S::elem) == 4>(g.activation, put);
}

// Gated products: the columns of B that a tile of BN holds are, for each WN of
// them that a wave takes, WN / 2 of the gate and the same ones of the other
// projection, so that both of a result's factors end in one lane.  Column of
// the tile's results from n0 on, and where its half of B begins.
template <int WN>
__device__ inline int gated_col(int i, int n0, int n, int *shift) {
  const int in = i % WN;
  *shift = in < WN / 2 ? 0 : n;
  return n0 + i / WN * (WN / 2) + in % (WN / 2);
}

// The scales of a stage: thread t's is that of row t of the tile, or of column
// t - rows.
struct ScaleLoader {
  const float *src;
  float held;
  __device__ inline void init(const GroupedArgs &g, const RowBlock &r, int rows, int cols, int n0,
                              int t, int st) {
    const int64_t k_blocks = (g.k + 127) / 128;
    if (t < rows) {
      const int s = r.lo + t < r.hi ? r.lo + t : r.hi - 1;
      src = g.a_scale + slot_row(g.a_rows, g.n_a, s) * k_blocks + st;
    } else {
      int n = n0 + (t - rows < cols ? t - rows : cols - 1);
      n = n < g.n ? n : g.n - 1;
      const int64_t n_blocks = (g.n + 127) / 128;
      src = g.b_scale + (r.group * n_blocks + n / 128) * k_blocks + st;
    }
  }
  // The next stage's, `step` stages on from the one before.
  template <int LOADS>
  __device__ inline void load(unsigned char *to, int wave, int step) {
    if constexpr (LOADS == kLoadDirect) load_word_to_lds(src, lds_address(to) + wave * 256);
    else held = *src;
    src += step;
  }
  __device__ inline void store(unsigned char *to, int t) const {
    *reinterpret_cast<float *>(to + t * 4) = held;
  }
};

// Loads of a K tile's stages, and of the scales', at 32 bits from a uniform address.
template <int ROWS, int NW>
struct NearLoader {
  static constexpr int kLoads = ROWS * kRowB / 1024 / NW;
  static_assert(NW % 2 == 0, "one chunk of a row for each lane");
  const char *base;
  uint32_t off[kLoads];
  int line;  // first k element of the lane's chunk
  // row_off(i): offset of output row i from `from`
  template <class RowOff>
  __device__ inline void init(const char *from, int wave, int lane, RowOff row_off) {
    base = from;
#pragma unroll
    for (int v = 0; v < kLoads; ++v) {
      int row, chunk;
      Tile<OpF8, ROWS, true>::at((v * NW + wave) * 64 + lane, &row, &chunk);
      line = chunk * 16;
      off[v] = row_off(row) + chunk * 16;
    }
  }
  // Load v of stage st, of which `left` elements of k exist, to the tile at `lds`.
  __device__ inline void load(int v, int st, uint32_t lds, int wave, int left, bool part) const {
    const char *at = base + static_cast<int64_t>(st) * kRowB;
    const uint32_t to = lds + (v * NW + wave) * 1024;
    if (!part) {
      load_to_lds(at, off[v], to);
    } else {
      load_to_lds(line < left ? at + off[v] : reinterpret_cast<const char *>(&grouped_zeros), to);
    }
  }
};

// Row of the tile whose scale is t-th among a stage's in blocks_256: a lane's two
// of a pair of fragments lie side by side.
template <class S>
__device__ inline int blocks_row(int t) {
  const int r = t % S::WM;
  return t / S::WM * S::WM + (r / 32 * 2 + (r & 1)) * 16 + (r % 32) / 2;
}

// The pipelined loop of block-scaled products.  A wave takes its rows two
// fragments (a pair) at a time, which it reads while the pair before is
// multiplied; the fragments of its columns stay in registers for the stage:
//   pairs but the last:  read the next pair; load most of A and the scales of
//                        stage st + 2
//   every wave has read stage st and stage st + 1 has landed: one barrier
//   last pair:           read the first pair and, one by one as they become
//                        free, the columns of stage st + 1; load B and the last
//                        64 rows of A of stage st + 2
// so that no fragment is waited for behind the barrier and loads are under way
// all the time (see run_pipelined).  A lies in pieces of 64 rows in a ring of
// one piece less than three stages, which leaves the room for the scales.
// Its loads go by offsets of 32 bits: a pointer for each load in each lane would
// take a fifth of the vector instructions' time, which scaling the sums needs.
// 16384 rows in 8 groups, k = n = 4096: 245 us (2240 TFLOP/s; 272 with pointers).
// Bound by the issue of instructions: beside a matrix instruction (16 x 16 x 128,
// 13.8 ns in two waves a SIMD) four multiply-adds, the scaling, are free; with six it
// takes 18 ns, with eight 19.6.
template <class Op, class S>
__device__ inline void run_blocks(f32x4_t (&acc)[S::FM][S::FN], unsigned char *ring,
                                  const GroupedArgs &g, const RowBlock &r, int n0, int row0,
                                  int col0, int wave, int lane) {
  constexpr int kPieces = S::kPieces, kSlots = 3 * kPieces - 1, kPiece = 8192;
  constexpr int kB = kSlots * kPiece, kScale = kB + 2 * S::TB::kBytes;
  constexpr int kPairs = S::FM / 2, kLate = kPieces;  // kPieces - 1 of A and the scales
  static_assert(S::WM % 64 == 0 && S::FM % 4 == 0, "whole pieces of a wave");
  const int stages = (g.k + 127) / 128, k_left = g.k;
  NearLoader<S::kRows, S::kWaves> la;
  NearLoader<S::kCols, S::kWaves> lb;
  // rows that follow each other: from the block's first
  const int64_t row_from = g.a_rows ? 0 : r.lo < g.n_a ? r.lo : g.n_a - 1;
  auto near_row = [&](int i) {
    const int s = r.lo + i < r.hi ? r.lo + i : r.hi - 1;
    return static_cast<uint32_t>(slot_row(g.a_rows, g.n_a, s) - row_from);
  };
  auto near_col = [&](int i) { return static_cast<uint32_t>(n0 + i < g.n ? i : g.n - 1 - n0); };
  la.init(g.a + row_from * g.lda, wave, lane,
          [&](int i) { return near_row(i) * static_cast<uint32_t>(g.lda); });
  lb.init(g.b + r.group * g.b_group + n0 * g.ldb, wave, lane,
          [&](int i) { return near_col(i) * static_cast<uint32_t>(g.ldb); });
  // scales of rows in the first waves, of columns in the others
  const char *scale_base;
  uint32_t scale_off;
  if (wave * 64 < S::kRows) {
    scale_base = reinterpret_cast<const char *>(g.a_scale + row_from * stages);
    scale_off = near_row(blocks_row<S>(wave * 64 + lane)) * stages * 4;
  } else {
    const int64_t n_blocks = (g.n + 127) / 128;
    const int i = wave * 64 + lane - S::kRows, n = n0 + (i < S::kCols ? i : 0);
    scale_base = reinterpret_cast<const char *>(g.b_scale + (r.group * n_blocks) * stages);
    scale_off = static_cast<uint32_t>((n < g.n ? n : g.n - 1) / 128) * stages * 4;
  }
  if (stages == 0) return;
  const uint32_t base = lds_address(ring);
  typename S::FA fa;
  typename S::FB fb;
  fa.init(base, 0, lane);
  fb.init(base + kB, col0, lane);
  const uint32_t row_scale = base + kScale + row0 * 4 + (lane & 15) * 8;
  const uint32_t col_scale = base + kScale + (S::kRows + col0) * 4;
  const int piece0 = row0 / 64;
  // slot of piece q of the stage whose first piece lies in slot `first`
  auto slot_of = [&](int first, int q) {
    const int s = first + q;
    return s < kSlots ? s : s < 2 * kSlots ? s - kSlots : s - 2 * kSlots;
  };
  auto load_a = [&](int q, int st, int first, bool part) {
    la.load(q, st, base + (slot_of(first, q) - q) * kPiece, wave, k_left - st * 128, part);
  };
  auto load_b = [&](int v, int st, bool part) {
    lb.load(v, st, base + kB + (st & 1) * S::TB::kBytes, wave, k_left - st * 128, part);
  };
  auto load_scales = [&](int st, bool part) {
    const int there = !part || st < stages ? st : stages - 1;
    load_word_to_lds(scale_base + there * 4ll, scale_off,
                     base + kScale + (st & 3) * S::kScales + wave * 256);
  };
  BlockFragment<Op> a[2][2], b[S::FN];
  f32x2_t as[2] = {};
  float bs;
  auto read_a = [&](int first, int p, int h) {
    const uint32_t off = slot_of(first, piece0 + p / 2) * kPiece;
    const int i = p % 2 * 2 + h;
    a[p & 1][h].set(fa.read(off, i, 0), fa.read(off, i, 1));
  };
  auto read_b = [&](int j, int st) {
    const uint32_t off = (st & 1) * S::TB::kBytes;
    b[j].set(fb.read(off, j, 0), fb.read(off, j, 1));
  };
  auto read_scales = [&](int st, int p) {
    as[p & 1] = *reinterpret_cast<const __attribute__((address_space(3))) f32x2_t *>(
        (lds_u8 *)(size_t)(row_scale + (st & 3) * S::kScales + p * 128));
    if (p == 0) bs = ScalePlace::at(col_scale + (st & 3) * S::kScales);
  };
  // stages past the end are zeros, loaded from one cached line
  int first = 0, first1 = kPieces;  // slots of the first pieces of stages st and st + 1
#pragma unroll
  for (int q = 0; q < kPieces; ++q) load_a(q, 0, first, true);
#pragma unroll
  for (int v = 0; v < S::LB::kLoads; ++v) load_b(v, 0, true);
  load_scales(0, true);
#pragma unroll
  for (int q = 0; q < kPieces - 1; ++q) load_a(q, 1, first1, true);
  load_scales(1, true);
  load_a(kPieces - 1, 1, first1, true);
#pragma unroll
  for (int v = 0; v < S::LB::kLoads; ++v) load_b(v, 1, true);
  wait_vm<kLate + 1 + S::LB::kLoads>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  read_a(first, 0, 0);
  read_a(first, 0, 1);
  read_scales(0, 0);
#pragma unroll
  for (int j = 0; j < S::FN; ++j) read_b(j, 0);
  // steps of a stage: the matrix instructions of a pair and one fragment of
  // columns; their sums are scaled and added up a step later, while the next
  // ones are formed
  constexpr int kSteps = kPairs * S::FN, kLastPair = kSteps - S::FN;
  f32x4_t t[2][2] = {};
  auto add_sums = [&](int step, int h) {
    const int p = step / S::FN, j = step % S::FN;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      acc[2 * p + h][j][c] = fmaf(t[step & 1][h][c], as[p & 1][h], acc[2 * p + h][j][c]);
  };
  int st = 0;
  auto stage = [&](auto kWhole) {
    constexpr bool part = !decltype(kWhole)::value;
    const int first2 = slot_of(first1, kPieces);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int p = s / S::FN, j = s % S::FN;
      if (s == kLastPair) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLate) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      }
      // (of none yet: zeros)
      constexpr int kEnd = kSteps - 1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        t[s & 1][h] = mma_block(b[j], a[p & 1][h]);
        __builtin_amdgcn_sched_barrier(0);
        add_sums(s > 0 ? s - 1 : kEnd, h);
        if (h == 0) __builtin_amdgcn_sched_barrier(0);
      }
      if (s < kLastPair) {
        if (j < 2) read_a(first, p + 1, j);
        if (j == 1) read_scales(st, p + 1);
        // the late loads of stage st + 2
        if (s % (kLastPair / kLate) == 0) {
          constexpr int kEach = kLastPair / kLate;
          if (s / kEach < kPieces - 1) load_a(s / kEach, st + 2, first2, part);
          else if (s / kEach == kPieces - 1) load_scales(st + 2, part);
        }
      } else {
        read_b(j, st + 1);
        if (j < 2) read_a(first1, 0, j);
        if (j == 1) read_scales(st + 1, 0);
        if (j < S::LB::kLoads) load_b(j, st + 2, part);
        if (j == 0) load_a(kPieces - 1, st + 2, first2, part);
      }
      if (j == 0) as[p & 1] *= bs;
      __builtin_amdgcn_sched_barrier(0);
    }
    first = first1;
    first1 = first2;
    ++st;
  };
  static_assert(S::LB::kLoads <= S::FN && S::FN >= 2 && kPairs % 2 == 0 && kSteps % 2 == 0 &&
                    kLastPair % kLate == 0,
                "loads, buffers and reads of the steps");
  while (st + 3 < stages) stage(std::true_type());
  while (st < stages) stage(std::false_type());
  add_sums(kSteps - 1, 0);
  add_sums(kSteps - 1, 1);
  // no load may still be writing LDS when the workgroup ends
  wait_vm<0>();
}

// C rows of one row block of a group times the BN columns from n0; GATED: the
// BN / 2 gated columns from n0.
template <class Op, int BM, int BN, int WR, int WC, bool BKC, int LOADS, int NS,
          bool GATED = false>
__device__ inline void rows_block(GroupedArgs g, const RowBlock &r, int n0, unsigned char *ring) {
  using S = TileShape<Op, BM, BN, WR, WC, true, BKC, LOADS, NS>;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row0 = wave / WC * S::WM, col0 = wave % WC * S::WN;
  typename Op::acc acc[S::FM][S::FN];
#pragma unroll
  for (int i = 0; i < S::FM; ++i)
#pragma unroll
    for (int j = 0; j < S::FN; ++j) acc[i][j] = typename Op::acc{0, 0, 0, 0};
  if constexpr (kBlocks<Op> && NS == 0) {
    run_blocks<Op, S>(acc, ring, g, r, n0, row0, col0, wave, lane);
    put_results<S>(
        g, n0 + col0, lane,
        [&](int i, int64_t *at) {
          const int s = r.lo + row0 + i * 16 + (lane & 15);
          *at = s * g.ldc;
          return s < r.hi;
        },
        [&](int i, int j, int c) { return acc[i][j][c]; });
    return;
  }
  int st0, st1;
  part_of((g.k + kStep<Op> - 1) / kStep<Op>, blockIdx.y, g.splits, &st0, &st1);
  const int64_t k0 = static_cast<int64_t>(st0) * kStep<Op>;
  const int ks = g.k - static_cast<int>(k0);  // k left from the part's start

  typename S::LA la;
  typename S::LB lb;
  la.init_k(wave, lane, [&](int i) {
    const int s = r.lo + i < r.hi ? r.lo + i : r.hi - 1;
    return g.a + (slot_row(g.a_rows, g.n_a, s) * g.lda + k0) * kElem<Op>;
  });
  const char *bg = g.b + r.group * g.b_group * kElem<Op>;
  int64_t b_step;
  if constexpr (BKC) {
    lb.init_k(wave, lane, [&](int i) {
      int shift = 0, n = n0 + i;
      if constexpr (GATED) n = gated_col<S::WN>(i, n0, g.n, &shift);
      n = n < g.n ? n : g.n - 1;
      return bg + (static_cast<int64_t>(n + shift) * g.ldb + k0) * kElem<Op>;
    });
    b_step = kRowB;
  } else {
    if constexpr (GATED)
      lb.init_m(wave, lane, bg + k0 * g.ldb * kElem<Op>, g.ldb, g.n,
                [&](int i, int *shift) { return gated_col<S::WN>(i, n0, g.n, shift); });
    else
      lb.init_m(wave, lane, bg + k0 * g.ldb * kElem<Op>, g.ldb, n0, g.n);
    b_step = kStep<Op> * g.ldb * kElem<Op>;
  }

  ScaleLoader scales;
  if constexpr (kBlocks<Op>) scales.init(g, r, BM, BN, n0, tid, st0);

  run_stages<Op, S, LOADS, NS>(
      acc, ring, st1 - st0, row0, col0, lane,
      [&](int v, int st, unsigned char *slot, bool part) {
        const int left = ks - st * kStep<Op>;
        if (v < S::LA::kLoads)
          la.load(v, slot, wave, left, kRowB, part);
        else if (v < S::LA::kLoads + S::LB::kLoads)
          lb.load(v - S::LA::kLoads, slot + S::TA::kBytes, wave, left, b_step, part);
        else
          scales.load<LOADS>(slot + S::kScaleAt, wave, 1);
      },
      [&](unsigned char *slot) {
        la.store(slot, wave, lane);
        lb.store(slot + S::TA::kBytes, wave, lane);
        if constexpr (kBlocks<Op>) scales.store(slot + S::kScaleAt, tid);
      });

  if constexpr (GATED) {
    put_gated<S>(g, n0 + wave % WC * (S::WN / 2), lane, r.lo + row0, r.hi, acc);
    return;
  }
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
// registers: 29 us, 21 us at aligned extents; the rest are another column of
// tiles and stage of k, and the unaligned loads, two lines for most of them.
// Loads at words with the bytes moved into place when they are stored, the last
// word from the next lane, took 31.
template <class Op, int BM, int BN, int WR, int WC, bool BKC, int LOADS, int NS, bool GATED>
__global__ __launch_bounds__(WR *WC * 64) void grouped_rows_kernel(GroupedArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using S = TileShape<Op, BM, BN, WR, WC, true, BKC, LOADS, NS>;
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
  rows_block<Op, BM, BN, WR, WC, BKC, LOADS, NS, GATED>(g, find_row_block(g, BM, rb),
                                                         cb * (GATED ? BN / 2 : BN), ring);
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
template <class Op, bool BKC, bool GATED>
__global__ __launch_bounds__(512) void grouped_large_kernel(GroupedArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using S = TileShape<Op, 256, 256, 2, 4, true, BKC, kLoadDirect, 0>;
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
  const int n0 = (cb * 256 + u.col) / (GATED ? 2 : 1);
  if (r.lo >= r.hi || n0 >= g.n) return;
  if (u.parts == 4)
    rows_block<Op, 128, 128, 2, 4, BKC, kLoadDirect, 0, GATED>(g, r, n0, ring);
  else if (u.parts == 2 || r.hi - r.lo <= 128)
    rows_block<Op, 128, 256, 2, 4, BKC, kLoadDirect, 0, GATED>(g, r, n0, ring);
  else
    rows_block<Op, 256, 256, 2, 4, BKC, kLoadDirect, 0, GATED>(g, r, n0, ring);
#endif
}

// D_e block: the BM columns of P from m0 (rows of the result) by the BN
// columns of Q from n0, over the slots of a group; one without slots writes
// zeros.  GATHER: 1 if P's rows go through an index, 2 if Q's do.
template <class Op, int BM, int BN, int WR, int WC, int LOADS, int NS, int GATHER>
__device__ inline void wgrad_block(GroupedArgs g, int group, int m0, int n0, unsigned char *ring) {
  using S = TileShape<Op, BM, BN, WR, WC, false, false, LOADS, NS>;
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
  // The gathered operand's rows of a stage, lane by lane, read a stage ahead.
  // Their bounds are checked when they are used: that waits for their load, and
  // with it for the loads before it.
  const int32_t *rows = GATHER == 1 ? g.a_rows : g.b_rows;
  const int64_t n_rows = GATHER == 1 ? g.n_a : g.n_b;
  auto rows_of = [&](int st) {
    const int64_t s = lo + static_cast<int64_t>(st) * kStep<Op> + lane;
    return rows[s < hi ? s : hi - 1];
  };
  auto in_bounds = [&](int r) {
    return r < 0 ? 0 : r < n_rows ? r : static_cast<int>(n_rows - 1);
  };
  int row_now = 0, row_next = 0;
  if (GATHER && st1 > st0) row_next = rows_of(0);

  typename Op::acc acc[S::FM][S::FN];
#pragma unroll
  for (int i = 0; i < S::FM; ++i)
#pragma unroll
    for (int j = 0; j < S::FN; ++j) acc[i][j] = typename Op::acc{0, 0, 0, 0};
  run_stages<Op, S, LOADS, NS>(
      acc, ring, st1 - st0, row0, col0, lane,
      [&](int v, int st, unsigned char *slot, bool part) {
        const int left = hi - lo - st * kStep<Op>;
        // all sources of the gathered operand at its first load: the lane
        // moves wait for every LDS read before them
        if (v < S::LA::kLoads) {
          if constexpr (GATHER == 1) {
            if (v == 0) {
              row_now = in_bounds(row_next);
              row_next = rows_of(st + 1);
              la.seek(g.a, g.lda, row_now);
            }
          }
          la.load(v, slot, wave, left, kStep<Op> * g.lda * kElem<Op>, part);
        } else {
          const int u = v - S::LA::kLoads;
          if constexpr (GATHER == 2) {
            if (u == 0) {
              row_now = in_bounds(row_next);
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
template <class Op, int BM, int BN, int WR, int WC, int LOADS, int NS, int GATHER>
__global__ __launch_bounds__(WR *WC * 64) void grouped_wgrad_kernel(GroupedArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using S = TileShape<Op, BM, BN, WR, WC, false, false, LOADS, NS>;
  __shared__ __align__(1024) unsigned char ring[S::kLds];
  const uint32_t per = g.row_blocks * g.col_blocks;
  // runs of blocks dealt to the XCDs in turn: as one part each, the XCD of the
  // longest group ends last (16384 rows in 16 groups of unequal length, 2048 x
  // 4096 bf16, 256 x 256: 363 us so, 305 dealt; groups of equal length 285 and
  // 287)
  const uint32_t block = xcd_logical_block(gridDim.x, kXcdRun), group = block / per;
  int rb, cb;
  band_pos(block - group * per, g.row_blocks, g.col_blocks, 1024 / BM, &rb, &cb);
  wgrad_block<Op, BM, BN, WR, WC, LOADS, NS, GATHER>(g, group, rb * BM, cb * BN, ring);
#endif
}

// The same in blocks of 256 x 256, cut as grouped_large_kernel's.  16384 rows
// in 16 groups, 2048 x 4096 bf16: 269 us (1020 TFLOP/s), 300 with P gathered
// (bounds checked as soon as the index is loaded: 316).  A lane that uses an
// index waits for its load, and with it for the loads of the other operand issued
// before: each stage drains half of the ring.  Indices through the scalar cache
// took 321 to 400: with scalar loads under way every wait for LDS is one for all.
template <class Op, int GATHER>
__global__ __launch_bounds__(512) void grouped_wgrad_large_kernel(GroupedArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using S = TileShape<Op, 256, 256, 2, 4, false, false, kLoadDirect, 0>;
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
    wgrad_block<Op, 128, 128, 2, 4, kLoadDirect, 0, GATHER>(g, group, m0, n0, ring);
  else if (u.parts == 2 || g.m - m0 <= 128)
    wgrad_block<Op, 128, 256, 2, 4, kLoadDirect, 0, GATHER>(g, group, m0, n0, ring);
  else
    wgrad_block<Op, 256, 256, 2, 4, kLoadDirect, 0, GATHER>(g, group, m0, n0, ring);
#endif
}

// Columns col .. col + 3 of slot s from the sums of both projections.
template <bool FINE>
__device__ inline void put_gated_quad(const GroupedArgs &g, int64_t s, int col, const f32x4_t &gate,
                                      const f32x4_t &up) {
  const int64_t at = s * (2 * static_cast<int64_t>(g.n));
  if (g.gate_up) {
    const float a[4] = {gate[0], gate[1], gate[2], gate[3]}, b[4] = {up[0], up[1], up[2], up[3]};
    put4(g.gate_up, EJ_F32, at, col, g.n, a);
    put4(g.gate_up, EJ_F32, at + g.n, col, g.n, b);
  }
  if (!g.c) return;
  by_activation<FINE>(g.activation, [&](auto act) {
    const float v[4] = {act(gate[0]) * up[0], act(gate[1]) * up[1], act(gate[2]) * up[2],
                        act(gate[3]) * up[3]};
    put4(g.c, g.out, s * g.ldc, col, g.n, v);
  });
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
  using LA = Loader<Op, BM, true, 1, kLoadDirect>;
  using LB = Loader<Op, BN, BKC, 1, kLoadDirect>;
  static constexpr int kRows = BM;
  static constexpr int kScaleAt = TA::kBytes + TB::kBytes;
  static_assert(!kBlocks<Op> || BM + BN <= 64, "a lane for each scale");
  static constexpr int kSlot = TA::kBytes + TB::kBytes + (kBlocks<Op> ? 256 : 0);
  static constexpr int kLoads = LA::kLoads + LB::kLoads + (kBlocks<Op> ? 1 : 0);
  static constexpr int kRing = NS * kSlot;
  static constexpr int kPart = BM * BN * 4;  // bytes of a wave's sums
  static constexpr int kLds = NW * (kRing > kPart ? kRing : kPart);
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
};

template <class Op, int BN, int NW, bool BKC, int NS, bool GATED>
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
  const int n0 = cb * (GATED ? BN / 2 : BN);
  unsigned char *ring = lds + wave * S::kRing;

  typename S::LA la;
  typename S::LB lb;
  const int stages = (g.k + kStep<Op> - 1) / kStep<Op>;
  const int mine = stages > wave ? (stages - wave + NW - 1) / NW : 0;
  const int64_t k0 = static_cast<int64_t>(wave) * kStep<Op>;
  la.init_k(0, lane, [&](int i) {
    const int s = r.lo + i < r.hi ? r.lo + i : r.hi - 1;
    return g.a + (slot_row(g.a_rows, g.n_a, s) * g.lda + k0) * kElem<Op>;
  });
  const char *bg = g.b + r.group * g.b_group * kElem<Op>;
  int64_t b_step;
  if constexpr (BKC) {
    lb.init_k(0, lane, [&](int i) {
      int shift = 0, n = n0 + i;
      if constexpr (GATED) n = gated_col<BN>(i, n0, g.n, &shift);
      n = n < g.n ? n : g.n - 1;
      return bg + (static_cast<int64_t>(n + shift) * g.ldb + k0) * kElem<Op>;
    });
    b_step = kRowB;
  } else {
    if constexpr (GATED)
      lb.init_m(0, lane, bg + k0 * g.ldb * kElem<Op>, g.ldb, g.n,
                [&](int i, int *shift) { return gated_col<BN>(i, n0, g.n, shift); });
    else
      lb.init_m(0, lane, bg + k0 * g.ldb * kElem<Op>, g.ldb, n0, g.n);
    b_step = kStep<Op> * g.ldb * kElem<Op>;
  }
  ScaleLoader scales;
  if constexpr (kBlocks<Op>) scales.init(g, r, S::BM, BN, n0, lane, wave);
  auto load = [&](int i) {
    unsigned char *slot = ring + i % NS * S::kSlot;
    const int left = g.k - (wave + i * NW) * kStep<Op>;
#pragma unroll
    for (int v = 0; v < S::LA::kLoads; ++v) la.load(v, slot, 0, left, NW * kRowB, true);
#pragma unroll
    for (int v = 0; v < S::LB::kLoads; ++v)
      lb.load(v, slot + S::TA::kBytes, 0, left, NW * b_step, true);
    if constexpr (kBlocks<Op>) scales.load<kLoadDirect>(slot + S::kScaleAt, 0, NW);
  };
  typename S::FA fa;
  typename S::FB fb;
  fa.init(lds_address(ring), 0, lane);
  fb.init(lds_address(ring) + S::TA::kBytes, 0, lane);
  ScalePlace place;
  if constexpr (kBlocks<Op>) place.init(lds_address(ring) + S::kScaleAt, S::BM, 0, 0, lane);
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
    if constexpr (kBlocks<Op>) stage_blocks<Op, S>(acc, fa, fb, place, i % NS * S::kSlot);
    else stage_mma<Op, S>(acc, fa, fb, i % NS * S::kSlot);
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
  if constexpr (GATED) {
    for (int q = tid; q < S::BM * BN / 8; q += NW * 64) {
      const int row = q / (BN / 8), col = q % (BN / 8) * 4;
      const int s = r.lo + row;
      if (s >= r.hi || n0 + col >= g.n) continue;
      f32x4_t sum[2] = {};
#pragma unroll
      for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          sum[h] += *reinterpret_cast<f32x4_t *>(part + w * (S::BM * BN) + row * BN +
                                                 h * (BN / 2) + col);
      put_gated_quad<kElem<Op> == 4>(g, s, n0 + col, sum[0], sum[1]);
    }
    return;
  }
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

// Gated results from the sums of the parts, added in their order.  Rows of no
// group (offsets given) are zero already.
template <bool FINE>
__global__ __launch_bounds__(256) void gated_join_kernel(GroupedArgs g) {
  const int64_t quads = (g.n + 3) / 4, i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= g.slots * quads) return;
  const int64_t row = i / quads;
  const int col = static_cast<int>(i % quads) * 4;
  if (g.offsets && (row < g.offsets[0] || row >= g.offsets[g.n_groups])) return;
  f32x4_t sum[2] = {};
  const float *src = g.partial + row * (2 * static_cast<int64_t>(g.n)) + col;
  const int64_t part = g.slots * (2 * static_cast<int64_t>(g.n));
  for (int p = 0; p < g.splits; ++p)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float *v = src + p * part + h * static_cast<int64_t>(g.n);
      if (g.n % 4 == 0) {
        sum[h] += *reinterpret_cast<const f32x4_t *>(v);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (col + c < g.n) sum[h][c] += v[c];
      }
    }
  put_gated_quad<FINE>(g, row, col, sum[0], sum[1]);
}

}  // namespace ej
