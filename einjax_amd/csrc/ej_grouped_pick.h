// Choice of tile for one operand type.
#pragma once

#include <cmath>

#include "ej_grouped_launch.h"
#include "ej_grouped_tile.h"

namespace ej {

inline int join_parts(const GroupedArgs &g, int64_t rows, int64_t m, bool skip_dead,
                      hipStream_t stream) {
  dim3 grid;
  EJ_TRY(grouped_grid(ceil_div(rows * ceil_div(g.n, 4), 256), 256, &grid));
  hipLaunchKernelGGL(grouped_join_kernel, grid, dim3(256), 0, stream, g, rows, m, skip_dead);
  EJ_LAUNCH_CHECK();
  return EJ_OK;
}

template <class Op, int BM, int BN, int WR, int WC, bool BKC, bool DIRECT, int NS>
int launch_rows(GroupedArgs g, hipStream_t stream) {
  const int64_t groups = g.n_groups < g.slots ? g.n_groups : g.slots;
  g.row_blocks = static_cast<uint32_t>(g.slots / BM + groups);
  g.col_blocks = static_cast<uint32_t>(ceil_div(g.n, BN));
  dim3 grid;
  EJ_TRY(grouped_grid(static_cast<int64_t>(g.row_blocks) * g.col_blocks + kZeroBlocks,
                      WR * WC * 64, &grid));
  grid.y = g.splits;
  hipLaunchKernelGGL((grouped_rows_kernel<Op, BM, BN, WR, WC, BKC, DIRECT, NS>), grid,
                     dim3(WR * WC * 64), 0, stream, g);
  EJ_LAUNCH_CHECK();
  return g.splits > 1 ? join_parts(g, g.slots, g.slots, true, stream) : EJ_OK;
}

template <class Op, bool BKC>
int launch_large(GroupedArgs g, hipStream_t stream) {
  const int64_t groups = g.n_groups < g.slots ? g.n_groups : g.slots;
  g.row_blocks = static_cast<uint32_t>(g.slots / 256 + groups);
  g.col_blocks = static_cast<uint32_t>(ceil_div(g.n, 256));
  dim3 grid;
  EJ_TRY(grouped_grid(static_cast<int64_t>(g.row_blocks) * g.col_blocks + kLargeExtra + kZeroBlocks,
                      512, &grid));
  hipLaunchKernelGGL((grouped_large_kernel<Op, BKC>), grid, dim3(512), 0, stream, g);
  EJ_LAUNCH_CHECK();
  return EJ_OK;
}

template <class Op, int FM, int BN, int NW, bool BKC, int NS>
int launch_skinny(GroupedArgs g, hipStream_t stream) {
  const int64_t groups = g.n_groups < g.slots ? g.n_groups : g.slots;
  g.row_blocks = static_cast<uint32_t>(g.slots / (16 * FM) + groups);
  g.col_blocks = static_cast<uint32_t>(ceil_div(g.n, BN));
  dim3 grid;
  EJ_TRY(grouped_grid(static_cast<int64_t>(g.row_blocks) * g.col_blocks + kZeroBlocks, NW * 64,
                      &grid));
  hipLaunchKernelGGL((grouped_skinny_kernel<Op, FM, BN, NW, BKC, NS>), grid, dim3(NW * 64), 0,
                     stream, g);
  EJ_LAUNCH_CHECK();
  return EJ_OK;
}

template <class Op, int BM, int BN, int WR, int WC, bool DIRECT, int NS, int GATHER>
int launch_wgrad_as(GroupedArgs g, hipStream_t stream) {
  g.row_blocks = static_cast<uint32_t>(ceil_div(g.m, BM));
  g.col_blocks = static_cast<uint32_t>(ceil_div(g.n, BN));
  dim3 grid;
  EJ_TRY(grouped_grid(static_cast<int64_t>(g.row_blocks) * g.col_blocks * g.n_groups,
                      WR * WC * 64, &grid));
  grid.y = g.splits;
  hipLaunchKernelGGL((grouped_wgrad_kernel<Op, BM, BN, WR, WC, DIRECT, NS, GATHER>), grid,
                     dim3(WR * WC * 64), 0, stream, g);
  EJ_LAUNCH_CHECK();
  return g.splits > 1 ? join_parts(g, static_cast<int64_t>(g.n_groups) * g.m, g.m, false, stream)
                      : EJ_OK;
}

template <class Op, int BM, int BN, int WR, int WC, bool DIRECT, int NS>
int launch_wgrad(const GroupedArgs &g, hipStream_t stream) {
  if (g.a_rows) return launch_wgrad_as<Op, BM, BN, WR, WC, DIRECT, NS, 1>(g, stream);
  if (g.b_rows) return launch_wgrad_as<Op, BM, BN, WR, WC, DIRECT, NS, 2>(g, stream);
  return launch_wgrad_as<Op, BM, BN, WR, WC, DIRECT, NS, 0>(g, stream);
}

template <class Op, int GATHER>
int launch_wgrad_large_as(GroupedArgs g, hipStream_t stream) {
  g.row_blocks = static_cast<uint32_t>(ceil_div(g.m, 256));
  g.col_blocks = static_cast<uint32_t>(ceil_div(g.n, 256));
  dim3 grid;
  EJ_TRY(grouped_grid(static_cast<int64_t>(g.row_blocks) * g.col_blocks * g.n_groups + kLargeExtra,
                      512, &grid));
  hipLaunchKernelGGL((grouped_wgrad_large_kernel<Op, GATHER>), grid, dim3(512), 0, stream, g);
  EJ_LAUNCH_CHECK();
  return EJ_OK;
}

template <class Op>
int launch_wgrad_large(const GroupedArgs &g, hipStream_t stream) {
  if (g.a_rows) return launch_wgrad_large_as<Op, 1>(g, stream);
  if (g.b_rows) return launch_wgrad_large_as<Op, 2>(g, stream);
  return launch_wgrad_large_as<Op, 0>(g, stream);
}

// Tiles of a rows product: full row blocks and, on average, half of one for
// each group.
inline double expected_tiles(const GroupedArgs &g, int bm, int bn, int64_t groups) {
  return (static_cast<double>(g.slots) / bm + 0.5 * groups) * ceil_div(g.n, bn);
}

// Rounds of the large kernel for `tiles` blocks: the last one cut in four or
// two where that fills it.
inline double large_rounds(double tiles) {
  const double whole = std::floor(tiles / kLargeRound), last = tiles / kLargeRound - whole;
  return whole + (last <= 0 ? 0 : last <= 0.25 ? 0.4 : last <= 0.5 ? 0.6 : 1);
}

// The choice goes by the mean rows of a group (all that the host knows of the
// sizes) and the number of tiles.  Measured (us) with k = n = 2048, bf16, W
// [n][k] / [k][n], groups of unequal length; skinny 16 rows at k = n = 1024:
//   rows/group  groups   skinny 16  64 x 64   64 x 128  128 x 128  large
//        2         8      6.5/8.0   9.6       11.4      17.9
//       16         8     15.2/19.5  16.5      19.5      29
//       50         8                17/18     21/20     28/27      21/21
//       50        16                33/33     31/32     29/29      29/31
//      100         8                18/18     21/20     27/27      21/22
//      100        16                41/41     34/35     33/32      30/33
//      200        16                57/59     49/50     42/40      50/51
//      512        16                                    98/98      78/80
//       64 (k 1024)  64             63/63     59/58     67/69      61/62
template <class Op, bool BKC>
int pick_rows(const GroupedRows &r, hipStream_t stream) {
  const GroupedArgs &g = r.g;
  if (g.splits > 1) {
    if (!r.direct) return launch_rows<Op, 64, 64, 2, 2, BKC, false, 2>(g, stream);
    return launch_rows<Op, 64, 64, 2, 2, BKC, true, 3>(g, stream);
  }
  const int64_t groups = g.n_groups < g.slots ? (g.n_groups > 0 ? g.n_groups : 1) : g.slots;
  const double rows = static_cast<double>(g.slots) / groups;
  if (!r.direct) {
    if (rows > 128) return launch_rows<Op, 128, 128, 2, 4, BKC, false, 2>(g, stream);
    return launch_rows<Op, 64, 64, 2, 2, BKC, false, 2>(g, stream);
  }
  // columns of a skinny block: 32, or what fills 128 bytes of a [k][n] row
  constexpr int kSkinny = BKC || kElem<Op> == 4 ? 32 : 64;
  if (rows <= (BKC ? 16 : 8)) return launch_skinny<Op, 1, kSkinny, 4, BKC, 2>(g, stream);
  if constexpr (kElem<Op> == 4) {
    // bound by the fp32 matrix instructions at any tile: the finest spreads
    // best (4096 x 1024 x 2048 in 8 groups 164 us, 212 with 128 x 128; equal
    // within 2% at 16384 x 2048 x 2048)
    return launch_rows<Op, 64, 64, 2, 2, BKC, true, 0>(g, stream);
  } else {
    // up to about two small tiles to a CU the finest spread best
    if (rows <= 48 || expected_tiles(g, 64, 64, groups) <= 576)
      return launch_rows<Op, 64, 64, 2, 2, BKC, true, 3>(g, stream);
    if (rows <= 100) return launch_rows<Op, 64, 128, 2, 2, BKC, true, 3>(g, stream);
    // rounds of large blocks against a fifth less time for a round of 512
    // quarter-size ones (two to a CU, which even out)
    const double small = expected_tiles(g, 128, 128, groups) / 512;
    if (large_rounds(expected_tiles(g, 256, 256, groups)) <= 0.8 * (small > 1 ? small : 1))
      return launch_large<Op, BKC>(g, stream);
    return launch_rows<Op, 128, 128, 2, 2, BKC, true, 2>(g, stream);
  }
}

// 64 x 64 where larger tiles leave CUs idle, then 128 x 128 (two to a CU)
// against rounds of the large blocks.  Measured (us), bf16, rows as they lie /
// gathered, groups of unequal length:
//   rows   groups    m x n       64 x 64   128 x 128  large
//    4096     3   1024 x 1024    20/29      26/36     21/31
//    8192     5   1024 x 1024    37/44      32/46     34/48
//    8192    17   1024 x 1024    41/57      33/41     32/37
//    8192    17   1536 x 1536               62/78     60/67
//    8192     8   2048 x 2560              107/137    92/107
//   16384    16   2048 x 4096   547/729    378/474   300/336
// fp32: 4096 rows, 8 groups, 1024 x 2048: 128 x 128 157, 64 x 64 167; 1200
// rows, 5 groups, 320 x 520: 32 and 13.
template <class Op>
int pick_wgrad(const GroupedArgs &g, bool direct, hipStream_t stream) {
  if (!direct) return launch_wgrad<Op, 64, 64, 2, 2, false, 2>(g, stream);
  if (g.splits > 1) return launch_wgrad<Op, 64, 64, 2, 2, true, 3>(g, stream);
  auto tiles = [&](int b) {
    return static_cast<double>(ceil_div(g.m, b) * ceil_div(g.n, b) * g.n_groups);
  };
  if (tiles(128) < 256) return launch_wgrad<Op, 64, 64, 2, 2, true, 3>(g, stream);
  if constexpr (kElem<Op> == 2) {
    const double small = tiles(128) / 512;
    if (large_rounds(tiles(256)) <= 0.55 * (small > 1 ? small : 1))
      return launch_wgrad_large<Op>(g, stream);
  }
  return launch_wgrad<Op, 128, 128, 2, 2, true, 2>(g, stream);
}

}  // namespace ej
