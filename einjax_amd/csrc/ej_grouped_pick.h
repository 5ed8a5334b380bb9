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

template <class Op, int BN, int NW, bool BKC, int NS>
int launch_skinny(GroupedArgs g, hipStream_t stream) {
  const int64_t groups = g.n_groups < g.slots ? g.n_groups : g.slots;
  g.row_blocks = static_cast<uint32_t>(g.slots / 16 + groups);
  g.col_blocks = static_cast<uint32_t>(ceil_div(g.n, BN));
  dim3 grid;
  EJ_TRY(grouped_grid(static_cast<int64_t>(g.row_blocks) * g.col_blocks + kZeroBlocks, NW * 64,
                      &grid));
  hipLaunchKernelGGL((grouped_skinny_kernel<Op, BN, NW, BKC, NS>), grid, dim3(NW * 64), 0,
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
// sizes) and the number of tiles.  Measured (us), bf16, W [n][k] / [k][n]:
//   rows/group  groups     k x n      skinny  64 x 64  64 x 128  128 x 128  large
//      4..16       8   1024 x 1024     7/7     9/10     11/11      15/15    10/11
//        48        8   1024 x 1024     9/9     9/10
//      4..16       1   4096 x 8192    13/16   25/26
//        48        1   4096 x 8192    17/20   25/29
//         4       16   2048 x 4096    40/41   44/43
//        16       16   2048 x 4096    42/45   45/44
//        32       16   2048 x 4096    61/55   51/50
//        50        8   2048 x 2048            16/17    20/19      26/25    20/21
//        50       16   2048 x 2048            32/32    30/31      28/27    28/30
//       100        8   2048 x 2048            20/18    20/20      26/26    20/21
//       100       16   2048 x 2048            40/41    33/36      31/30    29/31
//       200       16   2048 x 2048            56/55    47/51      41/39    48/49
//       512       16   2048 x 2048           115/119  111/112     90/92    74/75
//        64       64   1024 x 2048            64/63    58/58      65/66    58/59
// fp32, 16 groups, 2048 x 4096: 24 rows 134/142 skinny, 159/160 in 64 x 64; 32
// rows 156/155 and 156/158.
template <class Op, bool BKC>
int pick_rows(const GroupedRows &r, hipStream_t stream) {
  const GroupedArgs &g = r.g;
  if (g.splits > 1) {
    if (!r.direct) return launch_rows<Op, 64, 64, 2, 2, BKC, false, 2>(g, stream);
    return launch_rows<Op, 64, 64, 2, 2, BKC, true, kElem<Op> == 4 ? 0 : 3>(g, stream);
  }
  const int64_t groups = g.n_groups < g.slots ? (g.n_groups > 0 ? g.n_groups : 1) : g.slots;
  const double rows = static_cast<double>(g.slots) / groups;
  const double tiles = expected_tiles(g, 64, 64, groups);
  if (!r.direct) {
    // (us) 64 x 64, 64 x 128 and 128 x 128; in 12 groups 3022 x 771 x 1283
    // f16 38, 31, 33, fp32 120, 103, 130; in 4 groups 6000 x 1001 x 1001 fp32
    // 157, 126, 157; in 6 3000 x 517 x 2051 f16 31, 32, 25; few tiles: in 8
    // groups 800 x 771 x 1283 f16 19, 18, 22; in 4 2000 x 255 x 333 fp32 13, 16,
    // 24, 8 bits 7 and 9 in 128 x 128
    if (tiles <= 512 || rows <= 128)
      return launch_rows<Op, 64, 64, 2, 2, BKC, false, 2>(g, stream);
    if constexpr (kElem<Op> == 4)
      return launch_rows<Op, 64, 128, 2, 4, BKC, false, 2>(g, stream);
    else
      return launch_rows<Op, 128, 128, 2, 4, BKC, false, 2>(g, stream);
  }
  // columns of a skinny block: 32, or what fills 128 bytes of a [k][n] row
  constexpr int kSkinny = BKC || kElem<Op> == 4 ? 32 : 64;
  if (few_rows(rows, tiles, kElem<Op>))
    return launch_skinny<Op, kSkinny, 4, BKC, 2>(g, stream);
  if constexpr (kElem<Op> == 4) {
    // bound by the fp32 matrix instructions at any tile: the finest spreads
    // best (4096 x 1024 x 2048 in 8 groups 164 us, 212 with 128 x 128; equal
    // within 2% at 16384 x 2048 x 2048)
    return launch_rows<Op, 64, 64, 2, 2, BKC, true, 0>(g, stream);
  } else {
    // up to about two small tiles to a CU the finest spread best
    if (rows <= 48 || tiles <= 576)
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
//    4096     3   1024 x 1024    21/29      26/36     21/31
//    8192     5   1024 x 1024    37/46      33/46     34/47
//    8192    17   1024 x 1024    40/58      35/38     28/34
//    8192    17   1536 x 1536    82/123     61/74     54/62
//    8192     8   2048 x 2560   153/219    101/129    86/102
//   16384    16   2048 x 4096   522/721    350/442   273/308
// fp32: 4096 rows, 8 groups, 1024 x 2048: 128 x 128 153, 64 x 64 173; 1200
// rows, 5 groups, 320 x 520: 32 and 13.  Through registers, f16, 64 x 64 and 128
// x 128: 16384 rows, 8 groups, 1023 x 2047 267/294 and 182/200; 4096, 4, 771 x
// 1283 52/56 and 43/49; 5820, 7, 512 x 1477 43/51 and 43/47, in very
// unequal groups 16 more (few tiles of the longest one); fp32 4096, 4, 771 x
// 1283 153 and 200.
template <class Op>
int pick_wgrad(const GroupedArgs &g, bool direct, hipStream_t stream) {
  auto tiles = [&](int b) {
    return static_cast<double>(ceil_div(g.m, b) * ceil_div(g.n, b) * g.n_groups);
  };
  if (!direct) {
    if constexpr (kElem<Op> == 2) {
      if (g.splits == 1 && tiles(128) >= 512)
        return launch_wgrad<Op, 128, 128, 2, 4, false, 2>(g, stream);
    }
    return launch_wgrad<Op, 64, 64, 2, 2, false, 2>(g, stream);
  }
  if (g.splits > 1) return launch_wgrad<Op, 64, 64, 2, 2, true, 3>(g, stream);
  if (tiles(128) < 256) return launch_wgrad<Op, 64, 64, 2, 2, true, 3>(g, stream);
  if constexpr (kElem<Op> == 2) {
    const double small = tiles(128) / 512;
    if (large_rounds(tiles(256)) <= 0.55 * (small > 1 ? small : 1))
      return launch_wgrad_large<Op>(g, stream);
  }
  return launch_wgrad<Op, 128, 128, 2, 2, true, 2>(g, stream);
}

}  // namespace ej
