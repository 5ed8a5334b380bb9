// Choice of tile for one operand type.
#pragma once

#include <cmath>

#include "ej_grouped_launch.h"
#include "ej_grouped_tile.h"

namespace ej {

// Whether rows of the operands are shorter than 16 bytes.
template <class Op, bool BKC>
bool short_rows(const GroupedArgs &g) {
  return g.k < kChunk<Op> || (!BKC && g.n < kChunk<Op>);
}

inline int join_parts(const GroupedArgs &g, int64_t rows, int64_t m, bool skip_dead,
                      hipStream_t stream) {
  dim3 grid;
  EJ_TRY(grouped_grid(ceil_div(rows * ceil_div(g.n, 4), 256), 256, &grid));
  hipLaunchKernelGGL(grouped_join_kernel, grid, dim3(256), 0, stream, g, rows, m, skip_dead);
  EJ_LAUNCH_CHECK();
  return EJ_OK;
}

template <bool FINE>
int join_gated(const GroupedArgs &g, hipStream_t stream) {
  dim3 grid;
  EJ_TRY(grouped_grid(ceil_div(g.slots * ceil_div(g.n, 4), 256), 256, &grid));
  hipLaunchKernelGGL(gated_join_kernel<FINE>, grid, dim3(256), 0, stream, g);
  EJ_LAUNCH_CHECK();
  return EJ_OK;
}

// Columns of the results that a tile of `bn` columns of B gives.
template <bool GATED>
constexpr int result_cols(int bn) {
  return GATED ? bn / 2 : bn;
}

template <class Op, int BM, int BN, int WR, int WC, bool BKC, int LOADS, int NS,
          bool GATED = false>
int launch_rows(GroupedArgs g, hipStream_t stream) {
  const int64_t groups = g.n_groups < g.slots ? g.n_groups : g.slots;
  g.row_blocks = static_cast<uint32_t>(g.slots / BM + groups);
  g.col_blocks = static_cast<uint32_t>(ceil_div(g.n, result_cols<GATED>(BN)));
  dim3 grid;
  EJ_TRY(grouped_grid(static_cast<int64_t>(g.row_blocks) * g.col_blocks + kZeroBlocks,
                      WR * WC * 64, &grid));
  grid.y = g.splits;
  hipLaunchKernelGGL((grouped_rows_kernel<Op, BM, BN, WR, WC, BKC, LOADS, NS, GATED>), grid,
                     dim3(WR * WC * 64), 0, stream, g);
  EJ_LAUNCH_CHECK();
  if (g.splits == 1) return EJ_OK;
  if constexpr (GATED) return join_gated<kElem<Op> == 4>(g, stream);
  else return join_parts(g, g.slots, g.slots, true, stream);
}

template <class Op, bool BKC, bool GATED = false>
int launch_large(GroupedArgs g, hipStream_t stream) {
  const int64_t groups = g.n_groups < g.slots ? g.n_groups : g.slots;
  g.row_blocks = static_cast<uint32_t>(g.slots / 256 + groups);
  g.col_blocks = static_cast<uint32_t>(ceil_div(g.n, result_cols<GATED>(256)));
  dim3 grid;
  EJ_TRY(grouped_grid(static_cast<int64_t>(g.row_blocks) * g.col_blocks + kLargeExtra + kZeroBlocks,
                      512, &grid));
  hipLaunchKernelGGL((grouped_large_kernel<Op, BKC, GATED>), grid, dim3(512), 0, stream, g);
  EJ_LAUNCH_CHECK();
  return EJ_OK;
}

template <class Op, int BN, int NW, bool BKC, int NS, bool GATED = false>
int launch_skinny(GroupedArgs g, hipStream_t stream) {
  const int64_t groups = g.n_groups < g.slots ? g.n_groups : g.slots;
  g.row_blocks = static_cast<uint32_t>(g.slots / 16 + groups);
  g.col_blocks = static_cast<uint32_t>(ceil_div(g.n, result_cols<GATED>(BN)));
  dim3 grid;
  EJ_TRY(grouped_grid(static_cast<int64_t>(g.row_blocks) * g.col_blocks + kZeroBlocks, NW * 64,
                      &grid));
  hipLaunchKernelGGL((grouped_skinny_kernel<Op, BN, NW, BKC, NS, GATED>), grid, dim3(NW * 64), 0,
                     stream, g);
  EJ_LAUNCH_CHECK();
  return EJ_OK;
}

template <class Op, int BM, int BN, int WR, int WC, int LOADS, int NS, int GATHER>
int launch_wgrad_as(GroupedArgs g, hipStream_t stream) {
  g.row_blocks = static_cast<uint32_t>(ceil_div(g.m, BM));
  g.col_blocks = static_cast<uint32_t>(ceil_div(g.n, BN));
  dim3 grid;
  EJ_TRY(grouped_grid(static_cast<int64_t>(g.row_blocks) * g.col_blocks * g.n_groups,
                      WR * WC * 64, &grid));
  grid.y = g.splits;
  hipLaunchKernelGGL((grouped_wgrad_kernel<Op, BM, BN, WR, WC, LOADS, NS, GATHER>), grid,
                     dim3(WR * WC * 64), 0, stream, g);
  EJ_LAUNCH_CHECK();
  return g.splits > 1 ? join_parts(g, static_cast<int64_t>(g.n_groups) * g.m, g.m, false, stream)
                      : EJ_OK;
}

template <class Op, int BM, int BN, int WR, int WC, int LOADS, int NS>
int launch_wgrad(const GroupedArgs &g, hipStream_t stream) {
  if (g.a_rows) return launch_wgrad_as<Op, BM, BN, WR, WC, LOADS, NS, 1>(g, stream);
  if (g.b_rows) return launch_wgrad_as<Op, BM, BN, WR, WC, LOADS, NS, 2>(g, stream);
  return launch_wgrad_as<Op, BM, BN, WR, WC, LOADS, NS, 0>(g, stream);
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
  if (!r.direct && short_rows<Op, BKC>(g))
    return launch_rows<Op, 64, 64, 2, 2, BKC, kLoadElements, 2>(g, stream);
  if (g.splits > 1) {
    if (!r.direct) return launch_rows<Op, 64, 64, 2, 2, BKC, kLoadPieces, 2>(g, stream);
    return launch_rows<Op, 64, 64, 2, 2, BKC, kLoadDirect, kElem<Op> == 4 ? 0 : 3>(g, stream);
  }
  const int64_t groups = g.n_groups < g.slots ? (g.n_groups > 0 ? g.n_groups : 1) : g.slots;
  const double rows = static_cast<double>(g.slots) / groups;
  const double tiles = expected_tiles(g, 64, 64, groups);
  if (!r.direct) {
    // (us) 64 x 64, 64 x 128 and 128 x 128; in 12 groups 3022 x 771 x 1283
    // f16 34, 30, 29, fp32 85, 88, 113; in 4 groups 6000 x 1001 x 1001 f16 45,
    // 33, 34, fp32 135, 112, 145; in 6 3000 x 517 x 2051 f16 29, 28, 23; few
    // tiles: in 8 groups 800 x 771 x 1283 f16 14, 15, 19; in 4 2000 x 255 x 333
    // fp32 11, 14, 22, 8 bits 7 and 9 in 128 x 128
    if (tiles <= 512 || rows <= 128)
      return launch_rows<Op, 64, 64, 2, 2, BKC, kLoadPieces, 2>(g, stream);
    if constexpr (kElem<Op> == 4)
      return launch_rows<Op, 64, 128, 2, 4, BKC, kLoadPieces, 2>(g, stream);
    else
      return launch_rows<Op, 128, 128, 2, 4, BKC, kLoadPieces, 2>(g, stream);
  }
  // columns of a skinny block: 32, or what fills 128 bytes of a [k][n] row
  constexpr int kSkinny = BKC || kElem<Op> == 4 ? 32 : 64;
  if (few_rows(rows, tiles, kElem<Op>))
    return launch_skinny<Op, kSkinny, 4, BKC, 2>(g, stream);
  if constexpr (kElem<Op> == 4) {
    // bound by the fp32 matrix instructions at any tile: the finest spreads
    // best (4096 x 1024 x 2048 in 8 groups 164 us, 212 with 128 x 128; equal
    // within 2% at 16384 x 2048 x 2048)
    return launch_rows<Op, 64, 64, 2, 2, BKC, kLoadDirect, 0>(g, stream);
  } else {
    // up to about two small tiles to a CU the finest spread best
    if (rows <= 48 || tiles <= 576)
      return launch_rows<Op, 64, 64, 2, 2, BKC, kLoadDirect, 3>(g, stream);
    if (rows <= 100) return launch_rows<Op, 64, 128, 2, 2, BKC, kLoadDirect, 3>(g, stream);
    // rounds of large blocks against a fifth less time for a round of 512
    // quarter-size ones (two to a CU, which even out)
    const double small = expected_tiles(g, 128, 128, groups) / 512;
    if (large_rounds(expected_tiles(g, 256, 256, groups)) <= 0.8 * (small > 1 ? small : 1))
      return launch_large<Op, BKC>(g, stream);
    return launch_rows<Op, 128, 128, 2, 2, BKC, kLoadDirect, 2>(g, stream);
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
// x 128: 16384 rows, 8 groups, 1023 x 2047 209/205 and 122/125; 4096, 4, 771 x
// 1283 36/39 and 30/34; 5820, 7, 512 x 1477 29/31 and 25/27; fp32 4096, 4, 771 x
// 1283 108 and 138.
template <class Op>
int pick_wgrad(const GroupedArgs &g, bool direct, hipStream_t stream) {
  auto tiles = [&](int b) {
    return static_cast<double>(ceil_div(g.m, b) * ceil_div(g.n, b) * g.n_groups);
  };
  if (!direct) {
    if (g.m < kChunk<Op> || g.n < kChunk<Op>)
      return launch_wgrad<Op, 64, 64, 2, 2, kLoadElements, 2>(g, stream);
    if constexpr (kElem<Op> == 2) {
      if (g.splits == 1 && tiles(128) >= 256)
        return launch_wgrad<Op, 128, 128, 2, 4, kLoadPieces, 2>(g, stream);
    }
    return launch_wgrad<Op, 64, 64, 2, 2, kLoadPieces, 2>(g, stream);
  }
  if (g.splits > 1) return launch_wgrad<Op, 64, 64, 2, 2, kLoadDirect, 3>(g, stream);
  if (tiles(128) < 256) return launch_wgrad<Op, 64, 64, 2, 2, kLoadDirect, 3>(g, stream);
  if constexpr (kElem<Op> == 2) {
    const double small = tiles(128) / 512;
    if (large_rounds(tiles(256)) <= 0.55 * (small > 1 ? small : 1))
      return launch_wgrad_large<Op>(g, stream);
  }
  return launch_wgrad<Op, 128, 128, 2, 2, kLoadDirect, 2>(g, stream);
}

// Gated rows, by the columns of both projections.  Measured (us), bf16, W [n][k] /
// [k][n], n both projections', weights from memory in the first five lines:
//   rows/group  groups     k x n      skinny  64 x 64  64 x 128  128 x 128  large
//        16        1   4096 x 8192    15/34   29/36     34/38      61/60    50/56
//         8        8   1024 x 1024     6/11   10/11     12/12      18/19    15/17
//         2       16   2048 x 4096    44/49   60/57     56/48      59/46    60/51
//        16       16   2048 x 4096    55/70   63/61     63/53      67/55    69/54
//        32       16   2048 x 4096    79/100  65/64     63/54      67/56    69/54
//        50        8   2048 x 2048    21/27   15/16     19/19      25/25    20/23
//        50       16   2048 x 2048    40/50   27/28     26/28      27/27    28/30
//       100       16   2048 x 2048    67/80   37/38     33/31      27/28    28/30
//       200       16   2048 x 2048   126/142  55/77     46/48      36/34    33/33
//       512       16   2048 x 2048           115/147  102/101     86/86    75/77
//      8192        1   4096 x 8192           869/1137 720/748    522/530  391/388
// [k][n] in 64 columns takes half a line of each projection, so with many tiles 128
// are better from the first row on.  fp32 (128 x 128 as the pipelined loop):
//        16       16   2048 x 4096   105/135  156/160
//        24       16   2048 x 4096   130/176  156/161
//        32       16   2048 x 4096   134/181  159/160
//        64       16   1024 x 2048             46/45     42/42      70/73
//       100        8   1024 x 2048             40/42     38/40      67/72
//       512        8   1024 x 4096            278/278   262/270   255/262
//      8192        1   2048 x 4096           1065/1065 1011/1028  979/1006
// The choice, skinny up to 24 rows and 64 x 64 above, is within 9% of the best but at
// 32 rows of [n][k]: the matrix instructions bound all tiles (8192 rows: 129
// TFLOP/s in 64 x 64, 140 in 128 x 128).
template <class Op, bool BKC>
int pick_gated(const GroupedRows &r, hipStream_t stream) {
  const GroupedArgs &g = r.g;
  if (!r.direct && short_rows<Op, BKC>(g))
    return launch_rows<Op, 64, 64, 2, 2, BKC, kLoadElements, 2, true>(g, stream);
  if (g.splits > 1) {
    if (!r.direct) return launch_rows<Op, 64, 64, 2, 2, BKC, kLoadPieces, 2, true>(g, stream);
    return launch_rows<Op, 64, 64, 2, 2, BKC, kLoadDirect, kElem<Op> == 4 ? 0 : 3, true>(g, stream);
  }
  const int64_t groups = g.n_groups < g.slots ? (g.n_groups > 0 ? g.n_groups : 1) : g.slots;
  const double rows = static_cast<double>(g.slots) / groups;
  auto tiles_of = [&](int bm, int bn) {
    return (static_cast<double>(g.slots) / bm + 0.5 * groups) * ceil_div(g.n, bn / 2);
  };
  const double tiles = tiles_of(64, 64);
  if (!r.direct) {
    if constexpr (kElem<Op> == 4) {
      if (tiles <= 512 || rows <= 128)
        return launch_rows<Op, 64, 64, 2, 2, BKC, kLoadPieces, 2, true>(g, stream);
      return launch_rows<Op, 64, 128, 2, 4, BKC, kLoadPieces, 2, true>(g, stream);
    } else {
      // The columns of a wave lie in two runs, which its loads of [k][n] take one by
      // one: longer runs, fewer lines.  (us) 64 x 64 in 2 x 2 and 4 x 1 waves, 64 x
      // 128 in 4 x 2, 128 x 128 in 2 x 4 and 4 x 2, f16: 3022 picks in 12 groups, 771
      // x 2566 71, 56, 44, 53, 44, [n][k] 48, 48, 42, 42, 42; 12000 in 4, 1023 x 2042
      // 212, 155, 121, 117, 92; 600 in 12 26, 23, 20, 35, 25; 200 in 12, [n][k]
      // 16, 15, 16, 19, 19
      if (tiles <= 512)
        return launch_rows<Op, 64, 64, 4, 1, BKC, kLoadPieces, 2, true>(g, stream);
      if (rows <= 128)
        return launch_rows<Op, 64, 128, 4, 2, BKC, kLoadPieces, 2, true>(g, stream);
      return launch_rows<Op, 128, 128, 4, 2, BKC, kLoadPieces, 2, true>(g, stream);
    }
  }
  constexpr int kSkinny = BKC || kElem<Op> == 4 ? 32 : 64;
  const bool wide = !BKC && kElem<Op> == 2 && rows <= 48 && tiles > 512;
  if (!wide && few_rows(rows, tiles, kElem<Op>))
    return launch_skinny<Op, kSkinny, 4, BKC, 2, true>(g, stream);
  if constexpr (kElem<Op> == 4) {
    return launch_rows<Op, 64, 64, 2, 2, BKC, kLoadDirect, 0, true>(g, stream);
  } else {
    if (!wide && (rows <= 48 || tiles <= 576))
      return launch_rows<Op, 64, 64, 2, 2, BKC, kLoadDirect, 3, true>(g, stream);
    if (rows <= 64) return launch_rows<Op, 64, 128, 2, 2, BKC, kLoadDirect, 3, true>(g, stream);
    const double small = tiles_of(128, 128) / 512;
    if (large_rounds(tiles_of(256, 256)) <= 0.8 * (small > 1 ? small : 1))
      return launch_large<Op, BKC, true>(g, stream);
    return launch_rows<Op, 128, 128, 2, 2, BKC, kLoadDirect, 2, true>(g, stream);
  }
}

// Products of 8-bit floats with block scales.  Measured (us), 16-bit results:
//   rows/group  groups     k x n      skinny  64 x 64  64 x 128  128 x 128  large
//       48        1   4096 x 8192      11       19        26        26       23
//      128        1   4096 x 4096      14       18        26        25       21
//      256        1   4096 x 4096      25       19        26        26       21
//       50       16   2048 x 2048      28       15        16        16       20
//      100        8   2048 x 2048      28       13        17        16       16
//      100       16   2048 x 2048      48       21        19        18       21
//      200       16   2048 x 2048      88       35        34        26       23
//      512       16   2048 x 2048     208       65        68        46       37
//     1024        4   1024 x 1024      38       12        12        11       10
// 128 x 128 in four waves 23 to 54 where eight take 16 to 46.  Results in fp32 (no
// large blocks): 17 in 64 x 64 for 50 rows in 16 groups, 23 in 128 x 128; 28 and 25
// for 100; 97 and 77 for 512.  Through registers 64 x 64 in four waves and in
// eight, 128 x 128: 6 groups of 259, 1000 x 1283 14, 14, 14; 8 of 500, 1000 x 2000
// 29, 31, 27; 1 of 16, 4090 x 4096 24, 22, 36; 4 of 150, 4001 x 1000 32, 31, 48.
template <class Op>
int pick_f8(const GroupedRows &r, hipStream_t stream) {
  const GroupedArgs &g = r.g;
  const int64_t groups = g.n_groups < g.slots ? (g.n_groups > 0 ? g.n_groups : 1) : g.slots;
  const double rows = static_cast<double>(g.slots) / groups;
  const double tiles = expected_tiles(g, 64, 64, groups);
  if (!r.direct) {
    if (short_rows<Op, true>(g))
      return launch_rows<Op, 64, 64, 2, 2, true, kLoadElements, 2>(g, stream);
    if (tiles <= 256) return launch_rows<Op, 64, 64, 4, 2, true, kLoadPieces, 2>(g, stream);
    if (tiles <= 704) return launch_rows<Op, 64, 64, 2, 2, true, kLoadPieces, 2>(g, stream);
    return launch_rows<Op, 128, 128, 2, 4, true, kLoadPieces, 2>(g, stream);
  }
  if (rows <= 16 || (rows <= 128 && tiles <= 192))
    return launch_skinny<Op, 32, 4, true, 2>(g, stream);
  if (tiles <= 704) return launch_rows<Op, 64, 64, 2, 2, true, kLoadDirect, 2>(g, stream);
  if constexpr (__is_same(Op, OpF8)) {
    // the large blocks' offsets of rows, in 32 bits
    const bool near = g.ldb < (1 << 24) && g.lda < (1 << 24) &&
                      (!g.a_rows || g.n_a <= (int64_t{1} << 32) / (g.lda > 128 ? g.lda : 128));
    const double small = expected_tiles(g, 128, 128, groups) / 512;
    if (near && rows > 128 &&
        large_rounds(expected_tiles(g, 256, 256, groups)) <= (small > 1 ? small : 1))
      return launch_large<Op, true>(g, stream);
  }
  return launch_rows<Op, 128, 128, 2, 4, true, kLoadDirect, 2>(g, stream);
}

}  // namespace ej
