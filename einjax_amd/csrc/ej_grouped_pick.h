// Choice of tile for one operand type.
#pragma once

#include "ej_grouped_launch.h"
#include "ej_grouped_tile.h"

namespace ej {

template <class Op, int BM, int BN, int WR, int WC, bool BKC, bool DIRECT, int NS>
int launch_rows(GroupedArgs g, hipStream_t stream) {
  const int64_t groups = g.n_groups < g.slots ? g.n_groups : g.slots;
  g.row_blocks = static_cast<uint32_t>(g.slots / BM + groups);
  g.col_blocks = static_cast<uint32_t>(ceil_div(g.n, BN));
  dim3 grid;
  EJ_TRY(grouped_grid(static_cast<int64_t>(g.row_blocks) * g.col_blocks + kZeroBlocks,
                      WR * WC * 64, &grid));
  hipLaunchKernelGGL((grouped_rows_kernel<Op, BM, BN, WR, WC, BKC, DIRECT, NS>), grid,
                     dim3(WR * WC * 64), 0, stream, g);
  EJ_LAUNCH_CHECK();
  return EJ_OK;
}

template <class Op, int BM, int BN, int WR, int WC, bool DIRECT, int NS>
int launch_wgrad(GroupedArgs g, hipStream_t stream) {
  g.row_blocks = static_cast<uint32_t>(ceil_div(g.m, BM));
  g.col_blocks = static_cast<uint32_t>(ceil_div(g.n, BN));
  dim3 grid;
  EJ_TRY(grouped_grid(static_cast<int64_t>(g.row_blocks) * g.col_blocks * g.n_groups,
                      WR * WC * 64, &grid));
  hipLaunchKernelGGL((grouped_wgrad_kernel<Op, BM, BN, WR, WC, DIRECT, NS>), grid,
                     dim3(WR * WC * 64), 0, stream, g);
  EJ_LAUNCH_CHECK();
  return EJ_OK;
}

template <class Op, bool BKC>
int pick_rows(const GroupedRows &r, hipStream_t stream) {
  if (!r.direct) return launch_rows<Op, 128, 128, 2, 2, BKC, false, 2>(r.g, stream);
  return launch_rows<Op, 128, 128, 2, 2, BKC, true, 2>(r.g, stream);
}

template <class Op>
int pick_wgrad(const GroupedArgs &g, bool direct, hipStream_t stream) {
  if (!direct) return launch_wgrad<Op, 128, 128, 2, 2, false, 2>(g, stream);
  return launch_wgrad<Op, 128, 128, 2, 2, true, 2>(g, stream);
}

}  // namespace ej
