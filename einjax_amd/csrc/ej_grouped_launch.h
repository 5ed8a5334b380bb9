// Launches of the products grouped by expert, one translation unit for each
// operand type.
#pragma once

#include "ej_grouped.h"

namespace ej {

struct GroupedRows {
  GroupedArgs g;
  bool nk;      // k-contiguous weights
  bool direct;  // 16-byte aligned operands of whole chunks
};

int grouped_rows_bf16(const GroupedRows &r, hipStream_t stream);
int grouped_rows_f16(const GroupedRows &r, hipStream_t stream);
int grouped_rows_f32(const GroupedRows &r, hipStream_t stream);
int grouped_rows_i8(const GroupedRows &r, hipStream_t stream);
int grouped_rows_f8(const GroupedRows &r, hipStream_t stream);
int gated_rows_bf16(const GroupedRows &r, hipStream_t stream);
int gated_rows_f16(const GroupedRows &r, hipStream_t stream);
int gated_rows_f32(const GroupedRows &r, hipStream_t stream);
int grouped_wgrad_bf16(const GroupedArgs &g, bool direct, hipStream_t stream);
int grouped_wgrad_f16(const GroupedArgs &g, bool direct, hipStream_t stream);
int grouped_wgrad_f32(const GroupedArgs &g, bool direct, hipStream_t stream);

// Whether a rows product takes the kernel for few rows a group; tiles: 64 x 64
// ones (measured beside the choice of kernel).
inline bool few_rows(double rows, double tiles, int elem) {
  return rows <= (elem == 4 ? 24 : 16) || (rows <= 48 && tiles <= 192);
}

// A grid of `blocks` workgroups of `threads`, or EJ_E_UNSUPPORTED: launches
// hold fewer than 2^32 threads.
inline int grouped_grid(int64_t blocks, int threads, dim3 *grid) {
  if (blocks * threads >= (int64_t{1} << 32)) {
    set_error("%lld workgroups of %d threads: too many for one launch", (long long)blocks,
              threads);
    return EJ_E_UNSUPPORTED;
  }
  *grid = dim3(static_cast<unsigned>(blocks));
  return EJ_OK;
}

}  // namespace ej
