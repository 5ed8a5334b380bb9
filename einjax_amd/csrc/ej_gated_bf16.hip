// Gated products grouped by expert on bf16 operands.
#include "ej_grouped_pick.h"

namespace ej {

int gated_rows_bf16(const GroupedRows &r, hipStream_t stream) {
  return r.nk ? pick_gated<OpBf16, true>(r, stream) : pick_gated<OpBf16, false>(r, stream);
}

}  // namespace ej
