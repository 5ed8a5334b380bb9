// Gated products grouped by expert on fp32 operands.
#include "ej_grouped_pick.h"

namespace ej {

int gated_rows_f32(const GroupedRows &r, hipStream_t stream) {
  return r.nk ? pick_gated<OpF32, true>(r, stream) : pick_gated<OpF32, false>(r, stream);
}

}  // namespace ej
