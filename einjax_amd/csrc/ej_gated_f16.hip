// Gated products grouped by expert on f16 operands.
#include "ej_grouped_pick.h"

namespace ej {

int gated_rows_f16(const GroupedRows &r, hipStream_t stream) {
  return r.nk ? pick_gated<OpF16, true>(r, stream) : pick_gated<OpF16, false>(r, stream);
}

}  // namespace ej
