// Products grouped by expert on f16 operands.
#include "ej_grouped_pick.h"

namespace ej {

int grouped_rows_f16(const GroupedRows &r, hipStream_t stream) {
  return r.nk ? pick_rows<OpF16, true>(r, stream) : pick_rows<OpF16, false>(r, stream);
}

int grouped_wgrad_f16(const GroupedArgs &g, bool direct, hipStream_t stream) {
  return pick_wgrad<OpF16>(g, direct, stream);
}

}  // namespace ej
