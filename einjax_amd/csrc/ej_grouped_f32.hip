// Products grouped by expert on f32 operands.
#include "ej_grouped_pick.h"

namespace ej {

int grouped_rows_f32(const GroupedRows &r, hipStream_t stream) {
  return r.nk ? pick_rows<OpF32, true>(r, stream) : pick_rows<OpF32, false>(r, stream);
}

int grouped_wgrad_f32(const GroupedArgs &g, bool direct, hipStream_t stream) {
  return pick_wgrad<OpF32>(g, direct, stream);
}

}  // namespace ej
