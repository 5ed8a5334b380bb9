// Products grouped by expert on bf16 operands.
#include "ej_grouped_pick.h"

namespace ej {

int grouped_rows_bf16(const GroupedRows &r, hipStream_t stream) {
  return r.nk ? pick_rows<OpBf16, true>(r, stream) : pick_rows<OpBf16, false>(r, stream);
}

int grouped_wgrad_bf16(const GroupedArgs &g, bool direct, hipStream_t stream) {
  return pick_wgrad<OpBf16>(g, direct, stream);
}

}  // namespace ej
