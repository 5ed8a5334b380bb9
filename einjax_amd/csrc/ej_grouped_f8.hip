// Products grouped by expert on 8-bit floats with a scale for each block of 128.
#include "ej_grouped_pick.h"

namespace ej {

int grouped_rows_f8(const GroupedRows &r, hipStream_t stream) {
  return r.g.out == EJ_F32 ? pick_f8<OpF8Fine>(r, stream) : pick_f8<OpF8>(r, stream);
}

}  // namespace ej
