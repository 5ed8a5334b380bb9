// Products grouped by expert on 8-bit operands with scales.
#include "ej_grouped_pick.h"

namespace ej {

int grouped_rows_i8(const GroupedRows &r, hipStream_t stream) {
  return pick_rows<OpI8, true>(r, stream);
}

}  // namespace ej
