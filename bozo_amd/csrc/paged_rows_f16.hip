// Paged decode on the vector units: float16 pages.
#include "paged_rows.h"

namespace tension {

bool launch_paged_rows_f16(const PagedDecodeParams& p, int waves, hipStream_t st) {
  return launch_rows<TENSION_F16, TENSION_F16, 8>(p, waves, st);
}

}  // namespace tension
