// Paged decode on the vector units: float32 pages.
#include "paged_rows.h"

namespace tension {

bool launch_paged_rows_f32(const PagedDecodeParams& p, int waves, hipStream_t st) {
  return launch_rows<TENSION_F32, TENSION_F32, 8>(p, waves, st);
}

}  // namespace tension
