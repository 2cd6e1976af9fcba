// Paged decode on the vector units: float32 keys with bfloat16 values pages.
#include "paged_rows.h"

namespace tension {

bool launch_paged_rows_mixed(const PagedDecodeParams& p, int waves, hipStream_t st) {
  return launch_rows<TENSION_F32, TENSION_BF16, 8>(p, waves, st);
}

}  // namespace tension
