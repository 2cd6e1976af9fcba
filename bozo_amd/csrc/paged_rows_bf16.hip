// Paged decode on the vector units: bfloat16 pages.
#include "paged_rows.h"

namespace tension {

bool launch_paged_rows_bf16(const PagedDecodeParams& p, int waves, hipStream_t st) {
  return launch_rows<TENSION_BF16, TENSION_BF16, 8>(p, waves, st);
}

}  // namespace tension
