// Paged decode on the vector units: e4m3 pages.
#include "paged_rows.h"

namespace tension {

// Sixteen codes to a lane; eight where sixteens would leave steps of 32 rows, or
// four query heads' sums 182 registers (two waves per SIMD).
bool launch_paged_rows_e4m3(const PagedDecodeParams& p, int waves, hipStream_t st) {
  if (p.D <= 32 || p.H / p.Hk > 2) return launch_rows<TENSION_E4M3, TENSION_E4M3, 8>(p, waves, st);
  return p.D % 16 == 0 && launch_rows<TENSION_E4M3, TENSION_E4M3, 16>(p, waves, st);
}

}  // namespace tension
