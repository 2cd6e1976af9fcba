// Paged decode on the vector units: e4m3 pages.
#include "paged_rows.h"

namespace tension {

// Sixteen codes to a lane; eight where rows are not whole pieces of sixteen,
// where sixteens would leave steps of 32 rows, or four query heads' sums 182
// registers (two waves per SIMD).
bool launch_paged_rows_e4m3(const PagedDecodeParams& p, int waves, hipStream_t st) {
  if (p.D > 32 && p.D % 16 == 0 && p.H / p.Hk <= 2 && row_pieces(p.c.k, 16) && row_pieces(p.c.v, 16))
    return launch_rows<TENSION_E4M3, TENSION_E4M3, 16>(p, waves, st);
  return launch_rows<TENSION_E4M3, TENSION_E4M3, 8>(p, waves, st);
}

}  // namespace tension
