// Which paged decode calls run on whole pieces of rows, and on how many waves.
#include "paged.h"

namespace tension {

bool launch_paged_rows_bf16(const PagedDecodeParams&, int waves, hipStream_t);
bool launch_paged_rows_f16(const PagedDecodeParams&, int waves, hipStream_t);
bool launch_paged_rows_f32(const PagedDecodeParams&, int waves, hipStream_t);
bool launch_paged_rows_mixed(const PagedDecodeParams&, int waves, hipStream_t);
bool launch_paged_rows_e4m3(const PagedDecodeParams&, int waves, hipStream_t);

namespace {

// Pieces of 8 values are whole pieces of memory.
bool rows_aligned(const Buf& b) { return row_pieces(b, b.dt == TENSION_E4M3 ? 8 : 16); }

// Waves of a workgroup.  Up to one workgroup per CU the call waits for memory
// (N16 H12, 1000 bf16 keys: eight waves 11.1 us, four 12.3), and where each
// takes long the last to end count (N128 H16, up to 4096 ragged bf16 keys, the
// longest first: 205.5 against 206.7).  Windows of two batches of a pair of
// waves leave the others nothing (N128 H16 W64 e4m3: two waves 8.5 us, four 10.7).
int waves_for(const PagedDecodeParams& p) {
  const int64_t groups = (int64_t)p.N * p.Hk * p.splits, cus = device_cus();
  const int64_t keys = p.splits > 1 ? p.chunk : p.most;
  if (groups <= cus) return keys > 64 ? 8 : 4;
  if (keys <= 128) return groups >= 3 * cus ? 2 : 4;
  return keys >= 2048 ? 8 : 4;
}

}  // namespace

bool launch_paged_decode_rows(const PagedDecodeParams& p, hipStream_t st) {
  if (p.D % 8 || !rows_aligned(p.c.k) || !rows_aligned(p.c.v)) return false;
  if (!DecodeGrid::fits(p)) return false;
  // A shared key head on the matrix units where its types allow (us, against the vector units, of back-to-back calls):
  // bf16 D64, 268 MB: two query heads 47 / 47, four 47 / 49, eight 47 / 96; e4m3 D128, 135 MB: 30.5 / 33.7, 30.6 / 58,
  // 31 / 87.
  if (p.H / p.Hk >= 2 && launch_paged_decode_mfma(p, st)) return true;
  const int waves = waves_for(p);
  if (p.c.k.dt == TENSION_F32 && p.c.v.dt == TENSION_BF16) return launch_paged_rows_mixed(p, waves, st);
  if (p.c.k.dt != p.c.v.dt) return false;
  switch (p.c.k.dt) {
    case TENSION_BF16: return launch_paged_rows_bf16(p, waves, st);
    case TENSION_F16: return launch_paged_rows_f16(p, waves, st);
    case TENSION_F32: return launch_paged_rows_f32(p, waves, st);
    default: return launch_paged_rows_e4m3(p, waves, st);
  }
}

}  // namespace tension
