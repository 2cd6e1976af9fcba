// Paged K/V cache: tokens written into pages (quantised to e4m3 on the way or
// as they are) and read back dense.  Both are streams: a row of D values is
// read once and written once, so HBM bounds them.
//
// Quantised rows: with E the biased exponent of a row's largest finite
// magnitude a and M its mantissa bits, 448 = 1.75 * 2^8 gives the smallest e
// with a <= 448 * 2^e as e + 127 = E - 8 + (M > 0x600000), at least 1.  A power
// of two scales exactly, so the one rounding of a value is that of its code
// (e4m3, half a step: 2^-4 relative), and a float scale would buy nothing: an
// e4m3 code's relative step does not depend on where in its range it lies.
#include "kernels.h"

namespace tension {

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxGrid = 1 << 20;  // workgroups along x; they loop over what is left

// Biased exponent byte of a row whose largest finite magnitude has these bits.
__device__ __forceinline__ int exp_byte(unsigned amax_bits) {
  const int e = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return e < 1 ? 1 : e;
}
__device__ __forceinline__ float pow2_of_byte(int b) { return __builtin_bit_cast(float, (unsigned)b << 23); }

// Magnitude bits of a finite value, 0 for infinities and NaN.
__device__ __forceinline__ unsigned finite_bits(float x) {
  const unsigned b = __builtin_bit_cast(unsigned, x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// Value to quantise: scaled, infinities as NaN (e4m3 has none).
__device__ __forceinline__ float to_code_range(float x, float inv) {
  return finite_bits(x) || x == 0.f ? x * inv : __builtin_nanf("");
}

__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Page and row of position pos of sequence n; false where there is no place.
__device__ __forceinline__ bool place(const PagedCache& c, int n, int pos, int64_t* page, int* row) {
  if (pos < 0 || pos / c.S >= c.table_len) return false;
  const int id = c.table[(int64_t)n * c.table_stride + pos / c.S];
  *page = id;
  *row = pos % c.S;
  return id >= 0 && id < c.P;
}

// Token t of sequence n is one of the call's (start[n] + t does not wrap:
// past INT_MAX it is no position).
__device__ __forceinline__ bool token_pos(const PagedRowsParams& p, int n, int t, int* pos) {
  if (t >= p.T || (p.counts && t >= p.counts[n])) return false;
  const int64_t q = (int64_t)p.start[n] + t;
  *pos = (int)q;
  return q >= 0 && q <= 0x7fffffff;
}

__device__ __forceinline__ float code_value(uint8_t c) {
  return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}

// ------------------------------------------------------------------ any head dim, any alignment

__device__ __forceinline__ float ld_page(const Buf& b, int64_t off) {
  return b.dt == TENSION_E4M3 ? code_value(((const uint8_t*)b.p)[off]) : ld<float>(b, off);
}

// Row r = (n, h, t) by one wave, lanes along the row.
template <bool APPEND>
__device__ __forceinline__ void any_row(const PagedRowsParams& p, int64_t r, int lane) {
  const int t = (int)(r % p.T);
  const int64_t nh = r / p.T;
  const int h = (int)(nh % p.Hk), n = (int)(nh / p.Hk);
  const bool isv = blockIdx.y != 0;
  const Buf& pg = isv ? p.c.v : p.c.k;
  const Buf& de = isv ? p.vd : p.kd;
  uint8_t* ex = const_cast<uint8_t*>(isv ? p.c.ve : p.c.ke);
  const int64_t e0 = isv ? p.c.ve0 : p.c.ke0, e1 = isv ? p.c.ve1 : p.c.ke1, e2 = isv ? p.c.ve2 : p.c.ke2;
  const int64_t doff = n * de.s0 + t * de.s1 + h * de.s2;
  int64_t page = 0;
  int pos = 0, row = 0;
  const bool live = token_pos(p, n, t, &pos) && place(p.c, n, pos, &page, &row);
  if (APPEND && !live) return;
  const int64_t poff = page * pg.s0 + h * pg.s1 + row * pg.s2, eoff = page * e0 + h * e1 + row * e2;
  if constexpr (APPEND) {
    if (pg.dt != TENSION_E4M3) {
      for (int d = lane; d < p.D; d += 64) st<float>(pg, poff + d, ld<float>(de, doff + d));
      return;
    }
    unsigned top = 0;
    for (int d = lane; d < p.D; d += 64) {
      const unsigned b = finite_bits(ld<float>(de, doff + d));
      top = b > top ? b : top;
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) {
      const unsigned o = (unsigned)__shfl_xor((int)top, m);
      top = o > top ? o : top;
    }
    const int b = exp_byte(top);
    const float inv = pow2_of_byte(254 - b);
    for (int d = lane; d < p.D; d += 64)
      ((uint8_t*)pg.p)[poff + d] = (uint8_t)pack4(to_code_range(ld<float>(de, doff + d), inv), 0.f, 0.f, 0.f);
    if (lane == 0) ex[eoff] = (uint8_t)b;
  } else {
    const float f = live && pg.dt == TENSION_E4M3 ? pow2_of_byte(ex[eoff]) : 1.f;
    for (int d = lane; d < p.D; d += 64) st<float>(de, doff + d, live ? ld_page(pg, poff + d) * f : 0.f);
  }
}

template <bool APPEND>
__global__ void __launch_bounds__(kThreads) paged_rows_any(PagedRowsParams p) {
  const int64_t rows = (int64_t)p.N * p.Hk * p.T, step = (int64_t)gridDim.x * (kThreads / 64);
  for (int64_t r = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); r < rows; r += step)
    any_row<APPEND>(p, r, threadIdx.x & 63);
}

}  // namespace

int launch_paged_rows(bool append, const PagedRowsParams& p, hipStream_t st, hipError_t* err) {
  const int64_t rows = (int64_t)p.N * p.Hk * p.T;
  int64_t grid = (rows + kThreads / 64 - 1) / (kThreads / 64);
  grid = grid < kMaxGrid ? grid : kMaxGrid;
  if (append)
    paged_rows_any<true><<<dim3((unsigned)grid, 2), kThreads, 0, st>>>(p);
  else
    paged_rows_any<false><<<dim3((unsigned)grid, 2), kThreads, 0, st>>>(p);
  *err = hipGetLastError();
  return 0;
}

}  // namespace tension
