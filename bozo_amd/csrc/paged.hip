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
#include <type_traits>

#include "paged.h"

namespace tension {

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxGrid = 1 << 20;  // workgroups along x; they loop over what is left

// Biased exponent byte of a row whose largest finite magnitude has these bits.
__device__ __forceinline__ int exp_byte(unsigned amax_bits) {
  const int e = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return e < 1 ? 1 : e;
}

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

// ------------------------------------------------------------------ whole pieces of 8 values

struct VecGeometry {
  FastDiv heads, tiles, page;
  int ntile, lg_tile;  // tiles of 2^lg_tile tokens of one sequence
  int units;           // N * ntile * Hk * 2^lg_tile rows
};

template <int CTRL>
__device__ __forceinline__ unsigned dpp_umax(unsigned x) {
  const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);
  return o > x ? o : x;
}

// Largest over an aligned group of LPR lanes.
template <int LPR>
__device__ __forceinline__ unsigned group_umax(unsigned x) {
  if constexpr (LPR >= 2) x = dpp_umax<0xB1>(x);    // lane ^ 1
  if constexpr (LPR >= 4) x = dpp_umax<0x4E>(x);    // lane ^ 2
  if constexpr (LPR >= 8) x = dpp_umax<0x141>(x);   // mirrored halves of 8
  if constexpr (LPR >= 16) x = dpp_umax<0x140>(x);  // mirrored rows of 16
  if constexpr (LPR >= 32) {
    const unsigned o = (unsigned)__shfl_xor((int)x, 16);
    x = o > x ? o : x;
  }
  return x;
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// Eight dense values as they are loaded, and as floats.
template <bool F32>
struct Eight {
  u32x4 a[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const Buf& b, int64_t off) {
    const u32x4* s = (const u32x4*)((const char*)b.p + off * (F32 ? 4 : 2));
    a[0] = s[0];
    if constexpr (F32) a[1] = s[1];
  }
  __device__ __forceinline__ void store(const Buf& b, int64_t off) const {
    u32x4* s = (u32x4*)((char*)const_cast<void*>(b.p) + off * (F32 ? 4 : 2));
    s[0] = a[0];
    if constexpr (F32) s[1] = a[1];
  }
  __device__ __forceinline__ void floats(bool half, float* x) const {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned w = a[i / 4][i % 4];  // a copy: bit_cast of a vector's element takes element 0
        x[i] = __builtin_bit_cast(float, w);
      }
    } else if (half) {
      const f16x8 h = __builtin_bit_cast(f16x8, a[0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
    } else {
      const bf16x8 h = __builtin_bit_cast(bf16x8, a[0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
    }
  }
  __device__ __forceinline__ void set(bool half, const float* x) {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i / 4][i % 4] = __builtin_bit_cast(unsigned, x[i]);
    } else if (half) {
      f16x8 h;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = (f16)x[i];
      a[0] = __builtin_bit_cast(u32x4, h);
    } else {
      bf16x8 h;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = (bf16)x[i];
      a[0] = __builtin_bit_cast(u32x4, h);
    }
  }
};

// LPR lanes to a row, eight values to a lane, R rows to a thread (their loads
// ahead of the first use).  A workgroup's consecutive rows are tokens of one
// head: their places in a page lie together, and in the dense tensor each is a
// piece of D values of its token.
template <bool APPEND, int LPR, int R, bool F32>
__device__ __forceinline__ void vec_rows(const PagedRowsParams& p, const VecGeometry& g, bool isv) {
  constexpr int kRows = kThreads / LPR;
  const Buf& pg = isv ? p.c.v : p.c.k;
  const Buf& de = isv ? p.vd : p.kd;
  uint8_t* ex = const_cast<uint8_t*>(isv ? p.c.ve : p.c.ke);
  const int64_t e0 = isv ? p.c.ve0 : p.c.ke0, e1 = isv ? p.c.ve1 : p.c.ke1, e2 = isv ? p.c.ve2 : p.c.ke2;
  const int ch = threadIdx.x % LPR * 8;
  int64_t doff[R], poff[R], eoff[R];
  bool live[R], in[R];
  Eight<F32> x[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int u = (blockIdx.x * R + r) * kRows + threadIdx.x / LPR;
    const int y = u >> g.lg_tile, z = fdiv(y, g.heads), h = y - z * p.Hk;
    const int n = fdiv(z, g.tiles), t = ((z - n * g.ntile) << g.lg_tile) + (u & ((1 << g.lg_tile) - 1));
    in[r] = u < g.units && t < p.T;
    doff[r] = n * de.s0 + t * de.s1 + h * de.s2 + ch;
    live[r] = false;
    int pos = 0;
    if (in[r] && token_pos(p, n, t, &pos)) {
      const int slot = fdiv(pos, g.page), row = pos - slot * p.c.S;
      if (APPEND) x[r].load(de, doff[r]);
      if (slot < p.c.table_len) {
        const int id = p.c.table[(int64_t)n * p.c.table_stride + slot];
        live[r] = id >= 0 && id < p.c.P;
        poff[r] = id * pg.s0 + h * pg.s1 + row * pg.s2 + ch;
        eoff[r] = id * e0 + h * e1 + row * e2;
      }
    }
  }
  const bool half = de.dt == TENSION_F16, quantised = pg.dt == TENSION_E4M3;
  if constexpr (APPEND) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (!live[r]) continue;  // a row's lanes agree
      if (!quantised) {
        if (pg.dt == de.dt) {
          x[r].store(pg, poff[r]);
        } else {  // float32 tokens, 16-bit pages
          float f[8];
          x[r].floats(half, f);
          Eight<false> y;
          y.set(pg.dt == TENSION_F16, f);
          y.store(pg, poff[r]);
        }
        continue;
      }
      float f[8];
      x[r].floats(half, f);
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned b = finite_bits(f[i]);
        top = b > top ? b : top;
      }
      const int b = exp_byte(group_umax<LPR>(top));
      const float inv = pow2_of_byte(254 - b);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = to_code_range(f[i], inv);
      *(u32x2*)((uint8_t*)pg.p + poff[r]) = u32x2{pack4(f[0], f[1], f[2], f[3]), pack4(f[4], f[5], f[6], f[7])};
      if (ch == 0) ex[eoff[r]] = (uint8_t)b;
    }
  } else {
    if (quantised) {
      u32x2 c[R];
      uint8_t b[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        c[r] = live[r] ? *(const u32x2*)((const uint8_t*)pg.p + poff[r]) : u32x2{0, 0};
        b[r] = live[r] ? ex[eoff[r]] : 127;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float f[8];
        const float s = pow2_of_byte(b[r]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f[4 * i] = __builtin_amdgcn_cvt_f32_fp8((int)c[r][i], 0) * s;
          f[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8((int)c[r][i], 1) * s;
          f[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8((int)c[r][i], 2) * s;
          f[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8((int)c[r][i], 3) * s;
        }
        x[r].set(half, f);
        if (in[r]) x[r].store(de, doff[r]);
      }
      return;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (!in[r]) continue;
      float f[8] = {};
      if (!live[r]) {
        x[r].set(half, f);
      } else if (pg.dt == de.dt) {
        x[r].load(pg, poff[r]);
      } else if (pg.dt == TENSION_F32) {
        Eight<true> y;
        y.load(pg, poff[r]);
        y.floats(false, f);
        x[r].set(half, f);
      } else {
        Eight<false> y;
        y.load(pg, poff[r]);
        y.floats(pg.dt == TENSION_F16, f);
        x[r].set(half, f);
      }
      x[r].store(de, doff[r]);
    }
  }
}

template <bool APPEND, int LPR, int R>
__global__ void __launch_bounds__(kThreads) paged_rows_vec(PagedRowsParams p, VecGeometry g) {
  const bool isv = blockIdx.y != 0;
  if ((isv ? p.vd.dt : p.kd.dt) == TENSION_F32)
    vec_rows<APPEND, LPR, R, true>(p, g, isv);
  else
    vec_rows<APPEND, LPR, R, false>(p, g, isv);
}

// Pieces of 8 values of a row are whole 16-byte (8-byte: e4m3) pieces of memory.
bool vec_aligned(const Buf& b) {
  const int64_t bytes = b.dt == TENSION_E4M3 ? 1 : b.dt == TENSION_F32 ? 4 : 2, to = b.dt == TENSION_E4M3 ? 8 : 16;
  return (uintptr_t)b.p % to == 0 && b.s0 * bytes % to == 0 && b.s1 * bytes % to == 0 && b.s2 * bytes % to == 0;
}

template <bool APPEND, int R>
bool launch_vec(const PagedRowsParams& p, const VecGeometry& g, hipStream_t st) {
  auto go = [&](auto lanes) {
    constexpr int LPR = decltype(lanes)::value;
    const int per = kThreads / LPR * R;
    paged_rows_vec<APPEND, LPR, R><<<dim3((unsigned)((g.units + per - 1) / per), 2), kThreads, 0, st>>>(p, g);
    return true;
  };
  switch (p.D) {
    case 32: return go(std::integral_constant<int, 4>{});
    case 64: return go(std::integral_constant<int, 8>{});
    case 128: return go(std::integral_constant<int, 16>{});
    case 256: return go(std::integral_constant<int, 32>{});
    default: return false;
  }
}

// Head dims 32 to 256 (powers of two) with aligned rows.
bool try_vec(bool append, const PagedRowsParams& p, hipStream_t st) {
  if (!vec_aligned(p.kd) || !vec_aligned(p.vd) || !vec_aligned(p.c.k) || !vec_aligned(p.c.v)) return false;
  VecGeometry g;
  g.lg_tile = 0;
  while (g.lg_tile < 5 && (1 << g.lg_tile) < p.T) ++g.lg_tile;
  g.ntile = (int)(((int64_t)p.T + (1 << g.lg_tile) - 1) >> g.lg_tile);
  const int64_t units = mul_cap(mul_cap((int64_t)p.N * g.ntile, p.Hk, 1 << 30), (int64_t)1 << g.lg_tile, 1 << 30);
  if (units < 0) return false;
  g.units = (int)units;
  g.heads = fast_div(p.Hk);
  g.tiles = fast_div(g.ntile);
  g.page = fast_div(p.c.S);
  // several rows to a thread once the grid fills the card many times over
  const bool many = units * (p.D / 8) >= (int64_t)kThreads * device_cus() * 32;
  if (append) return many ? launch_vec<true, 4>(p, g, st) : launch_vec<true, 1>(p, g, st);
  return many ? launch_vec<false, 4>(p, g, st) : launch_vec<false, 1>(p, g, st);
}

}  // namespace

int launch_paged_rows(bool append, const PagedRowsParams& p, hipStream_t st, hipError_t* err) {
  if (try_vec(append, p, st)) {
    *err = hipGetLastError();
    return 0;
  }
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
