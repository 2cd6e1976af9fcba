// Paged K/V cache: tokens written into pages (quantised to e4m3 on the way or
// as they are) and read back dense.  Both are streams: a row of D values is
// read once and written once, so HBM bounds them (bf16 prompts, 262 MB: 50 us,
// 5.3 TB/s, what a large copy reaches; e4m3 read back, 303 MB: 62-66 us), and below
// some 20 MB the chain of start, table, rows (about 4 us).  A read needs that
// chain; an append's dense rows do not depend on it, but are loaded for tokens
// that have a place only, so they wait for it too.
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
  int ntile;  // groups of R tokens of a sequence
  int units;  // N * ntile * Hk: R tokens of one head
  bool runs;  // order of the workgroups
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

// The eight values of a lane, two groups of four: side by side, or, for
// float32 dense rows, half a row apart, so that a wave's 16-byte accesses of
// them cover whole lines.
struct Quads {
  int a, b;
};
template <bool F32>
__device__ __forceinline__ Quads lane_quads(int lane, int D) {
  return F32 ? Quads{4 * lane, D / 2 + 4 * lane} : Quads{8 * lane, 8 * lane + 4};
}

template <typename V>
__device__ __forceinline__ void floats_as(u32x4 w, float* x) {
  const V h = __builtin_bit_cast(V, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
}
template <typename V, typename T>
__device__ __forceinline__ u32x4 rounded_as(const float* x) {
  V h;
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = (T)x[i];
  return __builtin_bit_cast(u32x4, h);
}

// A store past the L2s, whose lines a kernel has to write back at its end
// anyway: 16 x 256 tokens read 7.1 -> 5.6 us, 19.6 -> 18.9 with the kernel that
// reads the result; bf16 prompts 52.5 -> 49.6, 105.1 -> 103.3 with their read.
template <typename V>
__device__ __forceinline__ void stream(void* p, V v) {
  __builtin_nontemporal_store(v, (V*)p);
}

// Eight values of a row of float32 (WIDE) or 16-bit type, as they are loaded.
template <bool WIDE>
struct Eight {
  u32x4 a[WIDE ? 2 : 1];
  __device__ __forceinline__ void load(const Buf& b, int64_t off, Quads q) {
    if constexpr (WIDE) {
      a[0] = *(const u32x4*)((const float*)b.p + off + q.a);
      a[1] = *(const u32x4*)((const float*)b.p + off + q.b);
    } else if (q.b == q.a + 4) {
      a[0] = *(const u32x4*)((const f16*)b.p + off + q.a);
    } else {
      const u32x2 x = *(const u32x2*)((const f16*)b.p + off + q.a), y = *(const u32x2*)((const f16*)b.p + off + q.b);
      a[0] = u32x4{x[0], x[1], y[0], y[1]};
    }
  }
  __device__ __forceinline__ void store(const Buf& b, int64_t off, Quads q) const {
    void* p = const_cast<void*>(b.p);
    if constexpr (WIDE) {
      stream((float*)p + off + q.a, a[0]);
      stream((float*)p + off + q.b, a[1]);
    } else if (q.b == q.a + 4) {
      stream((f16*)p + off + q.a, a[0]);
    } else {
      stream((f16*)p + off + q.a, u32x2{a[0][0], a[0][1]});
      stream((f16*)p + off + q.b, u32x2{a[0][2], a[0][3]});
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (WIDE ? 2 : 1); ++i) a[i] = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void floats(bool half, float* x) const {
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned w = a[i / 4][i % 4];  // a copy: bit_cast of a vector's element takes element 0
        x[i] = __builtin_bit_cast(float, w);
      }
    } else if (half) {
      floats_as<f16x8>(a[0], x);
    } else {
      floats_as<bf16x8>(a[0], x);
    }
  }
  __device__ __forceinline__ void set(bool half, const float* x) {
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i / 4][i % 4] = __builtin_bit_cast(unsigned, x[i]);
    } else if (half) {
      a[0] = rounded_as<f16x8, f16>(x);
    } else {
      a[0] = rounded_as<bf16x8, bf16>(x);
    }
  }
};

// The places of R consecutive tokens of one head.
template <int R>
struct Places {
  int n, h, t, id[R], row[R];
  bool in[R], live[R];  // the call's tokens; those with a place
};

// One side (K or V) of R rows: eight values to a lane, all loads ahead of the
// first use.
template <bool APPEND, int LPR, int R, bool F32>
struct Side {
  Eight<F32> x[R];
  u32x2 c[R];
  uint8_t b[R];

  static __device__ __forceinline__ int64_t page_off(const Buf& pg, const Places<R>& w, int r) {
    return w.id[r] * pg.s0 + w.h * pg.s1 + w.row[r] * pg.s2;
  }

  __device__ __forceinline__ void load(const Buf& de, const Buf& pg, const uint8_t* ex, int64_t e0, int64_t e1, int64_t e2,
                                       const Places<R>& w, int lane, int D) {
    const Quads q = lane_quads<F32>(lane, D);
    const bool mine = 8 * lane < D;  // a lane past the head dim follows its row with zeros
    if constexpr (APPEND) {
      const int64_t off = w.n * de.s0 + w.t * de.s1 + w.h * de.s2;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (!mine) x[r].zero();
        if (mine && w.live[r]) x[r].load(de, off + r * de.s1, q);
      }
      return;
    }
    if (pg.dt == TENSION_E4M3) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool live = mine && w.live[r];
        const uint8_t* s = (const uint8_t*)pg.p + (live ? page_off(pg, w, r) : 0);
        if constexpr (F32)
          c[r] = u32x2{live ? *(const unsigned*)(s + q.a) : 0, live ? *(const unsigned*)(s + q.b) : 0};
        else
          c[r] = live ? *(const u32x2*)(s + q.a) : u32x2{0, 0};
        b[r] = w.live[r] ? ex[w.id[r] * e0 + w.h * e1 + w.row[r] * e2] : 127;
      }
    } else if (pg.dt == de.dt) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        x[r].zero();
        if (mine && w.live[r]) x[r].load(pg, page_off(pg, w, r), q);
      }
    }
  }

  __device__ __forceinline__ void store(const Buf& de, const Buf& pg, uint8_t* ex, int64_t e0, int64_t e1, int64_t e2,
                                        const Places<R>& w, int lane, int D) {
    const Quads q = lane_quads<F32>(lane, D);
    const bool mine = 8 * lane < D;  // a lane past the head dim follows its row with zeros
    const bool half = de.dt == TENSION_F16;
    if constexpr (APPEND) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (!w.live[r]) continue;  // a row's lanes agree
        const int64_t off = page_off(pg, w, r);
        if (pg.dt == de.dt) {
          if (mine) x[r].store(pg, off, q);
          continue;
        }
        float f[8];
        x[r].floats(half, f);
        if (pg.dt != TENSION_E4M3) {  // float32 tokens, 16-bit pages
          Eight<false> y;
          y.set(pg.dt == TENSION_F16, f);
          if (mine) y.store(pg, off, q);
          continue;
        }
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const unsigned m = finite_bits(f[i]);
          top = m > top ? m : top;
        }
        const int e = exp_byte(group_umax<LPR>(top));
        const float inv = pow2_of_byte(254 - e);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_code_range(f[i], inv);
        const u32x2 codes = {pack4(f[0], f[1], f[2], f[3]), pack4(f[4], f[5], f[6], f[7])};
        uint8_t* to = (uint8_t*)pg.p + off;
        if constexpr (F32) {
          if (mine) {
            *(unsigned*)(to + q.a) = codes[0];
            *(unsigned*)(to + q.b) = codes[1];
          }
        } else if (mine) {
          *(u32x2*)(to + q.a) = codes;
        }
        if (lane == 0) ex[w.id[r] * e0 + w.h * e1 + w.row[r] * e2] = (uint8_t)e;
      }
      return;
    }
    const int64_t off = w.n * de.s0 + w.t * de.s1 + w.h * de.s2;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (!mine || !w.in[r]) continue;
      if (pg.dt == TENSION_E4M3) {
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
      } else if (pg.dt != de.dt) {
        float f[8] = {};
        if (w.live[r]) {
          const int64_t from = page_off(pg, w, r);
          if (pg.dt == TENSION_F32) {
            Eight<true> y;
            y.load(pg, from, q);
            y.floats(false, f);
          } else {
            Eight<false> y;
            y.load(pg, from, q);
            y.floats(pg.dt == TENSION_F16, f);
          }
        }
        x[r].set(half, f);
      }
      x[r].store(de, off + r * de.s1, q);
    }
  }
};

// LPR lanes to a row, R tokens of one head to a thread, K and V both.
// Consecutive units are heads of one token, so a wave's rows lie together in
// the dense tensors, and a thread's tokens lie together in a page.  (Tokens of
// one head side by side, K and V apart: prompts 73.5 us for 52, read 123 for 62.)
// Neighbouring workgroups, whose rows share lines of a page, run on one XCD
// (16 x 256 tokens read 7.3 -> 6.9 us then, append of 8 x 4096 tokens to e4m3 52.6 -> 51.7).
template <bool APPEND, int LPR, int R, bool KF32, bool VF32>
__global__ void __launch_bounds__(kThreads) paged_rows_vec(PagedRowsParams p, VecGeometry g) {
  const int lane = threadIdx.x % LPR;
  // neighbours on one XCD: all of its share, or runs of eight for many prompts of different lengths
  const int id = (int)blockIdx.x, in64 = id % 64;
  const int b = g.runs ? id - in64 + in64 % 8 * 8 + in64 / 8 : xcd_swizzle(id, (int)gridDim.x);
  const int u = b * (kThreads / LPR) + threadIdx.x / LPR;
  if (u >= g.units) return;
  Places<R> w;
  const int y = fdiv(u, g.heads);
  w.h = u - y * p.Hk;
  w.n = fdiv(y, g.tiles);
  w.t = (y - w.n * g.ntile) * R;
  const int64_t first = (int64_t)p.start[w.n] + w.t;
  const int count = p.counts ? p.counts[w.n] : p.T;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t pos = first + r;
    w.in[r] = w.t + r < p.T;
    w.live[r] = false;
    w.id[r] = w.row[r] = 0;
    if (w.in[r] && w.t + r < count && pos >= 0 && pos <= 0x7fffffff) {
      const int slot = fdiv((int)pos, g.page);
      if (slot < p.c.table_len) {
        w.id[r] = p.c.table[(int64_t)w.n * p.c.table_stride + slot];
        w.row[r] = (int)pos - slot * p.c.S;
        w.live[r] = w.id[r] >= 0 && w.id[r] < p.c.P;
      }
    }
  }
  Side<APPEND, LPR, R, KF32> k;
  Side<APPEND, LPR, R, VF32> v;
  uint8_t *ke = const_cast<uint8_t*>(p.c.ke), *ve = const_cast<uint8_t*>(p.c.ve);
  k.load(p.kd, p.c.k, ke, p.c.ke0, p.c.ke1, p.c.ke2, w, lane, p.D);
  v.load(p.vd, p.c.v, ve, p.c.ve0, p.c.ve1, p.c.ve2, w, lane, p.D);
  k.store(p.kd, p.c.k, ke, p.c.ke0, p.c.ke1, p.c.ke2, w, lane, p.D);
  v.store(p.vd, p.c.v, ve, p.c.ve0, p.c.ve1, p.c.ve2, w, lane, p.D);
}

// Pieces of 8 values of a row are whole pieces of memory.
bool vec_aligned(const Buf& b) { return row_pieces(b, b.dt == TENSION_E4M3 ? 8 : 16); }

template <bool APPEND, int R, bool KF32, bool VF32>
bool launch_vec(const PagedRowsParams& p, hipStream_t st) {
  VecGeometry g;
  g.ntile = (p.T + R - 1) / R;
  const int64_t units = mul_cap((int64_t)p.N * g.ntile, p.Hk, 1 << 30);
  if (units < 0) return false;
  g.units = (int)units;
  g.heads = fast_div(p.Hk);
  g.tiles = fast_div(g.ntile);
  g.page = fast_div(p.c.S);
  auto go = [&](auto lanes) {
    constexpr int LPR = decltype(lanes)::value;
    const int per = kThreads / LPR;
    unsigned n = (unsigned)((g.units + per - 1) / per);
    g.runs = APPEND && n >= 2048;
    n = g.runs ? (n + 63) / 64 * 64 : (n + 7) / 8 * 8;
    if (!launchable(n, kThreads)) return false;  // the kernel for any rows loops over them
    paged_rows_vec<APPEND, LPR, R, KF32, VF32><<<n, kThreads, 0, st>>>(p, g);
    return true;
  };
  if (p.D <= 32) return go(std::integral_constant<int, 4>{});
  if (p.D <= 64) return go(std::integral_constant<int, 8>{});
  if (p.D <= 128) return go(std::integral_constant<int, 16>{});
  return go(std::integral_constant<int, 32>{});
}

template <bool APPEND, int R>
bool launch_types(const PagedRowsParams& p, hipStream_t st) {
  const bool k = p.kd.dt == TENSION_F32, v = p.vd.dt == TENSION_F32;
  if (k) return v ? launch_vec<APPEND, R, true, true>(p, st) : launch_vec<APPEND, R, true, false>(p, st);
  return v ? launch_vec<APPEND, R, false, true>(p, st) : launch_vec<APPEND, R, false, false>(p, st);
}

// Head dims in eights up to 256 with aligned rows.
bool try_vec(bool append, const PagedRowsParams& p, hipStream_t st) {
  if (p.D % 8 || p.D > 256) return false;
  if (!vec_aligned(p.kd) || !vec_aligned(p.vd) || !vec_aligned(p.c.k) || !vec_aligned(p.c.v)) return false;
  const int64_t threads = mul_cap((int64_t)p.N * p.T, (int64_t)p.Hk * p.D / 8, (int64_t)1 << 40);
  // Two tokens to a thread for reads that fill the card more than once (E4M3 to bf16, N8 Hk16 D64: T1024 12.6 -> 10.4
  // us, T4096 52.6 -> 40.4; T256 5.9 either way); four were no faster (41.8), and appending was fastest with one.
  const bool two = threads < 0 || threads >= (int64_t)kThreads * device_cus() * 8;
  if (append) return launch_types<true, 1>(p, st);
  return two ? launch_types<false, 2>(p, st) : launch_types<false, 1>(p, st);
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
