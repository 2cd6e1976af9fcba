// Paged decode on the matrix units, for a key head that two or more query
// heads share: bf16 pages with bf16 queries, e4m3 pages with 16-bit ones, head
// dims 64 and 128.
//
// A wave takes 32 keys at a time, two tiles of 16 (a tile lies in one page).
// S = K q^T (16 keys x 16 query heads a tile) leaves lane (g = lane / 16, c =
// lane % 16) with the scores of keys 4g .. 4g + 3 of both tiles for query c.
// That is an A operand of the second product already, with its k = 8g + 4t + i
// standing for key 4g + i of tile t: tau never moves between lanes.  Its B
// operand needs the same eight keys of one feature in a lane, so lane (g, c)
// loads the pieces c of those eight rows and transposes them in registers.
//
// Roundings: K, q and V enter as they are (an e4m3 code is a bf16 and an f16
// number; its row's scale is applied to the score, or to tau).  tau enters as
// three bf16 terms that make up its float32 value; sums are float32.
//
// Bound by HBM: vector instructions issue in a quarter of a wave's cycles (e4m3,
// head dim 128), and the time hardly grows with the heads (two to sixteen: bf16
// D64, 268 MB, 45-48 us, 5.6-6 TB/s; bf16 D128, 268 MB, 67-69 us; e4m3 D128, N2,
// 65500 keys, 135 MB: 25.8 us, 5.2 TB/s, 31-32 with the join).  The third term
// of tau costs e4m3 4% at D64 and 2% at D128, bf16 at most 1%.
// The next step's K and V are loaded as soon as this step's are operands.
// Three waves per SIMD for e4m3 at head dim 128 (158 registers); bf16 there
// keeps two (three spilled and took 12% longer).
#include "mfma_common.h"
#include "paged.h"

namespace tension {

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kTileKeys = 16, kStep = 32;

// Two codes of word w (the upper pair: HI) as bf16 or f16.
template <bool F16, bool HI>
__device__ __forceinline__ unsigned codes2(unsigned w) {
  if constexpr (F16) {
    const f16x2 x = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI);
    return __builtin_bit_cast(unsigned, x);
  } else {
    const bf16x2 x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI);
    return __builtin_bit_cast(unsigned, x);
  }
}

template <bool F16>
__device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Low (HI: high) halves of a and b.
template <bool HI>
__device__ __forceinline__ unsigned halves(unsigned a, unsigned b) {
  return __builtin_amdgcn_perm(b, a, HI ? 0x07060302u : 0x05040100u);
}

// F8: e4m3 pages, else bf16.  QF16: queries are f16 (F8 only).
template <bool F8, bool QF16, int D, int kWaves>
__global__ void __launch_bounds__(64 * kWaves, F8 || D == 64 ? 3 : 2) paged_decode_mfma(PagedDecodeParams p, DecodeGrid grid) {
  constexpr int kElt = F8 ? 1 : 2;
  constexpr int KP = D * kElt / 64;      // 16-byte pieces a lane loads of a tile's K: 64 bytes of a row each
  constexpr int KS = D / 32;             // products of a tile's scores
  constexpr int VN = D / 16;             // values of a lane's piece of a V row
  constexpr int VW = VN * kElt / 4;      // 32-bit words of it
  __shared__ float red[kWaves][16][D + 1];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int n, len, hk, grp, split;
  grid.place((int)blockIdx.x, p, &n, &len, &hk, &grp, &split);
  const int h0 = hk * grid.share + grp * 16, nh = grid.share - grp * 16 < 16 ? grid.share - grp * 16 : 16;
  const KeyRange all = key_range(p, len), r = split_range(p, all, split);
  if (p.splits > 1 && split >= used_splits(p, all)) return;

  const char* kbase = (const char*)p.c.k.p + (int64_t)hk * p.c.k.s1 * kElt;
  const char* vbase = (const char*)p.c.v.p + (int64_t)hk * p.c.v.s1 * kElt;
  const uint8_t* kebase = p.c.ke + (F8 ? (int64_t)hk * p.c.ke1 : 0);
  const uint8_t* vebase = p.c.ve + (F8 ? (int64_t)hk * p.c.ve1 : 0);
  const int32_t* table = p.c.table + (int64_t)n * p.c.table_stride;
  const unsigned koff = (unsigned)(c * p.c.k.s2) * kElt + 16 * g;       // row c, byte 16 g of each 64
  const unsigned voff = (unsigned)(4 * g * p.c.v.s2) * kElt + c * VW * 4;  // rows 4g .. 4g + 3, piece c
  const unsigned vrow = (unsigned)p.c.v.s2 * kElt;
  const float scale = -p.inv_scale * kLog2e;

  u32x4 kr[2][KP];       // tile t: row c
  unsigned vr[2][4][VW];  // tile t: rows 4g + i, piece c
  unsigned ke[2], ve[2];  // exponent bytes of rows 4g .. 4g + 3
  bool page_ok[2];
  auto where = [&](int64_t base, int t, int* id, int* row) {
    const unsigned pos = (unsigned)base + t * kTileKeys, hi = (unsigned)r.hi;
    const int at = pos < hi ? (int)pos : r.hi - 1;
    const int slot = fdiv(at, grid.page);
    const int x = table[slot];
    *row = pos < hi ? at - slot * p.c.S : 0;  // a tile past the end reads its page's first
    page_ok[t] = x >= 0 && x < p.c.P;
    *id = page_ok[t] ? x : 0;
  };
  DecodeGrid::Place at[2];
  auto load_k = [&](int64_t base) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      int id, row;
      where(base, t, &id, &row);
      at[t] = grid.at<F8, false>(id, row);
      const char* s = kbase + at[t].k * kElt;
#pragma unroll
      for (int i = 0; i < KP; ++i) kr[t][i] = __builtin_nontemporal_load((const u32x4*)(s + koff + 64 * i));
      if constexpr (F8) {
        ke[t] = *(const unsigned*)(kebase + at[t].ke + 4 * g);
        ve[t] = *(const unsigned*)(vebase + at[t].ve + 4 * g);
      }
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char* s = vbase + at[t].v * kElt;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        typedef unsigned piece __attribute__((ext_vector_type(VW)));
        if constexpr (VW == 1) {
          vr[t][i][0] = __builtin_nontemporal_load((const unsigned*)(s + (voff + i * vrow)));
        } else {
          const piece w = __builtin_nontemporal_load((const piece*)(s + (voff + i * vrow)));
#pragma unroll
          for (int j = 0; j < VW; ++j) vr[t][i][j] = w[j];
        }
      }
    }
  };

  f32x4 acc[VN];
#pragma unroll
  for (int j = 0; j < VN; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float mass = 0.f;
  const int64_t step = kWaves * kStep;
  int64_t base = r.lo / kTileKeys * kTileKeys + (int64_t)wave * kStep;
  if (base < r.hi) {
    load_k(base);
    load_v();
    // query c as the B operand of the scores: 8 values a product, in the order of K's pieces
    u32x4 q[KS];
    {
      const unsigned short* s = (const unsigned short*)p.q.p + (int64_t)n * p.q.s0 +
                                (int64_t)(h0 + (c < nh ? c : 0)) * p.q.s1;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int f = F8 ? 64 * (i / 2) + 16 * g + 8 * (i % 2) : 32 * i + 8 * g;
        q[i] = *(const u32x4*)(s + f);
      }
    }
    for (; base < r.hi; base += step) {
      const int64_t next = base + step;
      // scores
      f32x4 s[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          u32x4 a;
          if constexpr (F8) {
            const unsigned w0 = kr[t][i / 2][2 * (i % 2)], w1 = kr[t][i / 2][2 * (i % 2) + 1];
            a = u32x4{codes2<QF16, false>(w0), codes2<QF16, true>(w0), codes2<QF16, false>(w1), codes2<QF16, true>(w1)};
          } else {
            a = kr[t][i];
          }
          s[t] = product<QF16>(a, q[i], s[t]);
        }
      }
      bool ok[2][4];
      bool every = true;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned pos = (unsigned)base + t * kTileKeys + 4 * g + i;
          ok[t][i] = page_ok[t] && pos >= (unsigned)r.lo && pos < (unsigned)r.hi;
          every = every && ok[t][i];
        }
      const bool whole = __all(every);
      // tau, in A's order
      float tau[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = s[t][i] * scale;
          if constexpr (F8) x *= pow2_of_byte((ke[t] >> (8 * i)) & 0xff);
          x = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x));
          x = ok[t][i] ? x : 0.f;
          mass += x;
          if constexpr (F8) x = ok[t][i] ? x * pow2_of_byte((ve[t] >> (8 * i)) & 0xff) : 0.f;
          tau[t][i] = x;
        }
      // Three bf16 terms make up tau exactly: each of the first two is less than what is left and all are positive, so
      // an infinite value row stays infinite; the last has 8 significant bits at most.
      u32x4 term[3];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        unsigned w[3][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = tau[j / 2][2 * (j % 2) + e];
          const unsigned some = x == 0.f ? 0u : 0xffff0000u;
          w[0][e] = (__builtin_bit_cast(unsigned, x) - 1) & some;
          const float left = x - __builtin_bit_cast(float, w[0][e]);
          w[1][e] = (__builtin_bit_cast(unsigned, left) - 1) & some;
          w[2][e] = __builtin_bit_cast(unsigned, left - __builtin_bit_cast(float, w[1][e]));
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) term[i][j] = halves<true>(w[i][0], w[i][1]);
      }
      if (!whole) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < VW; ++j) vr[t][i][j] = ok[t][i] ? vr[t][i][j] : 0u;
      }
      // V: words of one key's values -> operands of one value's keys
      u32x4 bv[VN];
#pragma unroll
      for (int j = 0; j < VN / 2; ++j) {  // values 2j, 2j + 1
#pragma unroll
        for (int k = 0; k < 4; ++k) {     // keys 2k, 2k + 1: tile k / 2, rows 2 (k % 2), + 1
          unsigned a, d;
          if constexpr (F8) {
            const unsigned x = vr[k / 2][2 * (k % 2)][j / 2], y = vr[k / 2][2 * (k % 2) + 1][j / 2];
            a = j % 2 ? codes2<false, true>(x) : codes2<false, false>(x);
            d = j % 2 ? codes2<false, true>(y) : codes2<false, false>(y);
          } else {
            a = vr[k / 2][2 * (k % 2)][j];
            d = vr[k / 2][2 * (k % 2) + 1][j];
          }
          bv[2 * j][k] = halves<false>(a, d);
          bv[2 * j + 1][k] = halves<true>(a, d);
        }
      }
      if (next < r.hi) {
        load_k(next);
        load_v();
      }
#pragma unroll
      for (int j = 0; j < VN; ++j) {
#pragma unroll
        for (int i = 0; i < 3; ++i) acc[j] = product<false>(term[i], bv[j], acc[j]);
      }
    }
  }

  // acc[j]: rows = query heads 4g + i, column c = value c * VN + j
  mass += __shfl_xor(mass, 16);
  mass += __shfl_xor(mass, 32);
#pragma unroll
  for (int j = 0; j < VN; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[wave][4 * g + i][c * VN + j] = acc[j][i];
  if (g == 0) red[wave][c][D] = mass;
  __syncthreads();
  for (int i = tid; i < nh * D; i += 64 * kWaves) {
    const int h = i / D, d = i % D;
    float o = 0.f, m = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      o += red[w][h][d];
      m += red[w][h][D];
    }
    const int out_row = n * p.H + h0 + h;
    if (p.splits > 1) {
      split_sums(p, out_row, split)[d] = o;
      if (d == 0) *split_mass(p, out_row, split) = m;
    } else {
      st<float>(p.out, (int64_t)n * p.out.s0 + (int64_t)(h0 + h) * p.out.s1 + d, o * norm_factor(p, m, all));
    }
  }
}

template <bool F8, bool QF16>
void launch_as(const PagedDecodeParams& p, hipStream_t st) {
  const DecodeGrid grid(p, 16, 0);
  const unsigned n = grid.size(p);
  // eight waves where a CU has one workgroup
  const bool eight = n <= (unsigned)device_cus();
  if (p.D == 64)
    eight ? paged_decode_mfma<F8, QF16, 64, 8><<<n, 512, 0, st>>>(p, grid)
          : paged_decode_mfma<F8, QF16, 64, 4><<<n, 256, 0, st>>>(p, grid);
  else
    eight ? paged_decode_mfma<F8, QF16, 128, 8><<<n, 512, 0, st>>>(p, grid)
          : paged_decode_mfma<F8, QF16, 128, 4><<<n, 256, 0, st>>>(p, grid);
}

}  // namespace

bool launch_paged_decode_mfma(const PagedDecodeParams& p, hipStream_t st) {
  const bool f8 = p.c.k.dt == TENSION_E4M3;
  if ((p.D != 64 && p.D != 128) || p.c.S % kTileKeys || p.c.v.dt != p.c.k.dt) return false;
  if (f8 ? p.q.dt == TENSION_F32 : p.q.dt != TENSION_BF16 || p.c.k.dt != TENSION_BF16) return false;
  if (!row_pieces(p.c.k, 16) || !row_pieces(p.c.v, 16)) return false;
  if ((uintptr_t)p.q.p % 16 || p.q.s0 % 8 || p.q.s1 % 8) return false;
  if (f8) {  // exponents of four rows are one word
    const uintptr_t a = (uintptr_t)p.c.ke | (uintptr_t)p.c.ke0 | (uintptr_t)p.c.ke1;
    const uintptr_t b = (uintptr_t)p.c.ve | (uintptr_t)p.c.ve0 | (uintptr_t)p.c.ve1;
    if (p.c.ke2 != 1 || p.c.ve2 != 1 || (a | b) % 4) return false;
  }
  if (!f8) launch_as<false, false>(p, st);
  else if (p.q.dt == TENSION_F16) launch_as<true, true>(p, st);
  else launch_as<true, false>(p, st);
  return true;
}

}  // namespace tension
