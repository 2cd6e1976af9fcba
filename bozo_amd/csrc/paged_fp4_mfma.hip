// Paged decode of 4-bit pages on the matrix units, for a key head that two or
// more query heads share: head dims 32, 64, 96 and 128, queries of any type.
//
// A wave takes 32 keys at a time, two tiles of 16 (a tile lies in one page).
// S = K q^T (16 keys x 16 query heads a tile) leaves lane (g = lane / 16, c =
// lane % 16) with the scores of keys 4g .. 4g + 3 of both tiles for query c,
// which is an A operand of the second product already, with its k = 8g + 4t + i
// standing for key 4g + i of tile t: tau never moves between lanes.  The lane's
// quarter of key row c has one exponent; its values of V are those of the same
// eight keys, transposed in registers.
//
// Bound by HBM at head dim 128 (N64 H16 Hk4, 4000 keys, 139 MB: 27 us, 5.1 TB/s)
// and by its vector instructions below (64: 20 us for 70 MB; 32: 18 for 35): sixteen
// columns of tau are formed whatever the number of heads.  Head dim 96 is one of 64
// with one of 32 beside it, whose V comes in single bytes (37 us for 104 MB; a stream
// for each query head took 62, and 35 at 32).  What keeps them few: masks on their
// own branch, which whole steps skip (a second copy of the step instead took
// 60 registers more and a third of the speed of four-wave workgroups); an
// exponent turned into place by one rotation; a step under way and the places
// of the next looked up while one is added up.
//
// Roundings: codes become bf16 with their exponents, exactly; a query enters as
// it is, as two bf16 terms (f16) or as three (float32: all of a value's bits, if it
// is within 2^94 of the row's largest), tau as three bf16 terms that make up its
// float32 value; sums are float32.
#include "fp4.h"
#include "mfma_common.h"
#include "paged.h"

namespace tension {

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kTileKeys = 16, kStep = 32;

template <int SEL>
__device__ __forceinline__ unsigned codes2(unsigned w, float scale) {
  const bf16x2 x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL);
  return __builtin_bit_cast(unsigned, x);
}
// Eight codes as one operand.
__device__ __forceinline__ u32x4 codes8(unsigned w, float scale) {
  return u32x4{codes2<0>(w, scale), codes2<1>(w, scale), codes2<2>(w, scale), codes2<3>(w, scale)};
}

__device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Low (HI: high) halves of a and b.
template <bool HI>
__device__ __forceinline__ unsigned halves(unsigned a, unsigned b) {
  return __builtin_amdgcn_perm(b, a, HI ? 0x07060302u : 0x05040100u);
}

// Eight values of a query row as a bf16 operand.
__device__ __forceinline__ u32x4 query_bf16(const Buf& q, int64_t off, bool whole) {
  const unsigned short* s = (const unsigned short*)q.p + off;
  if (whole) return *(const u32x4*)s;
  u32x4 x;
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = s[2 * j] | (unsigned)s[2 * j + 1] << 16;
  return x;
}
// Eight values as NQ operands: bf16 terms that make them up, each but the last
// the leading eight bits of what is left.
template <int NQ>
__device__ __forceinline__ void query_terms(float* x, u32x4* term) {
#pragma unroll
  for (int i = 0; i < NQ; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      unsigned w[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float y = x[2 * j + e];
        w[e] = y == y ? __builtin_bit_cast(unsigned, y) & 0xffff0000u : 0x7fc00000u;
        const float left = y - __builtin_bit_cast(float, w[e]);
        // an infinity or a NaN is its first term's alone
        x[2 * j + e] = left == left ? left : 0.f;
      }
      term[i][j] = halves<true>(w[0], w[1]);
    }
}

// Which bytes of word w belong to row i, of four rows of G exponents each.
constexpr unsigned row_bytes(int G, int i, int w) {
  unsigned m = 0;
  for (int b = 0; b < 4; ++b)
    if ((4 * w + b) / G == i) m |= 0xffu << 8 * b;
  return m;
}

template <int QT, int D, int kWaves>
__global__ void __launch_bounds__(64 * kWaves) fp4_decode_mfma(PagedDecodeParams p, DecodeGrid grid) {
  constexpr int NQ = QT == TENSION_BF16 ? 1 : QT == TENSION_F16 ? 2 : 3;
  constexpr int G = D / 32;             // exponents of a row, and products of a tile's scores
  constexpr int W = D == 96 ? 64 : D;   // head dim 96 is one of 64 and one of 32 side by side
  constexpr bool kTail = W < D;
  constexpr int KS = W / 32, VN = W / 16, VA = D / 16;  // words, values of a lane's pieces of rows; its sums
  using VRaw = typename std::conditional<W == 128, unsigned, typename std::conditional<W == 64, unsigned short, uint8_t>::type>::type;
  typedef unsigned KRaw __attribute__((ext_vector_type(KS)));
  __shared__ float red[kWaves][16][D + 1];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int n, len, hk, grp, split;
  grid.place((int)blockIdx.x, p, &n, &len, &hk, &grp, &split);
  const int h0 = hk * grid.share + grp * 16, nh = grid.share - grp * 16 < 16 ? grid.share - grp * 16 : 16;
  const KeyRange all = key_range(p, len), r = split_range(p, all, split);
  if (p.splits > 1 && split >= used_splits(p, all)) return;

  const uint8_t* kbase = (const uint8_t*)p.c.k.p + (int64_t)hk * p.c.k.s1;
  const uint8_t* vbase = (const uint8_t*)p.c.v.p + (int64_t)hk * p.c.v.s1;
  const uint8_t* kebase = p.c.ke + (int64_t)hk * p.c.ke1;
  const uint8_t* vebase = p.c.ve + (int64_t)hk * p.c.ve1;
  const int32_t* table = p.c.table + (int64_t)n * p.c.table_stride;
  const unsigned krow = (unsigned)(c * p.c.k.s2), koff = krow + 4 * KS * g, kerow = (unsigned)(c * p.c.ke2), keoff = kerow + g * KS / 4;
  const unsigned vrow = (unsigned)p.c.v.s2, vfour = 4 * g * vrow, voff = vfour + c * (VN / 2), veoff = 4 * g * G;
  // Rotates the exponent of the lane's piece among its row's to where a scale operand has it; what else the word holds
  // falls on mantissa and sign, which the conversion does not take.
  const int vturn = c * KS / 16 * 8 + 9;
  float scale = -p.inv_scale * kLog2e;

  struct Places {
    int id[2], row[2];
    bool ok[2];
  };
  struct Raw {
    KRaw k[2];      // tile t: row c, quarter g
    VRaw v[2][4];   // tile t: rows 4g + i, piece c
    int ke[2];
    unsigned ve[2][G];  // of four rows
    unsigned kt[2];     // the tails
    uint8_t vt[2][4];
    int ket[2];
    bool ok[2];
  };
  auto look = [&](int64_t base) {
    Places w;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const unsigned pos = (unsigned)base + t * kTileKeys, hi = (unsigned)r.hi;
      const int at = pos < hi ? (int)pos : r.hi - 1;
      const int slot = fdiv(at, grid.page);
      const int id = table[slot];
      w.ok[t] = id >= 0 && id < p.c.P;
      w.id[t] = w.ok[t] ? id : 0;
      w.row[t] = pos < hi ? at - slot * p.c.S : 0;  // a tile past the end reads its page's first
    }
    return w;
  };
  auto load = [&](Raw& x, const Places& w) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const DecodeGrid::Place at = grid.at<true, false>(w.id[t], w.row[t]);
      x.ok[t] = w.ok[t];
      x.k[t] = __builtin_nontemporal_load((const KRaw*)(kbase + at.k + koff));
      x.ke[t] = (kebase + at.ke)[keoff];
#pragma unroll
      for (int i = 0; i < G; ++i) x.ve[t][i] = ((const unsigned*)(vebase + at.ve + veoff))[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) x.v[t][i] = __builtin_nontemporal_load((const VRaw*)(vbase + at.v + (voff + i * vrow)));
      if constexpr (kTail) {
        x.kt[t] = __builtin_nontemporal_load((const unsigned*)(kbase + at.k + (krow + W / 2 + 4 * g)));
        x.ket[t] = (kebase + at.ke)[kerow + KS];
#pragma unroll
        for (int i = 0; i < 4; ++i) x.vt[t][i] = __builtin_nontemporal_load(vbase + at.v + (vfour + i * vrow + W / 2 + c));
      }
    }
  };

  f32x4 acc[VA];
#pragma unroll
  for (int j = 0; j < VA; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float mass = 0.f;
  // query c as the B operand of the scores: values of quarter g, in the order of K's words
  u32x4 q[G][NQ];
  auto add = [&](Raw& x, int64_t base) {
    // scores
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      const float ks = fp4_scale(x.ke[t]);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const u32x4 a = codes8(x.k[t][i], ks);
#pragma unroll
        for (int j = 0; j < NQ; ++j) s[t] = product(a, q[i][j], s[t]);
      }
      if constexpr (kTail) {
        const u32x4 a = codes8(x.kt[t], fp4_scale(x.ket[t]));
#pragma unroll
        for (int j = 0; j < NQ; ++j) s[t] = product(a, q[KS][j], s[t]);
      }
    }
    // tau, in A's order
    float tau[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) tau[t][i] = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[t][i] * scale));
    if (!(x.ok[0] && x.ok[1] && base >= r.lo && base + kStep <= r.hi)) {
      // keys out of range hold anything: their tau is 0, and their exponents must be numbers
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned pos = (unsigned)base + t * kTileKeys + 4 * g + i;
          const bool ok = x.ok[t] & (pos >= (unsigned)r.lo) & (pos < (unsigned)r.hi);
          tau[t][i] = ok ? tau[t][i] : 0.f;
#pragma unroll
          for (int w = 0; w < G; ++w) {
            const unsigned gone = ok ? 0u : row_bytes(G, i, w);
            x.ve[t][w] = (x.ve[t][w] & ~gone) | (0x7f7f7f7fu & gone);
          }
        }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) mass += tau[t][i];
    u32x4 term[3];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      unsigned w[3][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float y = tau[j / 2][2 * (j % 2) + e];
        w[0][e] = __builtin_bit_cast(unsigned, y) & 0xffff0000u;
        const float left = y - __builtin_bit_cast(float, w[0][e]);
        w[1][e] = __builtin_bit_cast(unsigned, left) & 0xffff0000u;
        w[2][e] = __builtin_bit_cast(unsigned, left - __builtin_bit_cast(float, w[1][e]));
      }
#pragma unroll
      for (int i = 0; i < 3; ++i) term[i][j] = halves<true>(w[i][0], w[i][1]);
    }
    // V: pairs of one key's values -> operands of one value's keys
    u32x4 bv[VA];
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // keys 2k, 2k + 1: tile k / 2, rows 2 (k % 2), + 1
      unsigned w[2][VA / 2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = k / 2, i = 2 * (k % 2) + e;
        const int word = i * G / 4, at = i * G % 4;  // the first of the row's exponents
        unsigned e4 = x.ve[t][word], shift = 8 * at;
        if (at + KS > 4) e4 = __builtin_amdgcn_alignbit(x.ve[t][word + 1 < G ? word + 1 : word], e4, shift), shift = 0;
        const float vs = __builtin_bit_cast(float, __builtin_amdgcn_alignbit(e4, e4, (vturn + shift) & 31));
        const unsigned y = x.v[t][i];
        w[e][0] = codes2<0>(y, vs);
        if constexpr (kTail) {
          const unsigned t4 = x.ve[t][(i * G + KS) / 4];
          const float ts = __builtin_bit_cast(float, __builtin_amdgcn_alignbit(t4, t4, (8 * ((i * G + KS) % 4) + 9) & 31));
          w[e][VN / 2] = codes2<0>(x.vt[t][i], ts);
        }
        if constexpr (VN >= 4) w[e][1] = codes2<1>(y, vs);
        if constexpr (VN == 8) {
          w[e][2] = codes2<2>(y, vs);
          w[e][3] = codes2<3>(y, vs);
        }
      }
#pragma unroll
      for (int j = 0; j < VA / 2; ++j) {
        bv[2 * j][k] = halves<false>(w[0][j], w[1][j]);
        bv[2 * j + 1][k] = halves<true>(w[0][j], w[1][j]);
      }
    }
#pragma unroll
    for (int j = 0; j < VA; ++j) {
#pragma unroll
      for (int i = 0; i < 3; ++i) acc[j] = product(term[i], bv[j], acc[j]);
    }
  };
  const int64_t step = kWaves * kStep;
  int64_t base = r.lo / kTileKeys * kTileKeys + (int64_t)wave * kStep;
  if (base < r.hi) {
    Raw x0, x1;
    load(x0, look(base));
    Places w = look(base + step);
    {
      const bool whole = ((uintptr_t)p.q.p | (uintptr_t)(p.q.s0 * 2) | (uintptr_t)(p.q.s1 * 2)) % 16 == 0;
      const int64_t off = (int64_t)n * p.q.s0 + (int64_t)(h0 + (c < nh ? c : 0)) * p.q.s1;
      auto piece = [&](int i) { return off + (i < KS ? g * (W / 4) + 8 * i : W + 8 * g); };
      if constexpr (QT == TENSION_BF16) {
#pragma unroll
        for (int i = 0; i < G; ++i) q[i][0] = query_bf16(p.q, piece(i), whole);
      } else {
        float x[G][8];
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) x[i][j] = QT == TENSION_F16 ? (float)((const f16*)p.q.p)[piece(i) + j] : ((const float*)p.q.p)[piece(i) + j];
        if constexpr (QT == TENSION_F32) {
          // A bf16 ends at 2^-133: a row whose values are all small is brought up to 2^-16, and its scores down again.
          unsigned top = 0;
#pragma unroll
          for (int i = 0; i < G; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const unsigned b = magnitude_bits(x[i][j]);
              top = b > top ? b : top;
            }
#pragma unroll
          for (int m = 16; m < 64; m *= 2) {
            const unsigned o = (unsigned)__shfl_xor((int)top, m);
            top = o > top ? o : top;
          }
          const int turn = top >> 23 < 111 ? 111 - (int)(top >> 23) : 0;
          const float up = pow2_of_byte(127 + turn);
          scale *= pow2_of_byte(127 - turn);
#pragma unroll
          for (int i = 0; i < G; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] *= up;
        }
#pragma unroll
        for (int i = 0; i < G; ++i) query_terms<NQ>(x[i], q[i]);
      }
    }
    // one step is under way while another is added up, and the places of the next are looked up meanwhile
    for (; base + 2 * step < r.hi; base += 2 * step) {
      load(x1, w);
      w = look(base + 2 * step);
      add(x0, base);
      load(x0, w);
      w = look(base + 3 * step);
      add(x1, base + step);
    }
    if (base + step < r.hi) {
      load(x1, w);
      add(x0, base);
      add(x1, base + step);
    } else {
      add(x0, base);
    }
  }

  // acc[j]: rows = query heads 4g + i, column c = value c * VN + j, of a tail's two W + 2 c + j - VN
  mass += __shfl_xor(mass, 16);
  mass += __shfl_xor(mass, 32);
#pragma unroll
  for (int j = 0; j < VA; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[wave][4 * g + i][j < VN ? c * VN + j : W + 2 * c + j - VN] = acc[j][i];
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

template <int QT, int D>
void launch_as(const PagedDecodeParams& p, hipStream_t st) {
  const DecodeGrid grid(p, 16, 0);
  const unsigned n = grid.size(p);
  // eight waves where a CU has one workgroup
  if (n <= (unsigned)device_cus()) fp4_decode_mfma<QT, D, 8><<<n, 512, 0, st>>>(p, grid);
  else fp4_decode_mfma<QT, D, 4><<<n, 256, 0, st>>>(p, grid);
}

template <int D>
void launch_dim(const PagedDecodeParams& p, hipStream_t st) {
  if (p.q.dt == TENSION_F32) launch_as<TENSION_F32, D>(p, st);
  else if (p.q.dt == TENSION_F16) launch_as<TENSION_F16, D>(p, st);
  else launch_as<TENSION_BF16, D>(p, st);
}

}  // namespace

bool launch_fp4_mfma(const PagedDecodeParams& p, hipStream_t st) {
  if (p.D % 32 || p.D > 128 || p.c.S % kTileKeys || !DecodeGrid::fits(p)) return false;
  const unsigned piece = p.D == 96 ? 8 : p.D / 8;
  if (!row_pieces(p.c.k, piece) || !row_pieces(p.c.v, 4)) return false;
  // exponents of four rows of V are one load
  const uintptr_t at = (uintptr_t)p.c.ve | (uintptr_t)p.c.ve0 | (uintptr_t)p.c.ve1;
  if (p.c.ve2 != p.D / 32 || at % (p.D == 96 ? 4 : p.D / 8)) return false;
  if (p.D == 32) launch_dim<32>(p, st);
  else if (p.D == 64) launch_dim<64>(p, st);
  else if (p.D == 96) launch_dim<96>(p, st);
  else launch_dim<128>(p, st);
  return true;
}

}  // namespace tension
