// Paged decode on the vector units: one workgroup streams the keys of one
// (sequence, key head, split) for up to G query heads.
//
// tau_s = 1 / (1 + 2^(q . k_s)) with q scaled once by -log2(e) / scale, sums of
// tau and tau v in float32: one pass over K and V, no running maximum.  LPR
// lanes cover a row with VPL values each, so a wave takes RPW = 64 / LPR rows
// in one load of K and one of V, and a dot product is VPL multiplications and a
// lane sum.  Where a page holds whole steps of RPW rows (ALIGNED) a step lies
// in one page: its place is wave-uniform, the table is read through scalar
// loads and a lane's address is a constant offset from a scalar base.
// Otherwise each lane looks its row's page up.
//
// Bound by HBM where the caches are large (bf16 D64, N128 H16 to 4096 ragged
// tokens, 1.34 GB: 204 us, 6.6 TB/s; e4m3, 0.68 GB: 109 us, 6.3 TB/s), by
// latency where they are small (N1 H12, 200 keys: 4.2 us, of which an empty
// sequence takes 3.3).  Loads under way are what counts: a batch of two steps
// ahead of the one being added up (four: no faster); eight codes of e4m3 to a
// lane instead of sixteen halve them and cost 30%.
#pragma once

#include <type_traits>

#include "paged.h"

namespace tension {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int page_elt(int dt) { return dt == TENSION_F32 ? 4 : dt == TENSION_E4M3 ? 1 : 2; }

// One lane's values of a row: VPL of LPR * VPL, in 16-byte pieces (8-byte for
// eight codes).  float32 pieces lie LPR * 4 values apart, so that a load of
// the wave covers whole lines.
template <int DT, int VPL, int LPR>
struct Piece {
  static constexpr int kLoads = DT == TENSION_F32 ? VPL / 4 : 1;
  static constexpr bool kShort = VPL * page_elt(DT) == 8;
  using Raw = typename std::conditional<kShort, u32x2, u32x4>::type;
  Raw a[kLoads];

  // Value e of lane ch is value feat(ch, e) of its row.
  static __device__ __forceinline__ int feat(int ch, int e) {
    return DT == TENSION_F32 ? (e / 4) * (4 * LPR) + 4 * ch + e % 4 : ch * VPL + e;
  }
  // Pieces past the head dim read the row's first again; past() zeroes them.
  static __device__ __forceinline__ unsigned piece_off(int ch, int i, int D) {
    const int f = feat(ch, 4 * i);
    return (unsigned)((f < D ? f : 0) * page_elt(DT));
  }
  __device__ __forceinline__ void load(const char* base, const unsigned* off) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) a[i] = __builtin_nontemporal_load((const Raw*)(base + off[i]));
  }
  __device__ __forceinline__ void past(int ch, int D) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const bool in = feat(ch, 4 * i) < D;
#pragma unroll
      for (int j = 0; j < (kShort ? 2 : 4); ++j) a[i][j] = in ? a[i][j] : 0u;
    }
  }
  __device__ __forceinline__ void zero_unless(bool keep) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int j = 0; j < (kShort ? 2 : 4); ++j) a[i][j] = keep ? a[i][j] : 0u;
  }
  __device__ __forceinline__ void floats(float* x) const {
    if constexpr (DT == TENSION_F32) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const unsigned w = a[i / 4][i % 4];
        x[i] = __builtin_bit_cast(float, w);
      }
    } else if constexpr (DT == TENSION_F16) {
      const f16x8 h = __builtin_bit_cast(f16x8, a[0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
    } else if constexpr (DT == TENSION_BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned w = a[0][i];
        x[2 * i] = __builtin_bit_cast(float, w << 16);
        x[2 * i + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VPL / 4; ++i) {
        const int w = (int)a[0][i];
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        x[4 * i] = lo[0];
        x[4 * i + 1] = lo[1];
        x[4 * i + 2] = hi[0];
        x[4 * i + 3] = hi[1];
      }
    }
  }
};

// Sum over an aligned group of LPR lanes, on each of them.
template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
  if constexpr (LPR >= 2) x += dpp_move<0xB1>(x);    // lane ^ 1
  if constexpr (LPR >= 4) x += dpp_move<0x4E>(x);    // lane ^ 2
  if constexpr (LPR >= 8) x += dpp_move<0x141>(x);   // mirrored halves of 8
  if constexpr (LPR >= 16) x += dpp_move<0x140>(x);  // mirrored rows of 16
  if constexpr (LPR >= 32) x += __shfl_xor(x, 16);
  return x;
}

// Sums over the lanes with the same lane % LPR of a lane's N values x: halves
// of the wave trade one value of a pair for the other and add, then rows of 16
// do, so that value kept(lane, j) ends up in x[j], j < N / kParts, of the lanes
// that write().  Half the adds of a butterfly and no trip through LDS: N128 H16
// W64 e4m3 12.8 -> 10.6 us.
template <int LPR, int N>
struct Fold {
  static constexpr int kParts = LPR == 32 ? 2 : 4;
  static __device__ __forceinline__ int kept(int lane, int j) {
    return LPR == 32 ? 2 * j + lane / 32 : 4 * j + 2 * (lane / 16 % 2) + lane / 32;
  }
  static __device__ __forceinline__ bool write(int lane) { return LPR >= 16 || lane % 16 < LPR; }
  static __device__ __forceinline__ float in_row(float x) {
    if constexpr (LPR <= 8) x += dpp_move<0x128>(x);  // lane - 8 of its row
    if constexpr (LPR <= 4) x += dpp_move<0x124>(x);  // lane - 4
    return x;
  }
  static __device__ __forceinline__ float add_halves(float a, float b) {
    const auto w = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned lo = w[0], hi = w[1];
    return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
  }
  static __device__ __forceinline__ float add_rows(float a, float b) {
    const auto w = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned lo = w[0], hi = w[1];
    return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
  }
  static __device__ __forceinline__ void run(float* x) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) x[i] = add_halves(x[2 * i], x[2 * i + 1]);
    if constexpr (LPR < 32) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) x[i] = in_row(add_rows(x[2 * i], x[2 * i + 1]));
    }
  }
  // Of one value, on every lane.
  static __device__ __forceinline__ float sum(float x) {
    x = add_halves(x, x);
    if constexpr (LPR < 32) x = in_row(add_rows(x, x));
    return x;
  }
};

// The lane's values of G query rows, in the order of its K values.
template <int KD, int VPL, int LPR, int G>
struct Query {
  u32x4 a[G][VPL / 4];  // four values: float32, or 16-bit ones in the first half

  __device__ __forceinline__ void load(const PagedDecodeParams& p, int n, int h0, int nh, int ch) {
    const int elt = p.q.dt == TENSION_F32 ? 4 : 2;
    const bool whole = ((uintptr_t)p.q.p | (uintptr_t)(p.q.s0 * elt) | (uintptr_t)(p.q.s1 * elt)) % (4 * elt) == 0;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const char* row = (const char*)p.q.p + ((int64_t)n * p.q.s0 + (int64_t)(h0 + (g < nh ? g : 0)) * p.q.s1) * elt;
#pragma unroll
      for (int i = 0; i < VPL / 4; ++i) {
        const int f = Piece<KD, VPL, LPR>::feat(ch, 4 * i);
        const char* s = row + (f < p.D ? f : 0) * elt;
        if (whole && elt == 4) {
          a[g][i] = *(const u32x4*)s;
        } else if (whole) {
          const u32x2 w = *(const u32x2*)s;
          a[g][i][0] = w[0];
          a[g][i][1] = w[1];
        } else if (elt == 4) {
#pragma unroll
          for (int j = 0; j < 4; ++j) a[g][i][j] = ((const unsigned*)s)[j];
        } else {
          const unsigned short* x = (const unsigned short*)s;
          a[g][i][0] = x[0] | (unsigned)x[1] << 16;
          a[g][i][1] = x[2] | (unsigned)x[3] << 16;
        }
      }
    }
  }
  // Scaled so that tau = 1 / (1 + 2^(q . k)).
  __device__ __forceinline__ void floats(const PagedDecodeParams& p, int ch, float (*q)[VPL]) const {
    const float scale = -p.inv_scale * kLog2e;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < VPL / 4; ++i) {
        const bool in = Piece<KD, VPL, LPR>::feat(ch, 4 * i) < p.D;
        float x[4];
        if (p.q.dt == TENSION_F32) {
          const f32x4 w = __builtin_bit_cast(f32x4, a[g][i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = w[j];
        } else {
          const u32x2 w = {a[g][i][0], a[g][i][1]};
          const f16x4 h = __builtin_bit_cast(f16x4, w);
          const bf16x4 b = __builtin_bit_cast(bf16x4, w);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = p.q.dt == TENSION_F16 ? (float)h[j] : (float)b[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) q[g][4 * i + j] = in ? x[j] * scale : 0.f;
      }
  }
};

// PLAIN: the head dim fills a row's lanes, and values and their exponents lie as
// keys and theirs do.
template <int KD, int VD, int VPL, int LPR, int G, int U, bool ALIGNED, bool PLAIN>
__global__ void __launch_bounds__(512) paged_decode_rows(PagedDecodeParams p, DecodeGrid grid) {
  constexpr int RPW = 64 / LPR;
  constexpr bool KE = KD == TENSION_E4M3, VE = VD == TENSION_E4M3;
  using PK = Piece<KD, VPL, LPR>;
  using PV = Piece<VD, VPL, LPR>;
  extern __shared__ float red[];  // [waves][G][D + 1]
  const int tid = threadIdx.x, lane = tid & 63, ch = lane % LPR, lr = lane / LPR;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = grid.waves;
  int n, len, hk, grp, split;
  grid.place((int)blockIdx.x, p, &n, &len, &hk, &grp, &split);
  const int h0 = hk * grid.share + grp * G, nh = grid.share - grp * G < G ? grid.share - grp * G : G;
  const KeyRange all = key_range(p, len);
  KeyRange r = split_range(p, all, split);

  float q[G][VPL], acc[G][VPL], mass[G];
  Query<KD, VPL, LPR, G> qraw;
  qraw.load(p, n, h0, nh, ch);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    mass[g] = 0.f;
#pragma unroll
    for (int e = 0; e < VPL; ++e) acc[g][e] = 0.f;
  }

  const char* kbase = (const char*)p.c.k.p + (int64_t)hk * p.c.k.s1 * page_elt(KD);
  const char* vbase = (const char*)p.c.v.p + (int64_t)hk * p.c.v.s1 * page_elt(VD);
  const uint8_t* kebase = p.c.ke + (KE ? (int64_t)hk * p.c.ke1 : 0);
  const uint8_t* vebase = p.c.ve + (VE ? (int64_t)hk * p.c.ve1 : 0);
  const int32_t* table = p.c.table + (int64_t)n * p.c.table_stride;
  unsigned koff[PK::kLoads], voff[PV::kLoads];
#pragma unroll
  for (int i = 0; i < PK::kLoads; ++i)
    koff[i] = PK::piece_off(ch, i, p.D) + (ALIGNED ? (unsigned)(lr * p.c.k.s2) * page_elt(KD) : 0u);
#pragma unroll
  for (int i = 0; i < PV::kLoads; ++i)
    voff[i] = PV::piece_off(ch, i, p.D) + (ALIGNED ? (unsigned)(lr * p.c.v.s2) * page_elt(VD) : 0u);
  const unsigned keoff = ALIGNED ? (unsigned)(lr * p.c.ke2) : 0u, veoff = ALIGNED ? (unsigned)(lr * p.c.ve2) : 0u;

  // U steps of a wave, their loads ahead of their use: one batch is under way
  // while the one before it is added up, and the places of the next are looked
  // up meanwhile.
  struct Places {
    int id[U], row[U];
    bool ok[U];  // of this lane's row
  };
  struct Batch {
    PK k[U];
    PV v[U];
    int ke[U], ve[U];
    bool ok[U];
  };
  auto look = [&](int64_t base) {
    Places w;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned pos = (unsigned)base + u * RPW + (ALIGNED ? 0 : lr), hi = (unsigned)r.hi;
      const int at = pos < hi ? (int)pos : r.hi - 1;
      const int slot = fdiv(at, grid.page);
      const int id = table[slot];
      w.ok[u] = id >= 0 && id < p.c.P;
      w.id[u] = w.ok[u] ? id : 0;
      w.row[u] = at - slot * p.c.S;
      if (ALIGNED) {
        w.row[u] = pos < hi ? w.row[u] : 0;  // a whole step past the end reads its page's first
        w.ok[u] = w.ok[u] && pos + lr >= (unsigned)r.lo && pos + lr < hi;
      } else {
        w.ok[u] = w.ok[u] && pos < hi;
      }
    }
    return w;
  };
  auto load = [&](Batch& t, const Places& w) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      t.ok[u] = w.ok[u];
      const DecodeGrid::Place at = grid.at<KE, PLAIN>(w.id[u], w.row[u]);
      t.k[u].load(kbase + at.k * page_elt(KD), koff);
      if constexpr (KE) t.ke[u] = (kebase + at.ke)[keoff];
      t.v[u].load(vbase + at.v * page_elt(VD), voff);
      if constexpr (VE) t.ve[u] = (vebase + at.ve)[veoff];
    }
  };
  auto add = [&](Batch& t) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // rows out of range or without a page hold anything (a branch that most steps would skip costs more)
      t.v[u].zero_unless(t.ok[u]);
      if constexpr (VE) t.ve[u] = t.ok[u] ? t.ve[u] : 0;
      if (!PLAIN && p.D < LPR * VPL) t.k[u].past(ch, p.D);  // an infinite key times a query's zeros is no number
      float x[VPL], tau[G];
      t.k[u].floats(x);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < VPL; ++e) s += q[g][e] * x[e];
        s = row_sum<LPR>(s);
        if constexpr (KE) s *= pow2_of_byte(t.ke[u]);
        tau[g] = t.ok[u] ? __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s)) : 0.f;
        mass[g] += tau[g];
        if constexpr (VE) tau[g] *= pow2_of_byte(t.ve[u]);
      }
      t.v[u].floats(x);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < VPL; ++e) acc[g][e] += tau[g] * x[e];
    }
  };
  const int64_t step = (int64_t)waves * RPW * U;
  int64_t base = (ALIGNED ? r.lo / RPW * RPW : r.lo) + (int64_t)wave * RPW * U;
  if (base < r.hi) {
    Batch t0, t1;
    load(t0, look(base));
    Places w = look(base + step);
    qraw.floats(p, ch, q);
    for (; base + 2 * step < r.hi; base += 2 * step) {
      load(t1, w);
      w = look(base + 2 * step);
      add(t0);
      load(t0, w);
      w = look(base + 3 * step);
      add(t1);
    }
    if (base + step < r.hi) {
      load(t1, w);
      add(t0);
      add(t1);
    } else {
      add(t0);
    }
  }

  // rows of a wave, then the waves
  const int D = p.D;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    using F = Fold<LPR, VPL>;
    mass[g] = F::sum(mass[g]);
    F::run(acc[g]);
    float* o = red + (wave * G + g) * (D + 1);
    if (F::write(lane)) {
#pragma unroll
      for (int j = 0; j < VPL / F::kParts; ++j) {
        const int f = PV::feat(ch, F::kept(lane, j));
        if (f < D) o[f] = acc[g][j];
      }
    }
    if (lane == 0) o[D] = mass[g];
  }
  if (p.splits > 1 && split >= used_splits(p, all)) return;  // no keys, nobody waits for it
  __syncthreads();
  for (int i = tid; i < nh * D; i += 64 * waves) {
    const int g = fdiv(i, grid.dim), d = i - g * D;
    float o = 0.f, m = 0.f;
    for (int w = 0; w < waves; ++w) {
      o += red[(w * G + g) * (D + 1) + d];
      m += red[(w * G + g) * (D + 1) + D];
    }
    const int row = n * p.H + h0 + g;
    if (p.splits > 1) {
      split_sums(p, row, split)[d] = o;
      if (d == 0) *split_mass(p, row, split) = m;
    } else {
      st<float>(p.out, (int64_t)n * p.out.s0 + (int64_t)(h0 + g) * p.out.s1 + d, o * norm_factor(p, m, all));
    }
  }
}

template <int KD, int VD, int VPL, int LPR, int G, bool ALIGNED>
void launch_rows_as(const PagedDecodeParams& p, int waves, hipStream_t st) {
  constexpr bool kOne = ALIGNED && G == 1;
  constexpr int U = kOne ? 2 : 1;
  const DecodeGrid grid(p, G, waves);
  const unsigned n = grid.size(p), threads = 64 * waves, lds = waves * G * (p.D + 1) * sizeof(float);
  if constexpr (kOne) {
    if (p.D == LPR * VPL && grid.alike) {  // what the other form checks costs 5% and more of an e4m3 stream
      paged_decode_rows<KD, VD, VPL, LPR, G, U, ALIGNED, true><<<n, threads, lds, st>>>(p, grid);
      return;
    }
  }
  paged_decode_rows<KD, VD, VPL, LPR, G, U, ALIGNED, false><<<n, threads, lds, st>>>(p, grid);
}

// Rows of pieces for this type, head dim, page size: the lanes of a row, the
// query heads of a workgroup.
template <int KD, int VD, int VPL>
bool launch_rows(const PagedDecodeParams& p, int waves, hipStream_t st) {
  const int share = p.H / p.Hk;
  auto go = [&](auto lanes) {
    constexpr int LPR = decltype(lanes)::value;
    if (p.c.S % (64 / LPR)) launch_rows_as<KD, VD, VPL, LPR, 1, false>(p, waves, st);
    else if (share == 1) launch_rows_as<KD, VD, VPL, LPR, 1, true>(p, waves, st);
    else if (share == 2) launch_rows_as<KD, VD, VPL, LPR, 2, true>(p, waves, st);
    else if constexpr (VPL == 8) launch_rows_as<KD, VD, VPL, LPR, 4, true>(p, waves, st);
    return true;
  };
  const int pieces = (p.D + VPL - 1) / VPL;
  if (pieces <= 4) return go(std::integral_constant<int, 4>{});
  if (pieces <= 8) return go(std::integral_constant<int, 8>{});
  if (pieces <= 16) return go(std::integral_constant<int, 16>{});
  if constexpr (VPL == 8)
    if (pieces <= 32) return go(std::integral_constant<int, 32>{});
  return false;
}

}  // namespace tension
