// Device helpers of the paged cache: division by the page size, exponent bytes,
// the keys of a sequence, how they are split over workgroups, and where the
// sums of a split go.
#pragma once

#include "kernels.h"

namespace tension {

// n / d for n < 2^31 as a multiplication (rounded-up reciprocal).
struct FastDiv {
  unsigned m;
  int s;
};
__device__ __forceinline__ int fdiv(int n, FastDiv d) { return (int)((__umulhi((unsigned)n, d.m) + (unsigned)n) >> d.s); }

// A launch counts its threads in 32 bits.
inline bool launchable(int64_t workgroups, int64_t threads) { return workgroups * threads <= 0xffffffffll; }

inline FastDiv fast_div(int64_t d) {
  int s = 0;
  while (((int64_t)1 << s) < d) ++s;
  return {(unsigned)(((uint64_t)1 << 32) * (((uint64_t)1 << s) - d) / d + 1), s};
}

// Whether every row of b starts at a multiple of `bytes`, a power of two (of
// which a wrapped product keeps the remainder).
inline bool row_pieces(const Buf& b, uint64_t bytes) {
  const uint64_t elt = b.dt == TENSION_E4M3 ? 1 : b.dt == TENSION_F32 ? 4 : 2;
  auto whole = [&](int64_t s) { return (uint64_t)s * elt % bytes == 0; };
  return (uintptr_t)b.p % bytes == 0 && whole(b.s0) && whole(b.s1) && whole(b.s2);
}

struct KeyRange {
  int lo, hi;
};

// Keys of a sequence; its length is held to what the table can name.
__device__ __forceinline__ KeyRange key_range(const PagedDecodeParams& p, int len) {
  const int cap = (int)(p.c.table_len > 0x7fffffff / p.c.S ? 0x7fffffff : p.c.table_len * p.c.S);
  len = len < 0 ? 0 : len > cap ? cap : len;
  const int hi = (p.flags & TENSION_DECODE_SELF) ? len : len - 1;
  const int lo = p.W > 0 && len - 1 > p.W ? len - 1 - p.W : 0;
  return {lo, hi > lo ? hi : lo};
}

// Splits of a sequence that hold keys.
__device__ __forceinline__ int used_splits(const PagedDecodeParams& p, KeyRange r) {
  const int n = (int)(((int64_t)r.hi - r.lo + p.chunk - 1) / p.chunk);
  return n < p.splits ? n : p.splits;
}

// Keys of split i (the last one takes what is left).
__device__ __forceinline__ KeyRange split_range(const PagedDecodeParams& p, KeyRange r, int i) {
  const int64_t a = r.lo + (int64_t)i * p.chunk;
  const int64_t b = i == p.splits - 1 ? r.hi : a + p.chunk;
  return {(int)(a < r.hi ? a : r.hi), (int)(b < r.hi ? b : r.hi)};
}

__device__ __forceinline__ float norm_factor(const PagedDecodeParams& p, float mass, KeyRange r) {
  if (p.flags & TENSION_NORM_MASS) return 1.f / (mass > kMassEps ? mass : kMassEps);
  if (p.flags & TENSION_NORM_COUNT) return 1.f / (float)(r.hi - r.lo > 1 ? r.hi - r.lo : 1);
  return 1.f;
}

// Partial sums [N * H, splits, D], then the masses [N * H, splits].
__device__ __forceinline__ float* split_sums(const PagedDecodeParams& p, int nh, int i) {
  return p.ws + ((int64_t)nh * p.splits + i) * p.D;
}
__device__ __forceinline__ float* split_mass(const PagedDecodeParams& p, int nh, int i) {
  return p.ws + (int64_t)p.N * p.H * p.splits * p.D + (int64_t)nh * p.splits + i;
}

// Scale of an exponent byte.
__device__ __forceinline__ float pow2_of_byte(int b) { return __builtin_bit_cast(float, (unsigned)b << 23); }

// The k-th longest of N <= 256 sequences, by four bits of their lengths and
// then by index: a wave counts how many share each longer prefix.
__device__ __forceinline__ int nth_longest(const int32_t* lengths, int N, int shift, int k, int* len) {
  constexpr int kMost = 4;
  const int lane = threadIdx.x & 63;
  int own[kMost], v[kMost];
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    const int i = 64 * j + lane;
    own[j] = lengths[i < N ? i : 0];
  }
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    const int x = own[j] >> shift;
    v[j] = 64 * j + lane < N ? (x < 0 ? 0 : x > 15 ? 15 : x) : -1;
  }
  int prefix = 0;
#pragma unroll
  for (int bit = 3; bit >= 0; --bit) {
    const int want = 2 * prefix + 1;
    int n = 0;
#pragma unroll
    for (int j = 0; j < kMost; ++j) n += __popcll(__ballot((v[j] >> bit) == want));
    const bool in = k < n;
    k -= in ? 0 : n;
    prefix = in ? want : 2 * prefix;
  }
  int found = 0, length = 0;
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    const uint64_t same = __ballot(v[j] == prefix);
    const int n = __popcll(same);
    const int before = __builtin_amdgcn_mbcnt_hi((unsigned)(same >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)same, 0));
    const uint64_t hit = __ballot(v[j] == prefix && before == k);
    const int at = (int)__builtin_ctzll(hit | (1ull << 63));
    const int l = __builtin_amdgcn_readlane(own[j], at);
    const bool here = k >= 0 && k < n;
    found = here ? 64 * j + at : found;
    length = here ? l : length;
    k -= n;
  }
  *len = __builtin_amdgcn_readfirstlane(length);
  return __builtin_amdgcn_readfirstlane(found);
}

// Workgroups of a decode call: (sequence, key head, group of query heads, split).
struct DecodeGrid {
  FastDiv page, dim, splits, heads, group_div, fill;
  int share, groups;  // query heads of a key head, and their groups
  int waves;          // of a workgroup
  int in_runs;        // workgroups taken in runs of eight on one XCD
  int turn;           // sequences that give each CU one workgroup; 0: sequences in their order
  int shift;
  // Element strides of pages and rows: a step's place is a few scalar
  // instructions, which a short step waits for as it does for its vector ones.
  uint32_t k0, k2, v0, v2, ke0, ke2, ve0, ve2;
  bool alike;  // values and their exponents lie as keys and theirs do

  // Whether the strides are ones that the kernels take.
  static bool fits(const PagedDecodeParams& p) {
    auto ok = [&](int64_t page, int64_t row) {
      return page >= 0 && page < ((int64_t)1 << 31) && row >= 0 && row < (1 << 24) && row * p.c.S < ((int64_t)1 << 31);
    };
    return ok(p.c.k.s0, p.c.k.s2) && ok(p.c.v.s0, p.c.v.s2) && ok(p.c.ke0, p.c.ke2) && ok(p.c.ve0, p.c.ve2);
  }
  DecodeGrid(const PagedDecodeParams& p, int per_group, int waves_) : waves(waves_) {
    share = p.H / p.Hk;
    groups = (share + per_group - 1) / per_group;
    page = fast_div(p.c.S);
    dim = fast_div(p.D);
    splits = fast_div(p.splits);
    heads = fast_div(p.Hk);
    group_div = fast_div(groups);
    k0 = (uint32_t)p.c.k.s0, k2 = (uint32_t)p.c.k.s2, v0 = (uint32_t)p.c.v.s0, v2 = (uint32_t)p.c.v.s2;
    ke0 = (uint32_t)p.c.ke0, ke2 = (uint32_t)p.c.ke2, ve0 = (uint32_t)p.c.ve0, ve2 = (uint32_t)p.c.ve2;
    // Key heads side by side share lines of exponent bytes (16 a head at S = 16): one XCD's L2 fetches them once
    // (e4m3, N128 H16: W256 17.5 -> 16.2 us, 2000 ragged tokens 62.4 -> 60.5; other pages: the same either way).
    // Where CUs take several workgroups of whole sequences the longest go first, and the next fill of the CUs in
    // reverse, so that each gets its share.  Finding them stands before every load, so only for calls that may read 100
    // MB, e4m3 rows counted as they are and others as 16-bit ones (us, in the sequences' order / so: ragged N128 H16 L2000
    // e4m3 60.4 / 55.9, N32 L4096 float32 114 / 106, N128 L4096 bf16 209.6 / 204; all of one length, N64 H12 L1000 bf16,
    // 32.3 / 32.8).
    const int64_t cus = device_cus(), per = (int64_t)p.Hk * groups * p.splits;
    const float bytes = (float)p.N * (float)p.Hk * (float)p.most * (float)(p.D * (p.c.ke ? 2 : 4));
    turn = p.W == 0 && p.N > 1 && p.N <= 256 && p.N * per > cus && bytes > 100e6f ? (int)((cus + per - 1) / per) : 0;
    fill = fast_div(turn > 0 ? turn : 1);
    shift = 0;
    while ((p.most >> shift) > 15) ++shift;
    in_runs = p.c.ke ? (int)(size(p) / 64 * 64) : 0;
    alike = k0 == v0 && k2 == v2 && ke0 == ve0 && ke2 == ve2;
  }
  // Elements from the first page's first row to this one's, of a head.
  struct Place {
    uint64_t k, v, ke, ve;
  };
  template <bool EXP, bool ALIKE>
  __device__ __forceinline__ Place at(int id, int row) const {
    auto off = [&](uint32_t s0, uint32_t s2) { return (uint64_t)(uint32_t)id * s0 + (uint32_t)row * s2; };
    Place w{};
    w.k = off(k0, k2);
    if constexpr (EXP) w.ke = off(ke0, ke2);
    w.v = w.k;
    w.ve = w.ke;
    if (!ALIKE && !alike) {
      w.v = off(v0, v2);
      if constexpr (EXP) w.ve = off(ve0, ve2);
    }
    return w;
  }
  unsigned size(const PagedDecodeParams& p) const { return (unsigned)((int64_t)p.N * p.Hk * groups * p.splits); }
  __device__ __forceinline__ void place(int b, const PagedDecodeParams& p, int* n, int* len, int* hk, int* grp, int* split) const {
    if (b < in_runs) b = b - b % 64 + b % 8 * 8 + b % 64 / 8;
    int x = fdiv(b, splits);
    *split = b - x * p.splits;
    int y = fdiv(x, group_div);
    *grp = x - y * groups;
    const int z = fdiv(y, heads);
    *hk = y - z * p.Hk;
    if (turn) {
      const int f = fdiv(z, fill), a = f * turn, e = a + turn < p.N ? a + turn : p.N;
      *n = nth_longest(p.lengths, p.N, shift, f & 1 ? e - 1 - (z - a) : z, len);
    } else {
      *n = z;
      *len = p.lengths[z];
    }
  }
};

// Kernels for whole 16-byte pieces of a row.  False when the call has no such
// form; the caller then runs the kernel for any.
bool launch_paged_decode_rows(const PagedDecodeParams& p, hipStream_t st);
bool launch_paged_decode_mfma(const PagedDecodeParams& p, hipStream_t st);

}  // namespace tension
