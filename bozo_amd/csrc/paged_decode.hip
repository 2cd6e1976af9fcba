// One new token per sequence over its cached tokens in pages:
//   out = sum_s tau_s v_s / norm,  tau_s = sigmoid(q . k_s / scale),
// for the keys lo <= s < hi of each sequence.  Tau needs no running maximum,
// so the sums of disjoint key ranges simply add up: the axis is split over
// workgroups where there are few rows, and a second kernel adds the partial
// sums in order of the splits.
#include "paged.h"

namespace tension {

namespace {

// ------------------------------------------------------------------ any types, head dim <= 256, any page size

// Values ch, ch + 16, ... of a row as their bits, and as floats.
template <int VPL>
__device__ __forceinline__ void load_bits(const Buf& b, int64_t row, int ch, int D, unsigned* w) {
#pragma unroll
  for (int e = 0; e < VPL; ++e) w[e] = 0;
  auto go = [&](auto* s) {
#pragma unroll
    for (int e = 0; e < VPL; ++e)
      if (ch + 16 * e < D) w[e] = s[row + ch + 16 * e];
  };
  if (b.dt == TENSION_F32) go((const uint32_t*)b.p);
  else if (b.dt == TENSION_E4M3) go((const uint8_t*)b.p);
  else go((const uint16_t*)b.p);
}
template <int VPL>
__device__ __forceinline__ void bits_to_floats(int dt, const unsigned* w, float* x) {
#pragma unroll
  for (int e = 0; e < VPL; ++e) {
    if (dt == TENSION_F32) x[e] = __builtin_bit_cast(float, w[e]);
    else if (dt == TENSION_BF16) x[e] = __builtin_bit_cast(float, w[e] << 16);
    else if (dt == TENSION_F16) x[e] = (float)__builtin_bit_cast(f16, (unsigned short)w[e]);
    else x[e] = __builtin_amdgcn_cvt_f32_fp8((int)w[e], 0);
  }
}

// One workgroup per (n, h, split), sixteen lanes to a row, a value at a time:
// for rows that are no whole pieces of eight values, and pairs of types that
// have no kernel of their own.  Bound by its loads' number and latency (N16 H12,
// 1000 keys: bf16 D20 31 us, D100 150; D24 on the kernels for whole pieces 7.3).
template <int VPL, int kWaves>
__global__ void __launch_bounds__(64 * kWaves) paged_decode_any(PagedDecodeParams p) {
  constexpr int kRows = 4;
  __shared__ float red[kWaves][16 * VPL + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, ch = lane & 15;
  const int i = blockIdx.x % p.splits, nh = blockIdx.x / p.splits;
  const int n = nh / p.H, h = nh % p.H, hk = h / (p.H / p.Hk);
  const KeyRange all = key_range(p, p.lengths[n]), r = split_range(p, all, i);
  if (p.splits > 1 && i >= used_splits(p, all)) return;
  unsigned kw[VPL], vw[VPL];
  float q[VPL], acc[VPL], x[VPL], mass = 0.f;
  load_bits<VPL>(p.q, n * p.q.s0 + h * p.q.s1, ch, p.D, kw);
  bits_to_floats<VPL>(p.q.dt, kw, q);
#pragma unroll
  for (int e = 0; e < VPL; ++e) acc[e] = 0.f;
  for (int64_t base = (int64_t)r.lo + wave * kRows + (lane >> 4); base < r.hi; base += kWaves * kRows) {
    const int pos = (int)base, row = pos % p.c.S;
    const int page = p.c.table[(int64_t)n * p.c.table_stride + pos / p.c.S];
    if (page < 0 || page >= p.c.P) continue;  // the sixteen lanes of a row agree
    load_bits<VPL>(p.c.k, page * p.c.k.s0 + hk * p.c.k.s1 + row * p.c.k.s2, ch, p.D, kw);
    load_bits<VPL>(p.c.v, page * p.c.v.s0 + hk * p.c.v.s1 + row * p.c.v.s2, ch, p.D, vw);
    float s = 0.f, f = 1.f;
    if (p.c.ve) f = pow2_of_byte(p.c.ve[page * p.c.ve0 + hk * p.c.ve1 + row * p.c.ve2]);
    bits_to_floats<VPL>(p.c.k.dt, kw, x);
#pragma unroll
    for (int e = 0; e < VPL; ++e) s += q[e] * x[e];
    s += dpp_move<0xB1>(s);   // lane ^ 1
    s += dpp_move<0x4E>(s);   // lane ^ 2
    s += dpp_move<0x141>(s);  // mirrored halves of 8
    s += dpp_move<0x140>(s);  // mirrored rows of 16
    if (p.c.ke) s *= pow2_of_byte(p.c.ke[page * p.c.ke0 + hk * p.c.ke1 + row * p.c.ke2]);
    const float tau = sigmoid_exact(s / p.scale);
    mass += tau;
    bits_to_floats<VPL>(p.c.v.dt, vw, x);
#pragma unroll
    for (int e = 0; e < VPL; ++e) acc[e] += tau * f * x[e];
  }
#pragma unroll
  for (int e = 0; e < VPL; ++e) {
    acc[e] += __shfl_xor(acc[e], 16);
    acc[e] += __shfl_xor(acc[e], 32);
    if (lane < 16) red[wave][ch + 16 * e] = acc[e];
  }
  mass += __shfl_xor(mass, 16);
  mass += __shfl_xor(mass, 32);
  if (lane == 0) red[wave][16 * VPL] = mass;
  __syncthreads();
  if (tid >= p.D) return;
  float o = 0.f, m = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    o += red[w][tid];
    m += red[w][16 * VPL];
  }
  if (p.splits > 1) {
    split_sums(p, nh, i)[tid] = o;
    if (tid == 0) *split_mass(p, nh, i) = m;
  } else {
    st<float>(p.out, n * p.out.s0 + h * p.out.s1 + tid, o * norm_factor(p, m, all));
  }
}

// Partial sums of the splits of one (n, h): GROUPS of DP threads take every
// GROUPS-th split each, four loads under way at a time, and meet in LDS.  The
// order of the sums is fixed.
template <int DP, int GROUPS>
__global__ void __launch_bounds__(DP* GROUPS) paged_decode_join(PagedDecodeParams p) {
  __shared__ float red[GROUPS][DP], mred[DP * GROUPS / 64];
  const int nh = blockIdx.x, n = nh / p.H, h = nh % p.H, tid = threadIdx.x, d = tid % DP, g = tid / DP;
  const KeyRange all = key_range(p, p.lengths[n]);
  const int used = used_splits(p, all);
  float m = 0.f, acc = 0.f;
  const float* mass = split_mass(p, nh, 0);
  for (int i = tid; i < used; i += DP * GROUPS) m += mass[i];
  if (d < p.D) {
    const float* w = split_sums(p, nh, 0) + d;
    for (int i = g; i < used; i += 4 * GROUPS) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int s = i + j * GROUPS;
        x[j] = w[(int64_t)(s < used ? s : i) * p.D];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) acc += i + j * GROUPS < used ? x[j] : 0.f;
    }
  }
#pragma unroll
  for (int k = 32; k; k >>= 1) m += __shfl_xor(m, k);
  if ((tid & 63) == 0) mred[tid >> 6] = m;
  red[g][d] = acc;
  __syncthreads();
  if (tid >= p.D) return;
  m = 0.f;
  acc = 0.f;
#pragma unroll
  for (int i = 0; i < DP * GROUPS / 64; ++i) m += mred[i];
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) acc += red[i][tid];
  st<float>(p.out, n * p.out.s0 + h * p.out.s1 + tid, acc * norm_factor(p, m, all));
}

template <int DP>
void launch_join(const PagedDecodeParams& p, hipStream_t st) {
  if (p.splits > 1024 / DP)
    paged_decode_join<DP, 1024 / DP><<<(unsigned)(p.N * p.H), 1024, 0, st>>>(p);
  else
    paged_decode_join<DP, 256 / DP><<<(unsigned)(p.N * p.H), 256, 0, st>>>(p);
}

}  // namespace

// Splits of a sequence's keys.  A CU by itself streams 49 KB/us of cache, all
// of them 23 KB/us each; partial sums and the second kernel cost about 3 us on
// the card, 4 on the host (bf16 D64, us in one kernel / split: N1 H12 L512 5.5 /
// 7.2, L1024 9.2 / 7.1, L8192 47 / 10; N16 H12 L1000 10.1 / 12.3, L3000 25 / 28).
// Rows are counted as 16-bit ones whatever the pages' type: N1 H12 in one kernel
// / by this rule, 800 keys float32 9.8 / 9.8 (not split, though it would take
// about 8), 1200 keys e4m3 8.2 / 8.2, float32 13.9 / 8.3; 1700 e4m3 9.9 / 8.3.
// Tried: one split, and what gives each CU one to four workgroups (two where
// the matrix kernel holds head dim 128), with 128 keys to a split at least.
void paged_decode_split(int64_t N, int64_t H, int64_t Hk, int64_t D, int64_t keys, int* splits, int* chunk) {
  constexpr float kCuBytesPerUs = 49e3f, kAllBytesPerUs = 23e3f, kJoinUs = 3.5f;
  constexpr int64_t kLeast = 128, kMostGroups = ((int64_t)1 << 22) - 1;
  const int64_t rows = N * Hk, cus = device_cus();
  const float row_bytes = (float)keys * (float)(4 * D);
  const float all_us = (float)rows * row_bytes / (kAllBytesPerUs * (float)cus);
  const int fills = H > Hk && D > 64 ? 2 : 4;
  int64_t most = keys / kLeast;
  // workgroups of a launch, of 1024 threads at most
  if (N * H > 0 && most > kMostGroups / (N * H)) most = kMostGroups / (N * H);
  float best = 0.f;
  int64_t ns = 1;
  for (int f = 0; f <= fills; ++f) {
    int64_t s = f == 0 || rows <= 0 ? 1 : f * cus / rows;
    s = s < most ? s : most;
    if (f > 0 && s <= ns) continue;
    const float cu_us = (float)((rows * s + cus - 1) / cus) * row_bytes / (float)(s > 0 ? s : 1) / kCuBytesPerUs;
    const float t = (cu_us > all_us ? cu_us : all_us) + (f > 0 ? kJoinUs : 0.f);
    if (f == 0 || t < best) {
      best = t;
      ns = s;
    }
  }
  if (ns <= 1) {
    *splits = 1;
    *chunk = 0x40000000;
    return;
  }
  const int64_t c = ((keys + ns - 1) / ns + 31) / 32 * 32;
  *chunk = (int)c;
  *splits = (int)((keys + c - 1) / c);
}

int launch_paged_decode(const PagedDecodeParams& p, hipStream_t st, hipError_t* err) {
  if (!launch_paged_decode_rows(p, st)) {
    const unsigned grid = (unsigned)((int64_t)p.N * p.H * p.splits);
    if (p.D <= 64 && launchable(grid, 1024)) paged_decode_any<4, 16><<<grid, 1024, 0, st>>>(p);
    else if (p.D <= 64) paged_decode_any<4, 8><<<grid, 512, 0, st>>>(p);
    else paged_decode_any<16, 8><<<grid, 512, 0, st>>>(p);
  }
  *err = hipGetLastError();
  if (*err == hipSuccess && p.splits > 1) {
    if (p.D <= 64) launch_join<64>(p, st);
    else if (p.D <= 128) launch_join<128>(p, st);
    else launch_join<256>(p, st);
    *err = hipGetLastError();
  }
  return 0;
}

}  // namespace tension
