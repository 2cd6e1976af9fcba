// One new token per sequence over its cached tokens in pages:
//   out = sum_s tau_s v_s / norm,  tau_s = sigmoid(q . k_s / scale),
// for the keys lo <= s < hi of each sequence.  Tau needs no running maximum,
// so the sums of disjoint key ranges simply add up: the axis is split over
// workgroups where there are few rows, and a second kernel adds the partial
// sums in order of the splits.
#include "paged.h"

namespace tension {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float ld_page(const Buf& b, int64_t off) {
  return b.dt == TENSION_E4M3 ? __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)b.p)[off], 0) : ld<float>(b, off);
}

// ------------------------------------------------------------------ any types, head dim <= 256, any page size

// One workgroup per (n, h, split): a thread forms the tau of one key, then
// threads along the head dim add the value rows.
__global__ void __launch_bounds__(kThreads) paged_decode_any(PagedDecodeParams p) {
  __shared__ float qs[256], tau[kThreads], red[kThreads / 64];
  __shared__ int64_t voff[kThreads];
  const int tid = threadIdx.x;
  const int i = blockIdx.x % p.splits, nh = blockIdx.x / p.splits;
  const int n = nh / p.H, h = nh % p.H, hk = h / (p.H / p.Hk);
  const KeyRange all = key_range(p, n), r = split_range(p, all, i);
  if (p.splits > 1 && i >= used_splits(p, all)) return;
  for (int d = tid; d < p.D; d += kThreads) qs[d] = ld<float>(p.q, n * p.q.s0 + h * p.q.s1 + d);
  __syncthreads();
  float acc = 0.f, mass = 0.f;
  for (int base = r.lo; base < r.hi; base += kThreads) {
    const int m = r.hi - base < kThreads ? r.hi - base : kThreads;
    float w = 0.f;
    int64_t vo = -1;
    if (tid < m) {
      const int pos = base + tid, row = pos % p.c.S;
      const int page = p.c.table[(int64_t)n * p.c.table_stride + pos / p.c.S];
      if (page >= 0 && page < p.c.P) {
        const int64_t ko = page * p.c.k.s0 + hk * p.c.k.s1 + row * p.c.k.s2;
        float s = 0.f;
        for (int d = 0; d < p.D; ++d) s += qs[d] * ld_page(p.c.k, ko + d);
        if (p.c.ke) s *= pow2_of_byte(p.c.ke[page * p.c.ke0 + hk * p.c.ke1 + row * p.c.ke2]);
        w = sigmoid_exact(s / p.scale);
        mass += w;
        if (p.c.ve) w *= pow2_of_byte(p.c.ve[page * p.c.ve0 + hk * p.c.ve1 + row * p.c.ve2]);
        vo = page * p.c.v.s0 + hk * p.c.v.s1 + row * p.c.v.s2;
      }
    }
    tau[tid] = w;
    voff[tid] = vo;
    __syncthreads();
    if (tid < p.D)
      for (int j = 0; j < m; ++j)
        if (voff[j] >= 0) acc += tau[j] * ld_page(p.c.v, voff[j] + tid);
    __syncthreads();
  }
#pragma unroll
  for (int m = 32; m; m >>= 1) mass += __shfl_xor(mass, m);
  if ((tid & 63) == 0) red[tid >> 6] = mass;
  __syncthreads();
  mass = red[0] + red[1] + red[2] + red[3];
  if (p.splits > 1) {
    if (tid < p.D) split_sums(p, nh, i)[tid] = acc;
    if (tid == 0) *split_mass(p, nh, i) = mass;
  } else if (tid < p.D) {
    st<float>(p.out, n * p.out.s0 + h * p.out.s1 + tid, acc * norm_factor(p, mass, all));
  }
}

// Partial sums of the splits of one (n, h): GROUPS of DP threads take every
// GROUPS-th split each, four loads under way at a time, and meet in LDS.  The
// order of the sums is fixed.
template <int DP, int GROUPS>
__global__ void __launch_bounds__(DP* GROUPS) paged_decode_join(PagedDecodeParams p) {
  __shared__ float red[GROUPS][DP], mred[DP * GROUPS / 64];
  const int nh = blockIdx.x, n = nh / p.H, h = nh % p.H, tid = threadIdx.x, d = tid % DP, g = tid / DP;
  const KeyRange all = key_range(p, n);
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
// of them 23 KB/us each; partial sums and the second kernel cost about 3 us
// (bf16 D64, us for 1 / 21 splits: N1 H12 L512 6.3 / 7.2, L1024 9.2 / 7.3, L8192
// 47 / 10; N16 H12, 1 / 5: L1000 10.2 / 12.3, L3000 25 / 28).  Tried: one split,
// and what gives each CU one to four workgroups (two where the matrix kernel
// holds head dim 128), with 128 keys to a split at least.
void paged_decode_split(int64_t N, int64_t H, int64_t Hk, int64_t D, int64_t keys, int* splits, int* chunk) {
  constexpr float kCuBytesPerUs = 49e3f, kAllBytesPerUs = 23e3f, kJoinUs = 3.f;
  constexpr int64_t kLeast = 128;
  const int64_t rows = N * Hk, cus = device_cus();
  const float row_bytes = (float)keys * (float)(4 * D);
  const float all_us = (float)rows * row_bytes / (kAllBytesPerUs * (float)cus);
  const int fills = H > Hk && D > 64 ? 2 : 4;
  float best = 0.f;
  int64_t ns = 1;
  for (int f = 0; f <= fills; ++f) {
    int64_t s = f == 0 || rows <= 0 ? 1 : f * cus / rows;
    s = s < keys / kLeast ? s : keys / kLeast;
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
  if (!launch_paged_decode_rows(p, st))
    paged_decode_any<<<(unsigned)((int64_t)p.N * p.H * p.splits), kThreads, 0, st>>>(p);
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
