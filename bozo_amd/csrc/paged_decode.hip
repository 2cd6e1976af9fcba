// One new token per sequence over its cached tokens in pages:
//   out = sum_s tau_s v_s / norm,  tau_s = sigmoid(q . k_s / scale),
// for the keys lo <= s < hi of each sequence.  Tau needs no running maximum,
// so the sums of disjoint key ranges simply add up: the axis is split over
// workgroups where there are few rows, and a second kernel adds the partial
// sums in order of the splits.
#include "kernels.h"

namespace tension {

namespace {

constexpr int kThreads = 256;

struct KeyRange {
  int lo, hi;
};

// Keys of sequence n; the length is held to what the table can name.
__device__ __forceinline__ KeyRange key_range(const PagedDecodeParams& p, int n) {
  const int cap = (int)(p.c.table_len > 0x7fffffff / p.c.S ? 0x7fffffff : p.c.table_len * p.c.S);
  int len = p.lengths[n];
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
        if (p.c.ke) s *= __builtin_bit_cast(float, (unsigned)p.c.ke[page * p.c.ke0 + hk * p.c.ke1 + row * p.c.ke2] << 23);
        w = sigmoid_exact(s / p.scale);
        mass += w;
        if (p.c.ve) w *= __builtin_bit_cast(float, (unsigned)p.c.ve[page * p.c.ve0 + hk * p.c.ve1 + row * p.c.ve2] << 23);
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
    float* w = p.ws + ((int64_t)nh * p.splits + i) * (p.D + 1);
    if (tid < p.D) w[tid] = acc;
    if (tid == 0) w[p.D] = mass;
  } else if (tid < p.D) {
    st<float>(p.out, n * p.out.s0 + h * p.out.s1 + tid, acc * norm_factor(p, mass, all));
  }
}

// Partial sums of the splits of one (n, h), added in their order.
__global__ void __launch_bounds__(kThreads) paged_decode_join(PagedDecodeParams p) {
  const int nh = blockIdx.x, n = nh / p.H, h = nh % p.H;
  const KeyRange all = key_range(p, n);
  const int used = used_splits(p, all);
  const float* w = p.ws + (int64_t)nh * p.splits * (p.D + 1);
  float mass = 0.f;
  for (int i = 0; i < used; ++i) mass += w[(int64_t)i * (p.D + 1) + p.D];
  const float f = norm_factor(p, mass, all);
  for (int d = threadIdx.x; d < p.D; d += kThreads) {
    float acc = 0.f;
    for (int i = 0; i < used; ++i) acc += w[(int64_t)i * (p.D + 1) + d];
    st<float>(p.out, n * p.out.s0 + h * p.out.s1 + d, acc * f);
  }
}

}  // namespace

// About four workgroups per CU, splits of 256 keys at least.
void paged_decode_split(int64_t N, int64_t H, int64_t Hk, int64_t D, int64_t W, int64_t max_len, int* splits, int* chunk) {
  const int64_t keys = W > 0 && W + 1 < max_len ? W + 1 : max_len;
  const int64_t rows = N * H;
  int64_t ns = (1024 + rows - 1) / (rows > 0 ? rows : 1);
  const int64_t most = (keys + 255) / 256;
  ns = ns > most ? most : ns;
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
  paged_decode_any<<<(unsigned)((int64_t)p.N * p.H * p.splits), kThreads, 0, st>>>(p);
  *err = hipGetLastError();
  if (*err == hipSuccess && p.splits > 1) {
    paged_decode_join<<<(unsigned)(p.N * p.H), kThreads, 0, st>>>(p);
    *err = hipGetLastError();
  }
  return 0;
}

}  // namespace tension
