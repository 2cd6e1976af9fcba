// The best continuations of a group's beams over the vocabulary:
//   score(b, v) = scores[b] + x[b, v] - log sum_u exp x[b, u],
// the K largest of a group; of equal ones the lower beam's, within a beam the
// larger logit, then the lower token.
//
// Exponentials, sum and logarithm are taken in 64 bits, since they decide between
// beams.  Within a beam the logits' own order is the scores', also where scores
// round to one, so a beam's candidates are found by comparing what was stored, and
// only they get a score.
#include <float.h>

#include "paged.h"

namespace tension {

namespace {

constexpr int kThreads = 256, kSpan = 8192;
constexpr double kLog2e64 = 1.4426950408889634074;

// A candidate's place in its beam's order as one number: larger logits first,
// then lower indexes; 0 below every candidate.
__device__ __forceinline__ uint64_t order_key(float x, unsigned v) {
  const unsigned b = __builtin_bit_cast(unsigned, x == 0.f ? 0.f : x);  // -0 is 0
  const unsigned o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (uint64_t)o << 32 | (0xffffffffu - v);
}
__device__ __forceinline__ float key_logit(uint64_t k) {
  const unsigned o = (unsigned)(k >> 32);
  return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

__device__ __forceinline__ uint64_t shfl64(uint64_t x, int from) {
  const unsigned lo = (unsigned)__shfl((int)(unsigned)x, from), hi = (unsigned)__shfl((int)(x >> 32), from);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t wave_most(uint64_t x) {
#pragma unroll
  for (int m = 32; m; m >>= 1) {
    const uint64_t o = shfl64(x, (threadIdx.x & 63) ^ m);
    x = o > x ? o : x;
  }
  return x;
}

constexpr int kPowers = 64;

// 2^(j / 64), for add_exp: made by each workgroup, 1 exactly at 0.
__device__ __forceinline__ void make_powers(double* powers) {
  if (threadIdx.x < kPowers) powers[threadIdx.x] = exp2((double)threadIdx.x / kPowers);
}

// s + exp(d) for d <= 0 in 64 bits; exp(0) is 1 exactly, so that a beam's only
// token adds nothing to its score (what is below 2^-1000 counts as that).  With u =
// 64 d log2 e = 64 k + j + f, |f| <= 1/2: 2^k 2^(j / 64) times 1 + f q(f), where q
// interpolates (2^(f / 64) - 1) / f at Chebyshev points (2^-58 relative, below the
// roundings).  Adding 1.5 * 2^52 rounds, and leaves 64 k + j in the low bits.
__device__ __forceinline__ double add_exp(double s, double d, const double* powers) {
  constexpr double kRound = 6755399441055744.;
  const double u = fmax(d * (kPowers * kLog2e64), -1000. * kPowers);
  const double t = u + kRound;
  const double f = u - (t - kRound);
  double p = 0.001333356978334557 / (64. * 64. * 64. * 64. * 64.);
  p = __builtin_fma(p, f, 0.009618140859595685 / (64. * 64. * 64. * 64.));
  p = __builtin_fma(p, f, 0.055504108664803826 / (64. * 64. * 64.));
  p = __builtin_fma(p, f, 0.2402265069589214 / (64. * 64.));
  p = __builtin_fma(p, f, 0.6931471805599453 / 64.);
  p = __builtin_fma(p, f, 1.);
  const int n = (int)(unsigned)__builtin_bit_cast(uint64_t, t);
  const uint64_t b = __builtin_bit_cast(uint64_t, powers[n & (kPowers - 1)]);
  return __builtin_fma(__builtin_bit_cast(double, b + ((uint64_t)(unsigned)(n >> 6) << 52)), p, s);
}

template <int CTRL>
__device__ __forceinline__ double dpp_move64(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)b, CTRL, 0xF, 0xF, true);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sum over the wave, on every lane.
__device__ __forceinline__ double wave_sum(double x) {
  x += dpp_move64<0xB1>(x);   // lane ^ 1
  x += dpp_move64<0x4E>(x);   // lane ^ 2
  x += dpp_move64<0x141>(x);  // mirrored halves of 8
  x += dpp_move64<0x140>(x);  // mirrored rows of 16
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}
// Largest over the wave, NaN if one is.
__device__ __forceinline__ float wave_max(float x) {
  x = __builtin_elementwise_maximum(x, dpp_move<0xB1>(x));
  x = __builtin_elementwise_maximum(x, dpp_move<0x4E>(x));
  x = __builtin_elementwise_maximum(x, dpp_move<0x141>(x));
  x = __builtin_elementwise_maximum(x, dpp_move<0x140>(x));
  x = __builtin_elementwise_maximum(x, __shfl_xor(x, 16));
  return __builtin_elementwise_maximum(x, __shfl_xor(x, 32));
}

// Floats in the order of whole numbers.
__device__ __forceinline__ unsigned order_bits(float x) {
  const unsigned b = __builtin_bit_cast(unsigned, x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Whether a beam's logits decide anything: it is one, and goes on.
__device__ __forceinline__ bool goes_on(const BeamParams& p, int n, int b) {
  const float score = p.scores[n * p.score0 + b * p.score1];
  const bool ended = p.ended && p.ended[n * p.ended0 + b * p.ended1];  // both loads at once
  return (score > -INFINITY) & (score < INFINITY) & !ended;
}

// The K-th largest of the lanes' order_bits, M each, as a float, bit by bit: M
// comparisons and counts of lanes each.  (Zeros of both signs compare as one with it.)
template <int M>
__device__ __forceinline__ float kth_of_wave(const unsigned (&g)[M], int K) {
  unsigned bound = 0;
#pragma unroll
  for (int bit = 31; bit >= 0; --bit) {
    const unsigned at = bound | 1u << bit;
    int reach = 0;
#pragma unroll
    for (int m = 0; m < M; ++m) reach += __popcll(__ballot(g[m] >= at));
    bound = reach >= K ? at : bound;
  }
  return __builtin_bit_cast(float, bound & 0x80000000u ? bound & 0x7fffffffu : ~bound);
}

constexpr int kPer = kSpan / kThreads, kMost = 1024;

// One workgroup a (row, span of the vocabulary), 32 logits to a thread in
// registers: the largest one, the sum of exp(x - largest), whether one is no
// number, and the K best in order.
//
// The K-th largest of 64 groups' maxima (four threads each) is no larger than
// the K-th largest logit, so what reaches it holds the K best.  Few more than K
// do as a rule (18 for 16, 44 for 32 in random order, but 300 for 64, so from 33
// on each thread is a group), which are put in order by counting what is before
// each.  Where more than kMost do (equal logits) they are taken out one by one.
//
// 512 rows of 32768 bf16 logits: 18.6 us in a trace, 1.8 TB/s.  Loads, maximum,
// bound, sums and order follow each other in a workgroup, and five waves a SIMD hide
// a part of each: vector instructions, 19 a logit of them for the sums (fourteen on
// 64 bits), issue in 16% of a wave's cycles.  Exponentials without the table, by a
// polynomial of degree 11, took 0.9 us more, float32 ones 3.5, halved spans or twice
// the threads more as well.
template <typename T>
__global__ void __launch_bounds__(kThreads) beam_spans(BeamParams p) {
  constexpr int kVec = 16 / sizeof(T);
  typedef T Piece __attribute__((ext_vector_type(kVec), aligned(sizeof(T))));
  __shared__ uint64_t found[kMost];
  __shared__ float group[kThreads], top[kThreads / 64];
  __shared__ double sums[kThreads / 64];
  __shared__ uint64_t best[kThreads / 64];
  __shared__ double powers[kPowers];
  __shared__ int count;
  const int span = blockIdx.x % p.spans, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / p.spans, n = row / p.B, b = row % p.B;
  if (!goes_on(p, n, b)) {  // nobody asks for its candidates
    if (tid < p.K) p.keys[(int64_t)blockIdx.x * p.K + tid] = 0;
    return;
  }
  const int lo = span * kSpan, hi = lo + kSpan < p.V ? lo + kSpan : p.V;
  const T* x0 = (const T*)p.x.p + (n * p.x.s0 + b * p.x.s1);
  // value i of a thread is logit index(i)
  auto index = [&](int i) { return lo + (i / kVec * kThreads + tid) * kVec + i % kVec; };
  float x[kPer];
  Piece w[kPer / kVec];
  if (hi - lo == kSpan) {  // all loads ahead of the first use
#pragma unroll
    for (int i = 0; i < kPer; i += kVec) w[i / kVec] = *(const Piece*)(x0 + index(i));
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = (float)w[i / kVec][i % kVec];
  } else {
#pragma unroll
    for (int i = 0; i < kPer; i += kVec) {
      const int v = index(i);
      if (v + kVec <= hi) {
        w[i / kVec] = *(const Piece*)(x0 + v);
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[i + j] = (float)w[i / kVec][j];
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[i + j] = v + j < hi ? (float)x0[v + j] : -INFINITY;
      }
    }
  }
  make_powers(powers);
  if (tid == 0) count = 0;
  float own = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPer; ++i) own = __builtin_elementwise_maximum(own, x[i]);  // a NaN stays one
  group[tid] = own;
  float most = wave_max(own);
  if (lane == 0) top[wave] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) most = __builtin_elementwise_maximum(most, top[w]);
  uint64_t* out = p.keys + (int64_t)blockIdx.x * p.K;
  if (!(most > -INFINITY && most < INFINITY)) {  // nothing here, or nothing in the row
    if (tid < p.K) out[tid] = 0;
    if (tid == 0) {
      p.span[blockIdx.x].most = most;
      p.span[blockIdx.x].sum = most == -INFINITY ? 0. : (double)NAN;
    }
    return;
  }

  float least;
  if (p.K <= 32) {
    float of_group = group[lane];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) of_group = fmaxf(of_group, group[64 * w + lane]);
    least = kth_of_wave<1>({order_bits(of_group)}, p.K);
  } else {
    unsigned of_group[kThreads / 64];
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) of_group[w] = order_bits(group[64 * w + lane]);
    least = kth_of_wave(of_group, p.K);
  }
  least = fmaxf(least, -FLT_MAX);  // a logit above -infinity
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (x[i] >= least) {
      const int at = atomicAdd(&count, 1);
      if (at < kMost) found[at] = order_key(x[i], (unsigned)index(i));
    }

  double s = 0.;
#pragma unroll
  for (int i = 0; i < kPer; ++i) s = add_exp(s, (double)x[i] - (double)most, powers);
  s = wave_sum(s);
  if (lane == 0) sums[wave] = s;
  __syncthreads();
  if (tid == 0) {
    s = 0.;
    for (int w = 0; w < kThreads / 64; ++w) s += sums[w];
    p.span[blockIdx.x].most = most;
    p.span[blockIdx.x].sum = s;
  }
  const int all = count;
  if (all <= kMost) {
    for (int i = tid; i < all; i += kThreads) {
      const uint64_t mine = found[i];
      int before = 0;
      for (int j = 0; j < all; ++j) before += found[j] > mine;
      if (before < p.K) out[before] = mine;
    }
    for (int i = all + tid; i < p.K; i += kThreads) out[i] = 0;
    return;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < p.K; ++k) {
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint64_t o = x[i] > -INFINITY ? order_key(x[i], (unsigned)index(i)) : 0;
      if (o < last && o > mine) mine = o;
    }
    mine = wave_most(mine);
    if (lane == 0) best[wave] = mine;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) mine = best[w] > mine ? best[w] : mine;
    __syncthreads();
    if (tid == 0) out[k] = mine;
    last = mine;
  }
}

// What a beam adds to its logits: its largest logit, and its score less the
// logarithm of its sum of exp(x - largest); -infinity where it has no candidates.
// A beam at its end has an infinite largest logit, and its score alone.  One
// thread takes a beam, or the lanes of a wave one together.
template <bool WAVE>
__device__ __forceinline__ void beam_base_of(const BeamParams& p, float score, bool ended, const BeamSpan* s,
                                             double* most_out, double* base_out) {
  const int first = WAVE ? threadIdx.x & 63 : 0, step = WAVE ? 64 : 1;
  const bool live = score > -INFINITY && score < INFINITY;
  float most = -INFINITY;
  double sum = 0.;
  if (live && !ended) {
    for (int i = first; i < p.spans; i += step) most = __builtin_elementwise_maximum(most, s[i].most);
    if (WAVE) most = wave_max(most);
    for (int i = first; i < p.spans; i += step) {
      const double d = ((double)s[i].most - (double)most) * kLog2e64;
      sum += s[i].most > -INFINITY ? s[i].sum * exp2(d) : 0.;
    }
    if (WAVE) sum = wave_sum(sum);
  }
  const bool some = live && (ended || (most > -INFINITY && most < INFINITY));  // a NaN is neither
  *most_out = ended ? INFINITY : most;
  *base_out = some ? (double)score - (ended ? 0. : log(sum)) : -INFINITY;
}

// A candidate: its score, and what decides between equal ones as one number, the
// larger first: 63 - b, the logit's order, 2^20 - 1 - v; 0 behind every candidate.
struct Candidate {
  double c;
  uint64_t rank;
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
  return (a.c > b.c) | ((a.c == b.c) & (a.rank > b.rank));  // both loads at once
}
// The first of a candidate and another, by values: chosen by branches they lay in memory.
__device__ __forceinline__ Candidate first_of(const Candidate& a, double c, uint64_t rank) {
  const bool other = (c > a.c) | ((c == a.c) & (rank > a.rank));
  return {other ? c : a.c, other ? rank : a.rank};
}
__device__ __forceinline__ uint64_t rank_of(int b, uint64_t key) {
  return (uint64_t)(63 - b) << 52 | key >> 32 << 20 | (key & 0xfffff);
}
// Of a beam at its end, whose only candidate is token `pad`.
__device__ __forceinline__ uint64_t rank_of_end(const BeamParams& p, int b) { return rank_of(b, 0xffffffffu - (unsigned)p.pad); }
__device__ __forceinline__ int rank_beam(uint64_t rank) { return 63 - (int)(rank >> 52); }
__device__ __forceinline__ int rank_token(uint64_t rank) { return 0xfffff - (int)(rank & 0xfffff); }

constexpr int kCandidates = 2048, kLists = 512;  // of a group that beam_groups takes
constexpr int kEach = kCandidates / kThreads, kManyThreads = 1024;

struct GroupGeometry {
  FastDiv lists, spans, vocabulary;
  int each, ranks;  // of beam_groups_many: threads to a list, ranks that give the bound
};

__device__ __forceinline__ void put(const BeamParams& p, int k, double c, int b, int v) {
  const int64_t o = (int64_t)blockIdx.x * p.K + k;
  p.out[o] = (float)c;
  p.tokens[o] = v;
  p.parents[o] = b;
}
__device__ __forceinline__ void put(const BeamParams& p, int k, const Candidate& x) {
  put(p, k, x.c, rank_beam(x.rank), rank_token(x.rank));
}

// The K best of `some` candidates, which hold them, by counting what is before each.
__device__ __forceinline__ void put_best(const BeamParams& p, const GroupGeometry& g, const Candidate* found, int some,
                                         int threads) {
  const int tid = threadIdx.x;
  for (int i = tid; i < some; i += threads) {
    const Candidate mine = found[i];
    int ahead = 0;
#pragma unroll 8
    for (int j = 0; j < some; ++j) ahead += before(found[j], mine);
    if (ahead < p.K) put(p, ahead, mine);
  }
  if (some < p.K && tid < 64) {  // no more candidates: the lowest places that were not taken
    bool taken = tid >= p.K;
    for (int j = 0; j < some; ++j) taken |= rank_beam(found[j].rank) * p.V + rank_token(found[j].rank) == tid;
    const uint64_t free = __ballot(!taken);
    const int k = some + __popcll(free & ((1ull << tid) - 1));
    const int b = fdiv(tid, g.vocabulary);
    if (!taken && k < p.K) put(p, k, -INFINITY, b, tid - b * p.V);
  }
}

// The first in order of all threads' candidates, on each.
__device__ __forceinline__ Candidate best_of_block(Candidate mine, Candidate* best, int waves) {
#pragma unroll
  for (int m = 32; m; m >>= 1) {
    mine = first_of(mine, __shfl_xor(mine.c, m), shfl64(mine.rank, (threadIdx.x & 63) ^ m));
  }
  if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = mine;
  __syncthreads();
  for (int w = 0; w < waves; ++w) mine = first_of(mine, best[w].c, best[w].rank);
  __syncthreads();
  return mine;
}

constexpr int kFewLogits = 2048, kFewBeams = 16, kFewKept = 32;

// Small vocabularies in one launch: a workgroup a group, a wave a beam, 32 logits
// to a lane.  The bound is taken from the beams' scores at once: the K-th largest
// of the maxima of 64 sets, each a lane of every beam, 13 further on in each: a lane
// holds neighbouring logits, so a short row fills a few lanes only, and a set that
// none fills bounds nothing.
//
// Takes what saves a launch and a round trip of candidates, us a call, here / in two
// launches: N1 B4 V2048 K4 7.0 / 11.9, N1 B16 V2048 K16 12.2 / 12.1 (one CU's sums),
// N64 B16 V2048 K32 16.3 / 18.2, N512 B16 K16 32 / 67.  More than 2048 logits a wave
// need more registers than sixteen waves have (fewer beams would leave room for some).
// Twice as many sets as are kept have to be filled, or rows be so short that all
// candidates are few (N64 bf16 K32: B1 V250 31 / 16, B2 V250 15 / 16, B16 V200 16 / 22;
// with the same lanes of each beam in a set 1013 there).
template <typename T>
__global__ void __launch_bounds__(64 * kFewBeams) beam_few(BeamParams p, GroupGeometry g) {
  constexpr int kVec = 16 / sizeof(T), kOwn = kFewLogits / 64;
  typedef T Piece __attribute__((ext_vector_type(kVec), aligned(sizeof(T))));
  __shared__ Candidate found[kCandidates];
  __shared__ Candidate best[kFewBeams];
  __shared__ float head[kFewBeams][64];
  __shared__ double powers[kPowers];
  __shared__ int count;
  const int n = blockIdx.x, tid = threadIdx.x, lane = tid & 63, b = __builtin_amdgcn_readfirstlane(tid >> 6);
  const T* x0 = (const T*)p.x.p + (n * p.x.s0 + b * p.x.s1);
  auto index = [&](int i) { return (i / kVec * 64 + lane) * kVec + i % kVec; };
  const float score = p.scores[n * p.score0 + b * p.score1];
  const bool ended = p.ended && p.ended[n * p.ended0 + b * p.ended1], live = score > -INFINITY && score < INFINITY;
  float x[kOwn], own = -INFINITY;
#pragma unroll
  for (int i = 0; i < kOwn; i += kVec) {  // of every beam: the loads do not wait for what it is
    const int v = index(i);
    if (v + kVec <= p.V) {
      const Piece w = *(const Piece*)(x0 + v);
#pragma unroll
      for (int j = 0; j < kVec; ++j) x[i + j] = (float)w[j];
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) x[i + j] = v + j < p.V ? (float)x0[v + j] : -INFINITY;
    }
  }
  make_powers(powers);
  if (tid == 0) count = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOwn; ++i) own = __builtin_elementwise_maximum(own, x[i]);  // a NaN stays one
  const float most = wave_max(own);
  const bool reads = live && !ended && most > -INFINITY && most < INFINITY;
  double base = score;
  if (reads) {
    double s = 0.;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) s = add_exp(s, (double)x[i] - (double)most, powers);
    base -= log(wave_sum(s));
  }
  const Candidate end = {live && ended && lane == 0 ? base : -INFINITY, rank_of_end(p, b)};
  head[b][lane] = reads ? (float)((double)own - (double)most + base) : (float)end.c;
  __syncthreads();
  float of_set = -INFINITY;
  for (int w = 0; w < p.B; ++w) of_set = fmaxf(of_set, head[w][(lane + 13 * w) & 63]);
  const float least = kth_of_wave<1>({order_bits(of_set)}, p.K);
  // f for each candidate of this lane
  auto each = [&](auto f) {
    if (reads) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
        if (x[i] > -INFINITY) f(Candidate{(double)x[i] - (double)most + base, rank_of(b, order_key(x[i], (unsigned)index(i)))});
    } else if (end.c > -INFINITY) {
      f(end);
    }
  };
  each([&](Candidate c) {
    if ((float)c.c < least) return;
    const int i = atomicAdd(&count, 1);
    if (i < kCandidates) found[i] = c;
  });
  __syncthreads();
  // Counting what is before each takes 25 ns a comparison of all threads, a round of taking out the best 4 us.
  if (count <= kCandidates && (count + 64 * p.B - 1) / (64 * p.B) * count <= 128 * p.K) {
    put_best(p, g, found, count, 64 * p.B);
    return;
  }
  // Many equal scores: the best is taken out K times, and the next of its beam's logits stands in.
  uint64_t key = ~0ull;
  Candidate first = {-INFINITY, 0}, mine = end;
  for (int k = 0; k < p.K; ++k) {
    if (reads && (k == 0 || first.rank == mine.rank)) {
      uint64_t next = 0;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const uint64_t o = x[i] > -INFINITY ? order_key(x[i], (unsigned)index(i)) : 0;
        if (o < key && o > next) next = o;
      }
      key = wave_most(next);
      mine = Candidate{key ? (double)key_logit(key) - (double)most + base : -INFINITY, key ? rank_of(b, key) : 0};
    } else if (first.rank == mine.rank) {
      mine = Candidate{-INFINITY, 0};
    }
    first = best_of_block(mine, best, p.B);
    if (tid == 0) put(p, k, first);
  }
}

// One workgroup a group.  Every (beam, span) gave a list of candidates in order.
// As in a span, the K-th largest of 64 sets' maxima (scores rounded to float32,
// which keeps the order) is a bound that few more than the K best reach, and
// those are put in order by counting what is before each.  A group takes ranks
// 13 lists apart, so that neither the first ranks of all lists nor a good beam's
// lists share one.  Bound by its chain: keys, sums, maxima, order (5.4 us for 32
// lists of 16).
__global__ void __launch_bounds__(kThreads) beam_groups(BeamParams p, GroupGeometry g) {
  __shared__ Candidate found[kCandidates];
  __shared__ BeamSpan span[kLists];
  __shared__ double base[64], most[64];
  __shared__ unsigned group[64];
  __shared__ int count;
  const int n = blockIdx.x, tid = threadIdx.x, lists = p.B * p.spans, all = lists * p.K;
  const uint64_t* keys = p.keys + (int64_t)n * all;
  for (int l = tid; l < lists; l += kThreads) span[l] = p.span[(int64_t)n * lists + l];
  const float score = tid < p.B ? p.scores[n * p.score0 + tid * p.score1] : 0.f;
  const bool ended = tid < p.B && p.ended && p.ended[n * p.ended0 + tid * p.ended1];
  uint64_t key[kEach];
  int list[kEach], rank[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = tid + j * kThreads;
    rank[j] = fdiv(i, g.lists);
    list[j] = i - rank[j] * lists;
    key[j] = i < all ? keys[list[j] * p.K + rank[j]] : 0;
  }
  if (tid == 0) count = 0;
  if (tid < 64) group[tid] = order_bits(-INFINITY);
  __syncthreads();
  if (tid < p.B) beam_base_of<false>(p, score, ended, span + tid * p.spans, &most[tid], &base[tid]);
  __syncthreads();
  Candidate cand[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    cand[j] = Candidate{-INFINITY, 0};
    if (tid + j * kThreads >= all) continue;
    const int b = fdiv(list[j], g.spans);
    if (most[b] == INFINITY) {  // at its end: goes on as it is, once
      if (rank[j] == 0 && list[j] == b * p.spans) cand[j] = Candidate{base[b], rank_of_end(p, b)};
    } else if (key[j]) {
      cand[j] = Candidate{(double)key_logit(key[j]) - most[b] + base[b], rank_of(b, key[j])};
    }
    if (!(cand[j].c > -INFINITY)) cand[j].c = -INFINITY;  // of a beam that has none
    if (cand[j].c > -INFINITY) atomicMax(&group[(list[j] + 13 * rank[j]) & 63], order_bits((float)cand[j].c));
  }
  __syncthreads();
  const float least = kth_of_wave<1>({group[tid & 63]}, p.K);
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (cand[j].c > -INFINITY && (float)cand[j].c >= least) found[atomicAdd(&count, 1)] = cand[j];
  __syncthreads();
  put_best(p, g, found, count, kThreads);
}

// The same for more lists than that: a list's first threads' ranks are read as
// far as they reach the bound, the K-th largest of 256 sets' maxima over the
// lists' first ranks (8192 candidates).  Where more than kCandidates reach it (equal scores) the
// best is taken out K times.  A call of 64 beams, 131072 logits, K 64: 38 us (a
// merge of the lists' heads by one wave: 511).
__global__ void __launch_bounds__(kManyThreads) beam_groups_many(BeamParams p, GroupGeometry g) {
  constexpr int kWaves = kManyThreads / 64, kDeep = 4, kSets = 256;
  __shared__ Candidate found[kCandidates];
  __shared__ Candidate best[kWaves];
  __shared__ double base[64], most[64];
  __shared__ unsigned group[kSets];
  __shared__ int count;
  const int n = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lists = p.B * p.spans;
  const uint64_t* keys = p.keys + (int64_t)n * lists * p.K;
  if (tid == 0) count = 0;
  if (tid < kSets) group[tid] = order_bits(-INFINITY);
  for (int b = wave; b < p.B; b += kWaves) {
    const float score = p.scores[n * p.score0 + b * p.score1];
    const bool ended = p.ended && p.ended[n * p.ended0 + b * p.ended1];
    double m, add;
    beam_base_of<true>(p, score, ended, p.span + ((int64_t)n * p.B + b) * p.spans, &m, &add);
    if (lane == 0) most[b] = m, base[b] = add;
  }
  __syncthreads();
  // f(candidate, number of its maximum) for this thread's candidates below a rank, each list's until f is false
  auto walk = [&](int ranks, auto f) {
    const int sub = tid & (g.each - 1);
    for (int l = tid / g.each; l < lists; l += kManyThreads / g.each) {
      const int b = fdiv(l, g.spans);
      const double largest = most[b], add = base[b];
      if (!(add > -INFINITY)) continue;
      if (largest == INFINITY) {  // at its end: goes on as it is, once
        if (sub == 0 && l == b * p.spans) f(Candidate{add, rank_of_end(p, b)}, l);
        continue;
      }
      bool on = true;
      for (int r0 = sub; on && r0 < ranks; r0 += kDeep * g.each) {
        uint64_t key[kDeep];
#pragma unroll
        for (int j = 0; j < kDeep; ++j) {
          const int r = r0 + j * g.each;
          key[j] = r < ranks ? keys[(int64_t)l * p.K + r] : 0;
        }
#pragma unroll
        for (int j = 0; j < kDeep; ++j) {
          on = on && key[j];
          if (on)
            on = f(Candidate{(double)key_logit(key[j]) - largest + add, rank_of(b, key[j])}, l + 13 * (r0 + j * g.each));
        }
      }
    }
  };
  walk(g.ranks, [&](Candidate x, int at) {
    atomicMax(&group[at & (kSets - 1)], order_bits((float)x.c));
    return true;
  });
  __syncthreads();
  unsigned of_set[kSets / 64];
#pragma unroll
  for (int w = 0; w < kSets / 64; ++w) of_set[w] = group[64 * w + lane];
  const float least = kth_of_wave(of_set, p.K);
  walk(p.K, [&](Candidate x, int) {
    if ((float)x.c < least) return false;
    const int i = atomicAdd(&count, 1);
    if (i < kCandidates) found[i] = x;
    return true;
  });
  __syncthreads();
  if (count <= kCandidates) {
    put_best(p, g, found, count, kManyThreads);
    return;
  }
  Candidate last = {INFINITY, 0};
  for (int k = 0; k < p.K; ++k) {
    Candidate mine = {-INFINITY, 0};
    walk(p.K, [&](Candidate x, int) {
      mine = first_of(mine, before(last, x) ? x.c : -INFINITY, x.rank);
      return true;
    });
    mine = best_of_block(mine, best, kWaves);
    if (tid == 0) put(p, k, mine);
    last = mine;
  }
}

}  // namespace

int beam_spans_of(int64_t V) { return (int)((V + kSpan - 1) / kSpan); }

int launch_beam(const BeamParams& p, hipStream_t st, hipError_t* err) {
  const int lists = p.B * p.spans;
  GroupGeometry g = {fast_div(lists), fast_div(p.spans), fast_div(p.V), 1, 8192 / lists};
  const int64_t filled = p.B * ((p.V * (p.x.dt == TENSION_F32 ? 4 : 2) + 15) / 16);  // lanes, of all beams
  if (p.V <= kFewLogits && p.B <= kFewBeams && p.K <= kFewKept && (p.V <= 128 || filled >= 2 * p.K)) {
    const unsigned n = (unsigned)p.N, threads = 64 * (unsigned)p.B;
    if (p.x.dt == TENSION_F32) beam_few<float><<<n, threads, 0, st>>>(p, g);
    else if (p.x.dt == TENSION_F16) beam_few<f16><<<n, threads, 0, st>>>(p, g);
    else beam_few<bf16><<<n, threads, 0, st>>>(p, g);
    *err = hipGetLastError();
    return 0;
  }
  const unsigned n = (unsigned)((int64_t)p.N * p.B * p.spans);
  if (p.x.dt == TENSION_F32) beam_spans<float><<<n, kThreads, 0, st>>>(p);
  else if (p.x.dt == TENSION_F16) beam_spans<f16><<<n, kThreads, 0, st>>>(p);
  else beam_spans<bf16><<<n, kThreads, 0, st>>>(p);
  *err = hipGetLastError();
  if (*err != hipSuccess) return 0;
  if (lists <= kLists && lists * p.K <= kCandidates) {
    beam_groups<<<(unsigned)p.N, kThreads, 0, st>>>(p, g);
  } else {
    while (g.each < p.K && 2 * g.each * lists <= kManyThreads) g.each *= 2;
    g.ranks = g.ranks < 1 ? 1 : g.ranks < p.K ? g.ranks : p.K;
    beam_groups_many<<<(unsigned)p.N, kManyThreads, 0, st>>>(p, g);
  }
  *err = hipGetLastError();
  return 0;
}

}  // namespace tension
