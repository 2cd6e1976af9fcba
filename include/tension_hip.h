/*
 * tension_hip.h -- C ABI of the MI355X (gfx950) sigmoid-tension library
 * (libtension_hip.so).
 *
 * The reference has no native FFI for this path: its boundary is the Python
 * autograd op `causal_tension(Q, K, V, window, scale, return_tau=False,
 * bias=None)` (triton_tension/ops.py:192-224), which launches three Triton
 * kernels with raw pointers, sizes and strides (ops.py:104-112,165-182;
 * kernel.py:42-55,131-144,233-246).  The entry points below replace those
 * launches one for one; the Python host layer (bozo_amd/ops.py) binds them
 * with ctypes.
 *
 * Conventions
 *  - Every tensor is described by a tension_buf: device pointer, dtype code,
 *    and element strides.  4-D activations are [B,T,H,D] with strides
 *    s[0..3] for (B,T,H,D); s[3] must be 1.  tau is [B,T,H,W] (s[3] == 1),
 *    bias [B,T,W] (local) or [B,T,T] (global) uses s[0..2] and needs
 *    s[2] == 1; mass is [B,T,H] (s[0..2]).
 *  - A NULL tension_buf pointer means "absent" (no tau, no bias, ...).
 *  - The library never allocates device memory.  Work is enqueued on the
 *    given stream; no call synchronises the device.  All functions are
 *    reentrant; the only global state is the per-thread error string and
 *    the fixed device scratch of tension_global_bwd_noalloc.
 *  - Return value: TENSION_OK or a TENSION_ERR_* code; tension_last_error()
 *    describes the last failure on the calling thread.  Nothing throws
 *    across the ABI.
 */
#ifndef TENSION_HIP_H
#define TENSION_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* tension_stream_t; /* == hipStream_t */

/* dtype codes */
enum {
  TENSION_F32 = 0,
  TENSION_BF16 = 1,
  TENSION_F16 = 2,
  TENSION_F64 = 3,
  /* pages of a paged cache only */
  TENSION_E4M3 = 4, /* 8-bit float, 4 exponent and 3 mantissa bits, no infinity */
  TENSION_U8 = 5,   /* exponent bytes */
  TENSION_E2M1 = 6  /* 4-bit float, two to a byte (the first in its low half) */
};

/* status codes */
enum {
  TENSION_OK = 0,
  TENSION_ERR_ARG = 1,         /* bad pointer / shape / stride / dtype combination */
  TENSION_ERR_UNSUPPORTED = 2, /* valid request this build has no kernel for (e.g. D) */
  TENSION_ERR_LAUNCH = 3       /* hipGetLastError() after the launch was not hipSuccess */
};

/* flags */
enum {
  /* out = msg / max(sum_w tau, 1e-6)        (model.py:257-258,281-282) */
  TENSION_NORM_MASS = 1 << 0,
  /* out = msg / max(min(t, W), 1)            (model.py:159-163,264) */
  TENSION_NORM_COUNT = 1 << 1,
  /* bias is [B,T,T] indexed by key position (global block, model.py:224-225) */
  TENSION_GLOBAL = 1 << 2,
  /* force the exact (non-MFMA) kernels even when the MFMA path applies */
  TENSION_FORCE_EXACT = 1 << 3,
  /* decode: the new token is also a key (keys s <= t, the global block's
   * diagonal, model.py:221) */
  TENSION_DECODE_SELF = 1 << 4
};

typedef struct tension_buf {
  void* ptr;
  int32_t dtype;
  int32_t reserved;
  int64_t s[4];
} tension_buf;

/* ---------------------------------------------------------------------------
 * Local window forward.  Replaces `_fwd_kernel` (kernel.py:41-125) launched by
 * `_CausalTensionFn.forward` (ops.py:75-124).
 *   tau[b,t,h,w] = sigmoid(q_t . k_s / scale + bias[b,t,w]),  s = t-(W-w),
 *                  0 where s < 0;  msg = sum_w tau * v_s.
 *   out = msg (raw, the reference contract), or normalised per flags.
 *   q,k,v,out: [B,T,H,D]; tau (nullable, out): [B,T,H,W], written fully
 *   (zeros on empty slots); bias (nullable): [B,T,W];
 *   mass (nullable, out): [B,T,H] = sum_w tau (unclamped), f32 or f64.
 * ------------------------------------------------------------------------- */
int tension_window_fwd(const tension_buf* q, const tension_buf* k,
                       const tension_buf* v, const tension_buf* out,
                       const tension_buf* tau, const tension_buf* bias,
                       const tension_buf* mass, int64_t B, int64_t T,
                       int64_t H, int64_t D, int64_t W, double scale,
                       int32_t flags, tension_stream_t stream);

/* Bytes of device workspace tension_window_bwd needs (0 if none; -1 for
 * sizes the entry points reject: negative, or B*T*H above 2^40). */
int64_t tension_window_bwd_workspace(int64_t B, int64_t T, int64_t H,
                                     int32_t dtype_acc, int32_t flags);

/* ---------------------------------------------------------------------------
 * Local window backward.  Replaces `_bwd_dq_kernel` + `_bwd_dkv_kernel`
 * (kernel.py:130-341) launched by `_CausalTensionFn.backward`
 * (ops.py:126-187).  For windows W <= 64 with bf16 rows (head dim 64,
 * 16-byte aligned rows) it launches one kernel that produces dQ, dK and
 * dV in a single pass; otherwise tension_window_bwd_dq then
 * tension_window_bwd_dkv on `stream`.  Recomputes tau from q, k (and
 * bias); nothing from the forward is needed besides the inputs.
 *   dout: grad of out (of the raw msg without a NORM flag, of the
 *   normalised output with one); dtau (nullable): grad of tau [B,T,H,W];
 *   bias: as in the forward (sigma' is taken at the biased argument,
 *   kernel.py:24-29; bias gets no gradient).  dq/dk/dv are written, not
 *   accumulated, in their own dtypes.
 *   workspace: tension_window_bwd_workspace() bytes (NULL if that is 0);
 *   with TENSION_NORM_MASS it carries per-query coefficients from the dq
 *   kernel to the dkv kernel (the single-pass kernel forms them in
 *   registers and leaves the workspace untouched; it is required either
 *   way, so callers need not know which kernel runs).
 * ------------------------------------------------------------------------- */
int tension_window_bwd(const tension_buf* q, const tension_buf* k,
                       const tension_buf* v, const tension_buf* dout,
                       const tension_buf* dtau, const tension_buf* bias,
                       const tension_buf* dq, const tension_buf* dk,
                       const tension_buf* dv, void* workspace, int64_t B,
                       int64_t T, int64_t H, int64_t D, int64_t W,
                       double scale, int32_t flags, tension_stream_t stream);

/* tension_window_bwd with the forward's output rows `out` ([B,T,H,D], as
 * written by tension_window_fwd) and tau mass `mass` ([B,T,H] f32, the
 * forward's `mass` output), both required.  No counterpart in the reference
 * (its backward recomputes everything, ops.py:126-187): with
 * TENSION_NORM_MASS on the float32-Q/K split kernels and a window wider
 * than 64 the per-query coefficients then come from these rows --
 * a = 1/max(m, 1e-6), c = dout.out * a (0 where m < 1e-6) -- in one pass
 * over the band instead of two; every other case computes them as
 * tension_window_bwd does.  Same results to float32 rounding. */
int tension_window_bwd_saved(const tension_buf* q, const tension_buf* k,
                             const tension_buf* v, const tension_buf* dout,
                             const tension_buf* dtau, const tension_buf* bias,
                             const tension_buf* out, const tension_buf* mass,
                             const tension_buf* dq, const tension_buf* dk,
                             const tension_buf* dv, void* workspace, int64_t B,
                             int64_t T, int64_t H, int64_t D, int64_t W,
                             double scale, int32_t flags, tension_stream_t stream);

/* The two halves of tension_window_bwd, one kernel each.  _dq fills the
 * workspace that _dkv reads, so on one stream _dq must precede _dkv.
 * Counterparts: kernel.py:130-227 (dQ) and kernel.py:232-341 (dK/dV). */
int tension_window_bwd_dq(const tension_buf* q, const tension_buf* k,
                          const tension_buf* v, const tension_buf* dout,
                          const tension_buf* dtau, const tension_buf* bias,
                          const tension_buf* dq, void* workspace, int64_t B,
                          int64_t T, int64_t H, int64_t D, int64_t W,
                          double scale, int32_t flags, tension_stream_t stream);
int tension_window_bwd_dkv(const tension_buf* q, const tension_buf* k,
                           const tension_buf* v, const tension_buf* dout,
                           const tension_buf* dtau, const tension_buf* bias,
                           const tension_buf* dk, const tension_buf* dv,
                           void* workspace, int64_t B, int64_t T, int64_t H,
                           int64_t D, int64_t W, double scale, int32_t flags,
                           tension_stream_t stream);

/* ---------------------------------------------------------------------------
 * Global (full causal, diagonal included) block, tau-mass normalised.
 * Replaces the PyTorch einsum path of the global layer (model.py:217-238);
 * the reference has no kernel for it.
 *   bias (nullable): [B,T,T] indexed [b,t,s].
 *   tau_local (nullable, out): [B,T,H,Wl] with slot j = key s = T-1-j
 *   (model.py:231-237), zero where s > t.  mass (nullable, out): [B,T,H]
 *   = sum_s tau (unclamped).
 * ------------------------------------------------------------------------- */
int tension_global_fwd(const tension_buf* q, const tension_buf* k,
                       const tension_buf* v, const tension_buf* out,
                       const tension_buf* tau_local, const tension_buf* bias,
                       const tension_buf* mass, int64_t B, int64_t T,
                       int64_t H, int64_t D, int64_t Wl, double scale,
                       int32_t flags, tension_stream_t stream);

/* Bytes of device workspace tension_global_bwd needs (-1 as above). */
int64_t tension_global_bwd_workspace(int64_t B, int64_t T, int64_t H,
                                     int32_t dtype_acc, int32_t flags);

/* Backward of tension_global_fwd: dout (grad of out), dtau_local
 * (nullable, grad of tau_local [B,T,H,Wl]); recomputes tau like the local
 * backward.  workspace: tension_global_bwd_workspace() bytes (required).
 *   out, mass (nullable, in): the forward's output and mass.  When both are
 *   given (bf16 out, f32 mass, the bf16 head-dim-64 kernels), the per-query
 *   coefficients 1/m_t and dO_t.out_t/m_t come from one pass over these rows
 *   instead of a recompute of the whole causal band; otherwise they are
 *   ignored and the band is recomputed. */
int tension_global_bwd(const tension_buf* q, const tension_buf* k,
                       const tension_buf* v, const tension_buf* dout,
                       const tension_buf* dtau_local, const tension_buf* bias,
                       const tension_buf* out, const tension_buf* mass,
                       const tension_buf* dq, const tension_buf* dk,
                       const tension_buf* dv, void* workspace, int64_t B,
                       int64_t T, int64_t H, int64_t D, int64_t Wl,
                       double scale, int32_t flags, tension_stream_t stream);

/* ---------------------------------------------------------------------------
 * tension_global_bwd without a caller workspace.  No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  Same arguments and results as tension_global_bwd minus
 * `workspace`; the per-query coefficients live in a fixed device array inside
 * the library, TENSION_NOALLOC_SCRATCH_BYTES per GPU (one copy per device,
 * held until the process ends; its address is looked up on the first call
 * with that device current).  The call allocates nothing.  It needs
 * 2 * B * T * H * 4 bytes (8 with f64 activations) of that array; larger
 * requests return TENSION_ERR_ARG.  Every call on one GPU shares the array:
 * calls that overlap on one GPU (several streams, several host threads) race
 * and must be serialised by the caller.
 * ------------------------------------------------------------------------- */
#define TENSION_NOALLOC_SCRATCH_BYTES (8 << 20)

int tension_global_bwd_noalloc(const tension_buf* q, const tension_buf* k,
                               const tension_buf* v, const tension_buf* dout,
                               const tension_buf* dtau_local,
                               const tension_buf* bias, const tension_buf* out,
                               const tension_buf* mass, const tension_buf* dq,
                               const tension_buf* dk, const tension_buf* dv,
                               int64_t B, int64_t T, int64_t H, int64_t D,
                               int64_t Wl, double scale, int32_t flags,
                               tension_stream_t stream);

/* ---------------------------------------------------------------------------
 * Streaming decode step over a ring K/V cache (no reference kernel: the
 * reference re-runs the whole forward per token, model.py:617-652,719-768;
 * the streaming exporter reads tau[:, -1], ts_bridge/streaming.py:125-127).
 *   q, k_new, v_new, out: [N,H,D] (s[0..2] used, s[2] == 1).
 *   k_cache, v_cache: [N,H,W,D] (s[0..3], s[3] == 1), updated in place:
 *   after attending, k_new/v_new are written to slot pos[n] % W.
 *   pos_in: device int32 [N], tokens already cached per sequence.
 *   pos_out (nullable): device int32 [N], receives pos_in + 1 (must not
 *   alias pos_in).  tau (nullable, out): [N,H,W], w=0 oldest.
 *   Attends to the min(pos, W) most recent cached tokens (strictly past),
 *   plus the new token itself with TENSION_DECODE_SELF (a global layer's
 *   step: the cache then holds every earlier token, W >= positions; tau
 *   must be null).
 *   flags: TENSION_NORM_MASS (tau-mass normalised), TENSION_NORM_COUNT
 *   (divided by the number of keys, max(min(pos, W), 1) for a local layer,
 *   the valid count of model.py:159-163,264) or neither (raw); optionally
 *   TENSION_DECODE_SELF.
 * ------------------------------------------------------------------------- */
int tension_decode_step(const tension_buf* q, const tension_buf* k_new,
                        const tension_buf* v_new, const tension_buf* k_cache,
                        const tension_buf* v_cache, const tension_buf* out,
                        const tension_buf* tau, const int32_t* pos_in,
                        int32_t* pos_out, int64_t N, int64_t H, int64_t D,
                        int64_t W, double scale, int32_t flags,
                        tension_stream_t stream);

/* ---------------------------------------------------------------------------
 * RoPE (half-split rotation, model.py:54-81).  y = R(pos) x, or R(pos)^T x
 * when inverse != 0 (the backward).  cos/sin: contiguous float32
 * [table_rows, D/2] tables (the model's buffers); rows
 * pos_offset .. pos_offset+T-1 are used and must exist.
 * x, y: [B,T,H,D]; y may alias x.  A negative pos_in entry of
 * tension_decode_step is read as 0.
 * ------------------------------------------------------------------------- */
int tension_rope(const tension_buf* x, const tension_buf* y, const float* cos,
                 const float* sin, int64_t table_rows, int64_t B, int64_t T,
                 int64_t H, int64_t D, int64_t pos_offset, int32_t inverse,
                 tension_stream_t stream);

/* ---------------------------------------------------------------------------
 * tau export reductions (replace the host numpy passes of the reference's
 * graph exporter over .cpu() copies of tau).  taus: L <= 32 buffers of
 * tau [B,T,H,W] (s[3] == 1, any float dtype), one per local layer; every
 * statistic reads the batch mean of tau.
 *
 * tension_tau_head_stats -- ts_bridge/head_filter.py:98-130 (profile_heads)
 *   and, with TENSION_TAU_VALID_ONLY (cells with t + w < W read as 0),
 *   ts_bridge/corpus_profile.py:58-98 (_per_head_stats).  stats: device
 *   float [L,H,4] = mean over (t, w); 0.99 quantile over (t, w) (linear
 *   interpolation, numpy's default); mean over t of the first arg-max over
 *   w; mean over t of the max over w.
 * ------------------------------------------------------------------------- */
enum { TENSION_TAU_VALID_ONLY = 1 << 5 };

int tension_tau_head_stats(const tension_buf* taus, int32_t L, int64_t B,
                           int64_t T, int64_t H, int64_t W, float* stats,
                           int32_t flags, tension_stream_t stream);

/* tension_tau_aggregate -- ts_bridge/export.py:185-200 (and the per-step
 *   form of streaming.py:127-146): agg[t,w] (device float [T,W]) = mean over
 *   the selected (layer, head) pairs of tau; head_mask: device int32 [L,H],
 *   nonzero = selected; all pairs when none is.  H <= 64. */
int tension_tau_aggregate(const tension_buf* taus, int32_t L, int64_t B,
                          int64_t T, int64_t H, int64_t W,
                          const int32_t* head_mask, float* agg,
                          tension_stream_t stream);

/* ---------------------------------------------------------------------------
 * The model's tau regularisers (model.py:498-611: tension_diversity_loss,
 * constraint_consistency_loss, tension_entropy_loss) over the tau of L <= 32
 * layers, each [B,T,H,W] (W <= 256, s[3] == 1), computed in fp32.
 *
 * tension_aux_loss_fwd: partials (device double [L, P, 4], P =
 *   tension_aux_loss_partials(B,T,H)) receives, per layer and workgroup, the
 *   sums of: row entropy -sum p log(p + 1e-8) with p = tau / (sum tau +
 *   1e-8); the consistency terms relu(tau[r,w1-1] tau[r-1,0] - tau[r,w1])
 *   (w1 = 1..min(W-2,4), w1+1 <= r <= w1+T-min(W-2,4)-1); relu(0.05 - m);
 *   relu(m - 0.8), m the row mean.  The caller sums over P and forms the
 *   losses.
 * tension_aux_loss_bwd: dtaus[l] = k_div[l] d(row entropy)/dtau
 *   + k_cons[l] d(consistency terms)/dtau + k_ent[l] d(relu sums)/dtau,
 *   coef = device float [L, 3] (k_div, k_cons, k_ent); every element of
 *   every dtau is written.
 * ------------------------------------------------------------------------- */
int64_t tension_aux_loss_partials(int64_t B, int64_t T, int64_t H);

int tension_aux_loss_fwd(const tension_buf* taus, int32_t L, int64_t B,
                         int64_t T, int64_t H, int64_t W, double* partials,
                         tension_stream_t stream);

int tension_aux_loss_bwd(const tension_buf* taus, const tension_buf* dtaus,
                         int32_t L, int64_t B, int64_t T, int64_t H,
                         int64_t W, const float* coef,
                         tension_stream_t stream);

/* ---------------------------------------------------------------------------
 * Graph-bias builder (ts_bridge/bias.py:125-233 GraphBias.local_bias /
 * global_bias, whose O(T W) / O(T^2) host loops look up a content-pair ->
 * weight map per (query, key)).  The map lives on the device as an
 * open-addressing table: keys uint64 (src_id << 32 | dst_id), values double,
 * capacity 2^log2cap, empty slots hold ~0 (fill table_keys with 0xff bytes
 * first).  Hash: slot = (key * 0x9E3779B97F4A7C15) >> (64 - log2cap) (mod
 * 2^64), linear probing.
 *
 * tension_bias_table_insert: insert n distinct keys (2 n <= capacity).
 * tension_bias_build: content_ids device int32 [T] (-1 = no entry); bias
 *   [B,T,W] (W > 0, key s = t - (W - w), zero where s < 0) or [B,T,T]
 *   (W == 0, keys s < t), s[2] == 1, any float dtype; every element written:
 *   alpha * weight(ids[s] -> ids[t]) where the weight is > 0, else 0.
 *   stats (nullable, device double [3], caller-zeroed): += hits, += sum of
 *   the hit weights, max of the hit weights.
 * ------------------------------------------------------------------------- */
int tension_bias_table_insert(const uint64_t* keys_in, const double* vals_in,
                              int64_t n, uint64_t* table_keys,
                              double* table_vals, int32_t log2cap,
                              tension_stream_t stream);

int tension_bias_build(const int32_t* content_ids, int64_t B, int64_t T,
                       int64_t W, const uint64_t* table_keys,
                       const double* table_vals, int32_t log2cap,
                       double alpha, const tension_buf* bias, double* stats,
                       tension_stream_t stream);

/* ---------------------------------------------------------------------------
 * Paged K/V cache: tokens of sequences of different lengths in pages of S
 * tokens from one pool (no counterpart in the reference, whose generation
 * keeps no cache, model.py:736-739).
 *   k, v: [P,Hk,S,D] pages (s[0..3], s[3] == 1; P = pages, S = page_size),
 *     float32, bf16, f16 or e4m3, each its own type, or both e2m1: [P,Hk,S,D/2]
 *     bytes of two codes, D even.  A page may lie beyond 2^32 elements from the
 *     first.
 *   k_exp, v_exp: [P,Hk,S] exponent bytes (s[0..2], TENSION_U8) of an e4m3
 *     buffer, ptr NULL otherwise: a row's value is code * 2^(byte - 127).  Of an
 *     e2m1 buffer [P,Hk,S,ceil(D/32)] (s[3] == 1), a byte for every 32 values;
 *     255 makes them no numbers.
 *   table: device int32 [N,table_len], row stride table_stride: page
 *     table[n][pos / S] holds position pos of sequence n at row pos % S.
 *     An entry outside [0, P) is no page: its tokens are not written, read
 *     back as zeros, and attended to by nothing.
 * ------------------------------------------------------------------------- */
typedef struct tension_paged {
  tension_buf k, v, k_exp, v_exp;
  const int32_t* table;
  int64_t table_stride, table_len, pages, page_size;
} tension_paged;

/* Writes tokens k_new, v_new [N,T,Hk,D] (float32, bf16 or f16) at positions
 * start[n] .. start[n] + counts[n] - 1 (device int32 [N]; counts NULL = T,
 * clamped to [0, T]); positions below 0 or past the table are left out.
 *   Pages of the source's type take the values as they are, bf16 or f16
 * pages of float32 tokens the nearest ones (other mixes are refused), e4m3
 * pages per row the smallest power of two 2^e, e >= -126, with max |x| <=
 * 448 * 2^e over the row's finite values, and x / 2^e rounded to nearest
 * even; infinities become NaN.  e2m1 pages likewise per 32 values the smallest
 * 2^e, -126 <= e <= 125, with max |x| <= 6 * 2^e (larger values become 6 *
 * 2^125); 32 values with an infinity or a NaN among them are all stored as no
 * number (byte 255, codes 0).  Two tokens of one call in
 * one place leave one of them. */
int tension_paged_append(const tension_paged* cache, const tension_buf* k_new,
                         const tension_buf* v_new, const int32_t* start,
                         const int32_t* counts, int64_t N, int64_t T,
                         int64_t Hk, int64_t D, tension_stream_t stream);

/* The same for tokens whose places are known already: token t of row n goes to
 * page slots[n][t] / S, row slots[n][t] % S (device int64 [N,T], element
 * strides slot_s0, slot_s1); a slot outside [0, P * S) is none, and its token is
 * left out.  No two tokens of a call may share a slot: what is left there may be
 * parts of both.  The cache's table is not read and may be NULL. */
int tension_paged_store(const tension_paged* cache, const tension_buf* k_new,
                        const tension_buf* v_new, const int64_t* slots,
                        int64_t slot_s0, int64_t slot_s1, int64_t N, int64_t T,
                        int64_t Hk, int64_t D, tension_stream_t stream);

/* Reads positions start[n] + t back into k_out, v_out [N,T,Hk,D] (float32,
 * bf16 or f16, each its own type; every element written): zeros for t >=
 * counts[n], positions below 0 or past the table, and entries that are no
 * page. */
int tension_paged_read(const tension_paged* cache, const tension_buf* k_out,
                       const tension_buf* v_out, const int32_t* start,
                       const int32_t* counts, int64_t N, int64_t T, int64_t Hk,
                       int64_t D, tension_stream_t stream);

/* One new token per sequence over its cached tokens (the step of
 * tension_decode_step on pages; the new token is in the cache already).
 *   q, out: [N,H,D] (s[0..2]), float32, bf16 or f16, alike; H a multiple of
 *   Hk, query head h reads key head h / (H / Hk).  D <= 256.
 *   lengths: device int32 [N], cached tokens of each sequence, the newest at
 *   position lengths[n] - 1 (clamped to [0, table_len * S]).
 *   Keys lo <= s < hi: hi = lengths[n] with TENSION_DECODE_SELF, else
 *   lengths[n] - 1; lo = max(0, lengths[n] - 1 - W), or 0 with W == 0.
 *   out = sum tau v, tau = sigmoid(q . k / scale), divided by max(sum tau,
 *   1e-6) with TENSION_NORM_MASS, by max(hi - lo, 1) with
 *   TENSION_NORM_COUNT; zeros where there is no key.  Rows outside [lo, hi)
 *   have no part in the result, whatever they hold, but may be loaded: other
 *   rows of the pages that the range touches, and the first page for an entry
 *   that is no page.  So all P pages must be memory that can be read.
 *   max_len: a bound of the lengths that the host knows (0: none); it only
 *   shapes the launch, a longer sequence is attended to in full.
 *   workspace: tension_paged_decode_workspace() bytes for the same sizes, of
 *   e2m1 pages tension_paged_decode_workspace_e2m1() (NULL if that is 0; -1 for
 *   sizes the entry point rejects).  The keys
 *   of a sequence are split over workgroups where there are few rows; the
 *   partial sums meet there and are added in a fixed order. */
int64_t tension_paged_decode_workspace(int64_t N, int64_t H, int64_t Hk,
                                       int64_t D, int64_t W, int64_t max_len,
                                       int64_t table_len, int64_t page_size);
int64_t tension_paged_decode_workspace_e2m1(int64_t N, int64_t H, int64_t Hk,
                                            int64_t D, int64_t W, int64_t max_len,
                                            int64_t table_len, int64_t page_size);
int tension_paged_decode(const tension_paged* cache, const tension_buf* q,
                         const tension_buf* out, const int32_t* lengths,
                         void* workspace, int64_t N, int64_t H, int64_t Hk,
                         int64_t D, int64_t W, int64_t max_len, double scale,
                         int32_t flags, tension_stream_t stream);

/* Pages for the tokens of a call, taken from a stack of free ones or given
 * back, and the tokens' slots.
 *   table: device int32 [N,table_len], row stride table_stride, changed in
 *     place.  free, top: device int32 [pages] and [1]: the free pages are
 *     free[0 .. top - 1], the last on top.
 *   lengths, counts: device int32 [N]: tokens a sequence holds before the call
 *     (clamped to [0, table_len * page_size]) and by how many it grows, or with
 *     a negative count is cut (to nothing at the least).  window (0: none):
 *     queries read the last `window` positions before their own only.
 *   With L and E the tokens before and after: entries from ceil(E / S) to
 *   ceil(L / S) go back, and with a window those before
 *   (min(L, E) - window) / S, from the last of them down to the first that has
 *   no page; then a sequence that grows takes a page for each entry without one
 *   from max((E - window) / S, L / S) to ceil(E / S).  Pages go on top of the
 *   stack and come from there in the order of the sequences and their entries,
 *   the first given back the highest, so that a cut undoes a growth.
 *   missing: device int32 [1], 0; or the pages by which the stack is short
 *   (-1: more pages would be free than there are), and nothing has changed.
 *   slots: device int64 [N,T], contiguous: page * S + row of position lengths[n]
 *   + t for t < counts[n], -1 where there is no place or no page.  NULL with T
 *   0.
 *   workspace: tension_paged_plan_workspace() bytes. */
int64_t tension_paged_plan_workspace(int64_t N);
int tension_paged_plan(int32_t* table, int64_t table_stride, int64_t table_len,
                       int64_t pages, int64_t page_size, int32_t* free,
                       int32_t* top, const int32_t* lengths,
                       const int32_t* counts, int64_t* slots, int32_t* missing,
                       void* workspace, int64_t N, int64_t T, int64_t window,
                       tension_stream_t stream);

/* The beams of N groups go on from other beams of their group.
 *   layers: `count` caches alike in pages, page_size and table; the first one's
 *     table is read, [N * B, table_len].  Pages of each its own types, Hk heads
 *     of D values.
 *   lengths: device int32 [N], tokens of a group's beams.  parents: device int64
 *     [N,B] (element strides parent_s0, parent_s1): the beam of the group that
 *     beam b goes on from; one outside [0, B) is b itself.  B <= 64.
 *   out_table: device int32 [N * B, table_len], another buffer.  Entries before
 *   lengths[n] / S, whose pages are full, are the parent's.  The others are the
 *   parent's for the first beam that goes on from it; each further one takes
 *   those of a beam that nobody goes on from (in order), and if lengths[n] % S
 *   tokens lie in the first of them, they are copied there, in every layer.
 *   count <= 4096, N * B <= 254200, and Hk * page_size * D <= 2^28. */
int tension_paged_reorder(const tension_paged* layers, int32_t count,
                          int32_t* out_table, int64_t out_stride,
                          const int32_t* lengths, const int64_t* parents,
                          int64_t parent_s0, int64_t parent_s1, int64_t N,
                          int64_t B, int64_t Hk, int64_t D,
                          tension_stream_t stream);

/* ---------------------------------------------------------------------------
 * Beam search: the K best continuations of each group's B beams over a
 * vocabulary of V (no counterpart in the reference, which samples one sequence,
 * model.py:634-650).
 *   logits: [N,B,V] (s[0..2], s[2] == 1), float32, bf16 or f16.
 *   scores: float32 [N,B] (s[0..1]), a beam's log probability so far.
 *   ended: TENSION_U8 [N,B] (s[0..1]) or NULL; a beam with a byte other than 0
 *     has one continuation, token `pad` with the score it has.
 *   score(b, v) = scores[b] + x[b, v] - log sum_u exp x[b, u], taken in 64 bits.
 *   Larger ones come first, of equal ones the lower b; within a beam the order is
 *   that of its logits, then the lower v, also where scores round to one.  Sums of
 *   beams are good to about 1e-14.  A beam whose score is not below infinity or no
 *   number, or whose logits hold a NaN or +infinity or nothing above -infinity,
 *   has none but scores of -infinity.  Where fewer than K are above that, the
 *   lowest places that are not taken follow, with -infinity.
 *   out_scores: float32 [N,K]; tokens, parents: int64 [N,K]; contiguous.
 *   B <= 64, K <= 64, K <= B * V, V <= 2^20.
 *   workspace: tension_beam_select_workspace() bytes (-1 for sizes that the
 *   entry point rejects). */
int64_t tension_beam_select_workspace(int64_t N, int64_t B, int64_t V, int64_t K);
int tension_beam_select(const tension_buf* logits, const tension_buf* scores,
                        const tension_buf* ended, float* out_scores,
                        int64_t* tokens, int64_t* parents, void* workspace,
                        int64_t N, int64_t B, int64_t V, int64_t K, int64_t pad,
                        tension_stream_t stream);

/* Message for the last non-OK return on the calling thread ("" if none). */
const char* tension_last_error(void);

/* Library version string. */
const char* tension_version(void);

/* Kernel family of the last band launch (window / global forward, dq, dkv)
 * on the calling thread: TENSION_KERNEL_* below, or -1 before the first.
 * No counterpart in the reference (its router picks Triton or PyTorch,
 * ops.py:217-219); it lets callers and tests see which path ran. */
enum {
  TENSION_KERNEL_EXACT = 0,      /* one thread per row, any dtype / head dim */
  TENSION_KERNEL_MFMA = 1,       /* dedicated bf16 kernels, head dim 64 */
  TENSION_KERNEL_SPLIT_BF16 = 2, /* split-operand kernels, bf16, head dim 32 / 64 */
  TENSION_KERNEL_SPLIT_F32 = 3,  /* split-operand kernels, float32 Q / K with bf16 V */
  TENSION_KERNEL_SPLIT_F32V = 4, /* split-operand kernels, float32 Q / K / V */
  TENSION_KERNEL_SPLIT_F16 = 5   /* split-operand kernels, float16 Q / K / V */
};
int tension_last_kernel(void);

/* Key groups per workgroup of the last split-kernel forward launched on the
 * calling thread: 1, or 2 where a small grid takes two (0 before the first). */
int tension_last_key_groups(void);

#ifdef __cplusplus
}
#endif

#endif /* TENSION_HIP_H */
