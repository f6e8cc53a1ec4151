// lt_verify.hip -- verification of drafted tokens against the target's probabilities (speculative decoding),
// under the sampler's distributions.
//
// Row r of the target's logits l gives the distribution P_r over its candidates in rank order (larger logit
// first, ties to the lower index, -0 == +0), as lt_sample's:
//   k     the first clamp(top_k, 1, LT_SAMPLE_MAX_K) of them; 1 when temperature <= 0 or 1/temperature is not
//         finite, or when the top logit is not finite
//   w_i   exp((l_i - l_0) / T),  c_i their running sums
//   n     the smallest i + 1 with c_i >= top_p c_{k-1} (k when top_p >= 1);  P_r(i) = w_i / c_{n-1}
// and the drafter's logits give Q_r in the same way.  Draft x of row r is accepted when u Q_r(x) < P_r(x)
// (probability min(1, P/Q)); at the first one that is not, the token is drawn from max(P_r - Q_r, 0), and after
// the last draft from P_r, as the first j in rank order with C_j > u C_end.  Leviathan, Kalman and Matias, "Fast
// inference from transformers via speculative decoding" (ICML 2023): the tokens are then distributed as draws
// from P alone.  Weights and sums are binary64: the result is a choice of whole numbers, and a binary32 sum of
// 1024 weights would move a boundary by 1e-7 of the mass.
//
// Three launches.  (1) k_verify_slices: the candidates of each slice of each row -- the logits are read once,
// into registers; the k-th largest of the threads' maxima bounds the slice's k-th largest from below, so the
// radix select runs over the few keys past that bound.  (2) k_verify_rows: one workgroup a row merges its
// slices, sorts, and writes the distribution and the probability of the row's draft.  (3) k_verify_seqs: one
// workgroup a sequence finds the first draft not accepted and draws the last token.
#include "lt_internal.h"
#include "lt_q8_device.h"
#include "lt_select.h"
#include "lt_paged.h"

using namespace lt;

namespace {

constexpr int kVfMaxSlices = 32;                    // 262144 logits in slices of 8192
typedef unsigned long long u64;

struct VfWs {
  u64* cand;     // [rows][slices][kSmMaxK] (order key << 32) | ~index
  double* p;     // [rows][kSmMaxK] probabilities in rank order
  double* px;    // [rows] probability of the row's draft
  int* id;       // [rows][kSmMaxK]
  int* n;        // [rows] candidates with a probability
  int* cnt;      // [rows][slices]
};

struct VfArgs {
  const float* logits;
  const float* dlogits;
  const int* toks;
  const int* q_start;
  const float* u;
  lt_sample_params* params;
  int B, T, V, slices;
  int* out_tok;
  int* n_out;
  int* len;
  VfWs ws;
};

// The logits of row `row` of the launch (rows past T are the drafter's), its sequence, and its draft (-1: none);
// null where the row takes no part: past the last sequence, or the drafter's row after its last draft.
__device__ const float* vf_row(const VfArgs& A, int row, int* b, int* draft) {
  const int r = row < A.T ? row : row - A.T;
  *b = seq_of_row(A.q_start, A.B, r);
  if (*b < 0) return nullptr;
  const bool last = r + 1 >= A.q_start[*b + 1] || r + 1 >= A.T;
  *draft = last ? -1 : A.toks[r + 1];
  if (row < A.T) return A.logits + (size_t)r * A.V;
  return last ? nullptr : A.dlogits + (size_t)r * A.V;
}

template <int PER>
__global__ __launch_bounds__(kSmThreads) void k_verify_slices(VfArgs A) {
  __shared__ SmShared S;
  const int row = blockIdx.y, sl = blockIdx.x, t = threadIdx.x;
  int b, draft;
  const float* l = vf_row(A, row, &b, &draft);
  if (!l) return;
  const int base = sl * PER * kSmThreads;
  const int nvalid = A.V - base < PER * kSmThreads ? A.V - base : PER * kSmThreads;
  int k = sample_k(A.params + b, A.V);
  if (k > nvalid) k = nvalid;
  uint32_t key[PER];
  bool live[PER];
  float v[PER];
#pragma unroll
  for (int j = 0; j < PER; j++) {
    live[j] = j * kSmThreads + t < nvalid;
    v[j] = live[j] ? l[base + j * kSmThreads + t] : 0.0f;
  }
  uint32_t top[1] = {0u};
#pragma unroll
  for (int j = 0; j < PER; j++) {
    key[j] = order_key(v[j]);
    if (live[j] && key[j] > top[0]) top[0] = key[j];
  }
  // k <= min(threads with a logit, nvalid): at least k keys are at or above the k-th largest maximum
  const bool any[1] = {live[0]};
  int rem;
  const uint32_t bound = radix_select<1>(top, any, k, S, &rem);
#pragma unroll
  for (int j = 0; j < PER; j++) live[j] = live[j] && key[j] >= bound;
  const uint32_t thr = radix_select<PER>(key, live, k, S, &rem);
  // keys equal to thr: all of them, or (when the tie straddles rank k) the rem lowest indices
  bool eq[PER];
  int neq = 0;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    eq[j] = live[j] && key[j] == thr;
    neq += eq[j];
  }
  int eq_total;
  (void)block_excl_scan(neq, S, &eq_total);
  uint32_t nthr = 0u;
  if (eq_total > rem) {
    uint32_t nidx[PER];
#pragma unroll
    for (int j = 0; j < PER; j++) nidx[j] = ~(uint32_t)(base + j * kSmThreads + t);
    int rem2;
    nthr = radix_select<PER>(nidx, eq, rem, S, &rem2);
  }
  int nsel = 0;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    live[j] = live[j] && (key[j] > thr || (eq[j] && ~(uint32_t)(base + j * kSmThreads + t) >= nthr));
    nsel += live[j];
  }
  int total;
  int o = block_excl_scan(nsel, S, &total);
  const size_t at = (size_t)row * A.slices + sl;
  u64* out = A.ws.cand + at * kSmMaxK;
#pragma unroll
  for (int j = 0; j < PER; j++)
    if (live[j]) out[o++] = ((u64)key[j] << 32) | (uint32_t)~(uint32_t)(base + j * kSmThreads + t);
  if (t == 0) A.ws.cnt[at] = k;
}

// Inclusive prefix sum of x over the threads in thread order; *total gets the sum.
__device__ double scan_f64(double x, double* wave_sum, double* total) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();   // wave_sum may still be read from the scan before
  if (lane == 63) wave_sum[wv] = x;
  __syncthreads();
  double before = 0.0, all = 0.0;
#pragma unroll
  for (int w = 0; w < kSmWaves; w++) {
    const double s = wave_sum[w];
    if (w < wv) before += s;
    all += s;
  }
  *total = all;
  return before + x;
}

template <int NS>   // slices at most
__global__ __launch_bounds__(kSmThreads) void k_verify_rows(VfArgs A) {
  __shared__ SmShared S;
  __shared__ u64 s_key[kSmMaxK];
  __shared__ double s_sum[kSmWaves];
  __shared__ double s_c[kSmMaxK];
  __shared__ double s_px;
  __shared__ int s_n;
  const int row = blockIdx.x, t = threadIdx.x;
  int b, draft;
  if (!vf_row(A, row, &b, &draft)) return;
  const lt_sample_params* P = A.params + b;
  const int kc = sample_k(P, A.V);
  int cnt[NS];
  int M = 0;
#pragma unroll
  for (int r = 0; r < NS; r++) {
    cnt[r] = r < A.slices ? A.ws.cnt[(size_t)row * A.slices + r] : 0;
    M += cnt[r];
  }
  const u64* cand = A.ws.cand + (size_t)row * A.slices * kSmMaxK;
  int P2 = 1;
  u64 x = 0ull;   // padding: below every candidate
  if (M <= kSmThreads) {
    // thread t takes the t-th candidate in slice order
    while (P2 < M) P2 <<= 1;
    int r = 0, before = 0, end = 0;
#pragma unroll
    for (int q = 0; q < NS; q++) {
      end += cnt[q];
      if (end <= t) {
        r = q + 1;
        before = end;
      }
    }
    if (t < M) x = cand[(size_t)r * kSmMaxK + (t - before)];
  } else {
    // the first kc of them by a radix select, ties at the threshold by index
    uint32_t key[NS], nidx[NS];
    bool live[NS];
#pragma unroll
    for (int r = 0; r < NS; r++) {
      live[r] = t < cnt[r];
      const u64 c = live[r] ? cand[(size_t)r * kSmMaxK + t] : 0ull;
      key[r] = (uint32_t)(c >> 32);
      nidx[r] = (uint32_t)c;
    }
    int rem;
    const uint32_t thr = radix_select<NS>(key, live, kc, S, &rem);
    bool eq[NS];
    int neq = 0;
#pragma unroll
    for (int r = 0; r < NS; r++) {
      eq[r] = live[r] && key[r] == thr;
      neq += eq[r];
    }
    int eq_total;
    (void)block_excl_scan(neq, S, &eq_total);
    uint32_t nthr = 0u;
    if (eq_total > rem) {
      int rem2;
      nthr = radix_select<NS>(nidx, eq, rem, S, &rem2);
    }
    int nsel = 0;
#pragma unroll
    for (int r = 0; r < NS; r++) {
      live[r] = live[r] && (key[r] > thr || (eq[r] && nidx[r] >= nthr));
      nsel += live[r];
    }
    int total;
    int o = block_excl_scan(nsel, S, &total);
    while (P2 < kc) P2 <<= 1;
    s_key[t] = 0ull;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < NS; r++)
      if (live[r]) s_key[o++] = ((u64)key[r] << 32) | nidx[r];
    __syncthreads();
    x = s_key[t];
    __syncthreads();
  }
  // bitonic network, larger first, one key a thread; partners in the same wave trade by shuffles
  if (P2 > 64 || t < 64)
    for (int size = 2; size <= P2; size <<= 1)
      for (int stride = size >> 1; stride > 0; stride >>= 1) {
        u64 y;
        if (stride >= 64) {
          s_key[t] = x;
          __syncthreads();
          y = s_key[t ^ stride];
          __syncthreads();
        } else {
          y = __shfl_xor(x, stride, 64);
        }
        const bool first = ((t & size) == 0) == ((t & stride) == 0);
        x = first ? (x > y ? x : y) : (x > y ? y : x);
      }
  if (t == 0) {
    s_key[0] = x;
    s_px = 0.0;
  }
  __syncthreads();
  const float l0 = key_logit((uint32_t)(s_key[0] >> 32));
  const int k = __builtin_isfinite(l0) ? kc : 1;
  const double w = t >= k ? 0.0
                   : k == 1 ? 1.0
                            : exp(((double)key_logit((uint32_t)(x >> 32)) - (double)l0) / (double)P->temperature);
  double total;
  const double c = scan_f64(w, s_sum, &total);
  if (t == 0) s_n = k;
  s_c[t] = c;
  __syncthreads();
  const float topp = P->top_p;
  if (topp < 1.0f && t < k && c >= (double)topp * s_c[k - 1]) atomicMin(&s_n, t + 1);
  __syncthreads();
  const int n = s_n;
  const int id = (int)~(uint32_t)x;
  if (t < n) {
    const double p = w / s_c[n - 1];
    A.ws.p[(size_t)row * kSmMaxK + t] = p;
    A.ws.id[(size_t)row * kSmMaxK + t] = id;
    if (id == draft) s_px = p;
  }
  __syncthreads();
  if (t == 0) {
    A.ws.n[row] = n;
    A.ws.px[row] = s_px;
  }
}

// A row's candidates: within the list's room whatever the workspace holds (a row that q_start gives to two
// sequences may have been skipped).
__device__ __forceinline__ int vf_count(const VfArgs& A, int row) {
  const int n = A.ws.n[row];
  return n < 0 ? 0 : n < kSmMaxK ? n : kSmMaxK;
}

__global__ __launch_bounds__(kSmThreads) void k_verify_seqs(VfArgs A) {
  __shared__ double s_sum[kSmWaves];
  __shared__ double s_q[kSmMaxK];
  __shared__ int s_id[kSmMaxK];
  __shared__ int s_first, s_pick;
  const int b = blockIdx.x, t = threadIdx.x;
  const int r0 = A.q_start[b] > 0 ? A.q_start[b] : 0;
  const int r1 = A.q_start[b + 1] < A.T ? A.q_start[b + 1] : A.T;
  const int rows = r1 - r0;
  if (rows <= 0) {
    if (t == 0) A.n_out[b] = 0;
    return;
  }
  lt_sample_params* P = A.params + b;
  auto uniform = [&](int i) {
    if (A.u) return (double)A.u[r0 + i];
    return (double)(philox_x(P->counter + (u64)i, P->seed) >> 8) * 0x1.0p-24;
  };
  if (t == 0) s_first = rows - 1;
  __syncthreads();
  for (int i = t; i < rows - 1; i += kSmThreads) {
    const double q = A.dlogits ? A.ws.px[A.T + r0 + i] : 1.0;
    if (!(uniform(i) * q < A.ws.px[r0 + i])) atomicMin(&s_first, i);
  }
  __syncthreads();
  const int first = s_first, r = r0 + first;
  const bool all = first == rows - 1;
  const int n = vf_count(A, r);
  const double p = t < n ? A.ws.p[(size_t)r * kSmMaxK + t] : 0.0;
  const int id = t < n ? A.ws.id[(size_t)r * kSmMaxK + t] : -1;
  double w = p;
  if (!all) {
    double q = 0.0;
    if (A.dlogits) {
      const int nd = vf_count(A, A.T + r);
      if (t < nd) {
        s_q[t] = A.ws.p[(size_t)(A.T + r) * kSmMaxK + t];
        s_id[t] = A.ws.id[(size_t)(A.T + r) * kSmMaxK + t];
      }
      __syncthreads();
      for (int d = 0; d < nd; d++)
        if (s_id[d] == id) q = s_q[d];
    } else if (id == A.toks[r + 1]) {
      q = 1.0;
    }
    w = p > q ? p - q : 0.0;
  }
  double total;
  double c = scan_f64(w, s_sum, &total);
  if (!(total > 0.0)) c = scan_f64(p, s_sum, &total);   // nothing is left of P: P itself
  if (t == 0) s_pick = n - 1;
  __syncthreads();
  if (t < n && c > uniform(rows - 1) * total) atomicMin(&s_pick, t);
  __syncthreads();
  for (int i = t; i < rows; i += kSmThreads)
    if (i != first) A.out_tok[r0 + i] = i < first ? A.toks[r0 + i + 1] : -1;
  if (t == s_pick) A.out_tok[r] = id;
  if (t == 0) {
    A.n_out[b] = first + 1;
    if (A.len) A.len[b] += first + 1;
    if (!A.u) P->counter += (u64)rows;
  }
}

// Logits a thread holds: 32 when that leaves at least two workgroups a CU, else 8 (more workgroups).
int vf_per(int rows, int V) { return (long long)rows * ((V + 32767) / 32768) >= 512 ? 32 : 8; }

int vf_slices(int rows, int V) {
  const int n = vf_per(rows, V) * kSmThreads;
  return (V + n - 1) / n;
}

VfWs vf_layout(void* ws, int rows, int slices) {
  VfWs w;
  w.cand = (u64*)ws;
  w.p = (double*)(w.cand + (size_t)rows * slices * kSmMaxK);
  w.px = w.p + (size_t)rows * kSmMaxK;
  w.id = (int*)(w.px + rows);
  w.n = w.id + (size_t)rows * kSmMaxK;
  w.cnt = w.n + rows;
  return w;
}

bool vf_sizes(int T, int V) { return T >= 0 && T <= 32767 && V > 0 && V <= kVfMaxSlices * 8 * kSmThreads; }

}  // namespace

extern "C" {

size_t lt_verify_drafts_workspace_size(int T, int V, int drafter) {
  if (!vf_sizes(T, V)) return 0;
  const int rows = drafter ? 2 * T : T;
  const size_t per_row = (size_t)vf_slices(rows, V) * (kSmMaxK * sizeof(u64) + sizeof(int)) +
                         kSmMaxK * (sizeof(double) + sizeof(int)) + sizeof(double) + sizeof(int);
  return rows * per_row;
}

int lt_verify_drafts(lt_ctx* ctx, const float* logits, const float* draft_logits, const int* toks,
                     const int* q_start, const float* u, lt_sample_params* params, int B, int T, int V,
                     int* out_tok, int* n_out, int* len, void* ws, size_t ws_bytes) {
  LT_REQUIRE(logits && toks && q_start && params && out_tok && n_out && ws, "lt_verify_drafts: null argument");
  LT_REQUIRE(B > 0 && B <= 65535 && vf_sizes(T, V), "lt_verify_drafts: B=%d (1 .. 65535) T=%d (0 .. 32767) V=%d (1 .. %d)",
             B, T, V, kVfMaxSlices * 8 * kSmThreads);
  LT_REQUIRE(lt_aligned(params, 8) && lt_aligned(ws, 8) && lt_aligned(logits, 4) && lt_aligned(draft_logits, 4),
             "lt_verify_drafts: params and ws 8-byte, logits 4-byte aligned");
  const size_t need = lt_verify_drafts_workspace_size(T, V, draft_logits != nullptr);
  if (ws_bytes < need)
    return lt_fail(LT_ENOMEM, "lt_verify_drafts: workspace of %zu bytes, needs %zu", ws_bytes, need);
  LT_REQUIRE(ctx, "lt_verify_drafts: null ctx");
  const LtDeviceGuard guard(ctx);
  const int rows = draft_logits ? 2 * T : T;
  const int slices = vf_slices(rows ? rows : 1, V);
  const VfArgs A = {logits, draft_logits, toks, q_start, u, params, B, T, V, slices, out_tok, n_out, len,
                    vf_layout(ws, rows, slices)};
  if (rows) {
    if (vf_per(rows, V) == 32)
      k_verify_slices<32><<<dim3(slices, rows), kSmThreads, 0, ctx->stream>>>(A);
    else
      k_verify_slices<8><<<dim3(slices, rows), kSmThreads, 0, ctx->stream>>>(A);
    if (int rc = lt_check_launch("k_verify_slices")) return rc;
    if (slices <= 8)
      k_verify_rows<8><<<rows, kSmThreads, 0, ctx->stream>>>(A);
    else
      k_verify_rows<kVfMaxSlices><<<rows, kSmThreads, 0, ctx->stream>>>(A);
    if (int rc = lt_check_launch("k_verify_rows")) return rc;
  }
  k_verify_seqs<<<B, kSmThreads, 0, ctx->stream>>>(A);
  return lt_check_launch("k_verify_seqs");
}

}  // extern "C"
