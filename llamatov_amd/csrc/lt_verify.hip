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
// Three launches.  (1) k_verify_maxima reads the logits once and keeps the largest of each group of 4 to 64
// neighbours: the work of a pass over memory.  (2) k_verify_rows, one workgroup a row: the k groups with the
// largest maxima (ties to the lower group) hold the k largest logits -- any other group's logits have k larger ones, one
// in each of those -- and of them only those not below the k-th maximum, so that little more than k logits are read
// again, sorted, and turned into the distribution and the probability of the row's draft.  (3) k_verify_seqs, one
// workgroup a sequence: the first draft not accepted, and the last token.
#include "lt_internal.h"
#include "lt_q8_device.h"
#include "lt_select.h"
#include "lt_paged.h"

using namespace lt;

namespace {

constexpr int kVfMaxV = 262144;
constexpr int kVfGroups = 4 * kSmThreads;           // groups of a row at most: four a thread
constexpr int kVfCand = 4 * kSmThreads;             // logits not below the bound that LDS holds
constexpr int kVfSpan = 8192;                       // logits of a workgroup of k_verify_maxima
typedef unsigned long long u64;

struct VfWs {
  double* p;     // [rows][kSmMaxK] probabilities in rank order
  double* px;    // [rows] probability of the row's draft
  int* id;       // [rows][kSmMaxK]
  int* n;        // [rows] candidates with a probability
  uint32_t* top; // [rows][groups] largest order key of each group
};

struct VfArgs {
  const float* logits;
  const float* dlogits;
  const int* toks;
  const int* q_start;
  const float* u;
  lt_sample_params* params;
  int B, T, V, group, groups;
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

// Largest order keys of groups of GROUP neighbouring logits.  VEC: rows of whole 16-byte words, four logits a lane.
template <int GROUP, bool VEC>
__global__ __launch_bounds__(256) void k_verify_maxima(VfArgs A) {
  int b, draft;
  const float* l = vf_row(A, blockIdx.y, &b, &draft);
  if (!l) return;
  constexpr int PER = VEC ? 4 : 1, U = 8, LANES = GROUP / PER;   // lanes of a group
  uint32_t* top = A.ws.top + (size_t)blockIdx.y * A.groups;
  for (int base = blockIdx.x * kVfSpan; base < (blockIdx.x + 1) * kVfSpan; base += 256 * PER * U) {
    uint32_t key[U];
    float v[U][PER];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = base + (u * 256 + threadIdx.x) * PER;
      if constexpr (VEC) {
        const float4 x = i < A.V ? *(const float4*)(l + i) : make_float4(0, 0, 0, 0);
        v[u][0] = x.x;
        v[u][1] = x.y;
        v[u][2] = x.z;
        v[u][3] = x.w;
      } else {
        v[u][0] = i < A.V ? l[i] : 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = base + (u * 256 + threadIdx.x) * PER;
      key[u] = order_key(v[u][0]);
#pragma unroll
      for (int j = 1; j < PER; j++) {
        const uint32_t kj = order_key(v[u][j]);
        key[u] = kj > key[u] ? kj : key[u];
      }
      if (i >= A.V) key[u] = 0u;   // below or level with every logit's
#pragma unroll
      for (int o = 1; o < LANES; o <<= 1) {
        const uint32_t y = __shfl_xor(key[u], o, 64);
        key[u] = y > key[u] ? y : key[u];
      }
      if ((threadIdx.x & (LANES - 1)) == 0 && i < A.V) top[i / GROUP] = key[u];
    }
  }
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

// Calls f(pair, valid) for the logits of the selected groups, every lane of a wave together; pair orders logits by
// rank, (order key << 32) | ~index.
template <class F>
__device__ __forceinline__ void vf_each(const VfArgs& A, const float* l, const int* grp, int count, F f) {
  const int per = 64 / A.group;            // groups of a wave's load
  const int in = threadIdx.x & (A.group - 1), sub = (threadIdx.x & 63) / A.group;
  constexpr int U = 4;
  for (int g = (threadIdx.x >> 6) * per; g < count; g += kSmWaves * per * U) {
    float v[U];
    int idx[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int gi = g + u * kSmWaves * per + sub;
      idx[u] = gi < count ? grp[gi] * A.group + in : A.V;
      v[u] = idx[u] < A.V ? l[idx[u]] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; u++) f(((u64)order_key(v[u]) << 32) | (uint32_t)~(uint32_t)idx[u], idx[u] < A.V);
  }
}

__global__ __launch_bounds__(kSmThreads) void k_verify_rows(VfArgs A) {
  __shared__ SmShared S;
  __shared__ u64 s_key[kVfCand];
  __shared__ int s_grp[kSmMaxK];
  __shared__ double s_sum[kSmWaves];
  __shared__ double s_c[kSmMaxK];
  __shared__ double s_px;
  __shared__ int s_n, s_count;
  const int row = blockIdx.x, t = threadIdx.x;
  int b, draft;
  const float* l = vf_row(A, row, &b, &draft);
  if (!l) return;
  const lt_sample_params* P = A.params + b;
  const int kc = sample_k(P, A.V);
  // the kc groups of the largest maxima (all groups, if there are no more)
  uint32_t bound = 0u;
  int count;
  {
    uint32_t key[4];
    bool live[4];
    const uint32_t* top = A.ws.top + (size_t)row * A.groups;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      live[j] = j * kSmThreads + t < A.groups;
      key[j] = live[j] ? top[j * kSmThreads + t] : 0u;
    }
    if (t == 0) s_count = 0;
    if (A.groups > kc) {
      int rem;
      bound = radix_select<4>(key, live, kc, S, &rem);
      bool eq[4];
      int neq = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        eq[j] = live[j] && key[j] == bound;
        neq += eq[j];
      }
      int eq_total;
      (void)block_excl_scan(neq, S, &eq_total);
      uint32_t last = 0u;   // ties at the bound: the rem lowest groups
      if (eq_total > rem) {
        uint32_t ng[4];
#pragma unroll
        for (int j = 0; j < 4; j++) ng[j] = ~(uint32_t)(j * kSmThreads + t);
        int rem2;
        last = radix_select<4>(ng, eq, rem, S, &rem2);
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
        live[j] = live[j] && (key[j] > bound || (eq[j] && ~(uint32_t)(j * kSmThreads + t) >= last));
    }
    int sel = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) sel += live[j];
    int o = block_excl_scan(sel, S, &count);
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (live[j]) s_grp[o++] = j * kSmThreads + t;
    __syncthreads();
  }
  // their logits at or above the bound, in any order (the sort settles it)
  auto gather = [&](u64 least) {
    vf_each(A, l, s_grp, count, [&](u64 pair, bool on) {
      on = on && pair >= least;
      const u64 m = __ballot(on);
      if (!m) return;
      int at = 0;
      if ((t & 63) == 0) at = atomicAdd(&s_count, (int)__popcll(m));
      at = __builtin_amdgcn_readfirstlane(at) + (int)__popcll(m & ((1ull << (t & 63)) - 1));
      if (on && at < kVfCand) s_key[at] = pair;
    });
    __syncthreads();
    return s_count;
  };
  int M = gather((u64)bound << 32);
  if (M > kVfCand) {
    // too many of them (runs of large neighbours): the kc-th pair itself, digit by digit over the groups' logits
    u64 prefix = 0ull, mask = 0ull;
    int rem = kc;
#pragma unroll 1
    for (int shift = 56; shift >= 0; shift -= 8) {
      if (t < 256) S.hist[t] = 0;
      __syncthreads();
      vf_each(A, l, s_grp, count, [&](u64 pair, bool on) {
        if (on && (pair & mask) == prefix) atomicAdd(&S.hist[(int)(pair >> shift) & 255], 1);
      });
      __syncthreads();
      if (t < 64) find_digit(S, rem);
      __syncthreads();
      prefix |= (u64)S.sel_digit << shift;
      mask |= 255ull << shift;
      rem = S.sel_rem;
    }
    if (t == 0) s_count = 0;
    __syncthreads();
    M = gather(prefix);
  }
  int P2 = 1;
  u64 x = 0ull;   // padding: below every candidate
  if (M <= kSmThreads) {
    while (P2 < M) P2 <<= 1;
    if (t < M) x = s_key[t];
    __syncthreads();
  } else {
    // the first kc of them by a radix select, ties at the threshold by index
    uint32_t key[4], nidx[4];
    bool live[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      live[j] = j * kSmThreads + t < M;
      const u64 c = live[j] ? s_key[j * kSmThreads + t] : 0ull;
      key[j] = (uint32_t)(c >> 32);
      nidx[j] = (uint32_t)c;
    }
    int rem;
    const uint32_t thr = radix_select<4>(key, live, kc, S, &rem);
    bool eq[4];
    int neq = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      eq[j] = live[j] && key[j] == thr;
      neq += eq[j];
    }
    int eq_total;
    (void)block_excl_scan(neq, S, &eq_total);
    uint32_t nthr = 0u;
    if (eq_total > rem) {
      int rem2;
      nthr = radix_select<4>(nidx, eq, rem, S, &rem2);
    }
    int nsel = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      live[j] = live[j] && (key[j] > thr || (eq[j] && nidx[j] >= nthr));
      nsel += live[j];
    }
    int total;
    int o = block_excl_scan(nsel, S, &total);
    while (P2 < kc) P2 <<= 1;
    s_key[t] = 0ull;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (live[j]) s_key[o++] = ((u64)key[j] << 32) | nidx[j];
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

// Neighbours of a group: at most kVfGroups groups a row, and many more than the 1024 that a row may select.
int vf_group(int V) { return V <= 4 * kVfGroups ? 4 : V <= 16 * kVfGroups ? 16 : V <= 32 * kVfGroups ? 32 : 64; }

int vf_groups(int V) { return (V + vf_group(V) - 1) / vf_group(V); }

VfWs vf_layout(void* ws, int rows, int groups) {
  VfWs w;
  w.p = (double*)ws;
  w.px = w.p + (size_t)rows * kSmMaxK;
  w.id = (int*)(w.px + rows);
  w.n = w.id + (size_t)rows * kSmMaxK;
  w.top = (uint32_t*)(w.n + rows);
  return w;
}

bool vf_sizes(int T, int V) { return T >= 0 && T <= 32767 && V > 0 && V <= kVfMaxV; }

template <bool VEC>
void vf_maxima(const VfArgs& A, dim3 grid, hipStream_t stream) {
  switch (A.group) {
    case 4: k_verify_maxima<4, VEC><<<grid, 256, 0, stream>>>(A); break;
    case 16: k_verify_maxima<16, VEC><<<grid, 256, 0, stream>>>(A); break;
    case 32: k_verify_maxima<32, VEC><<<grid, 256, 0, stream>>>(A); break;
    default: k_verify_maxima<64, VEC><<<grid, 256, 0, stream>>>(A); break;
  }
}

}  // namespace

extern "C" {

size_t lt_verify_drafts_workspace_size(int T, int V, int drafter) {
  if (!vf_sizes(T, V)) return 0;
  const int rows = drafter ? 2 * T : T;
  return rows * (kSmMaxK * (sizeof(double) + sizeof(int)) + sizeof(double) + sizeof(int) + vf_groups(V) * sizeof(uint32_t));
}

int lt_verify_drafts(lt_ctx* ctx, const float* logits, const float* draft_logits, const int* toks,
                     const int* q_start, const float* u, lt_sample_params* params, int B, int T, int V,
                     int* out_tok, int* n_out, int* len, void* ws, size_t ws_bytes) {
  LT_REQUIRE(logits && toks && q_start && params && out_tok && n_out && ws, "lt_verify_drafts: null argument");
  LT_REQUIRE(B > 0 && B <= 65535 && vf_sizes(T, V), "lt_verify_drafts: B=%d (1 .. 65535) T=%d (0 .. 32767) V=%d (1 .. %d)",
             B, T, V, kVfMaxV);
  LT_REQUIRE(lt_aligned(params, 8) && lt_aligned(ws, 8) && lt_aligned(logits, 4) && lt_aligned(draft_logits, 4),
             "lt_verify_drafts: params and ws 8-byte, logits 4-byte aligned");
  const size_t need = lt_verify_drafts_workspace_size(T, V, draft_logits != nullptr);
  if (ws_bytes < need)
    return lt_fail(LT_ENOMEM, "lt_verify_drafts: workspace of %zu bytes, needs %zu", ws_bytes, need);
  LT_REQUIRE(ctx, "lt_verify_drafts: null ctx");
  const LtDeviceGuard guard(ctx);
  const int rows = draft_logits ? 2 * T : T;
  const VfArgs A = {logits, draft_logits, toks, q_start, u, params, B, T, V, vf_group(V), vf_groups(V), out_tok, n_out,
                    len, vf_layout(ws, rows, vf_groups(V))};
  if (rows) {
    const dim3 grid((V + kVfSpan - 1) / kVfSpan, rows);
    if (V % 4 == 0 && lt_aligned(logits, 16) && lt_aligned(draft_logits, 16)) vf_maxima<true>(A, grid, ctx->stream);
    else vf_maxima<false>(A, grid, ctx->stream);
    if (int rc = lt_check_launch("k_verify_maxima")) return rc;
    k_verify_rows<<<rows, kSmThreads, 0, ctx->stream>>>(A);
    if (int rc = lt_check_launch("k_verify_rows")) return rc;
  }
  k_verify_seqs<<<B, kSmThreads, 0, ctx->stream>>>(A);
  return lt_check_launch("k_verify_seqs");
}

}  // extern "C"
