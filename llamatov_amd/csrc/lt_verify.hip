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
// neighbours: the work of a pass over memory.  (2) k_verify_rows, one workgroup a row: k groups have a
// maximum at or above the k-th largest of the maxima, so the k largest logits are not below that one and lie in groups
// whose maxima are not either; little more than k logits are read again, sorted, and turned into the distribution and
// the probability of the row's draft.  The k-th maximum's leading 16 bits are bound enough.  (3) k_verify_seqs, one
// workgroup a sequence: the first draft not accepted, and the last token.
//
// Measured at V = 151936, top_k 40: 64 sequences of up to 4 drafts with a drafter's logits 30.6 + 15.0 + 6.5 us (193 MB in
// the first, 6.3 TB/s: bound by memory), one sequence 5.0 + 9.8 + 4.7 (latency); 72 rows of 128256 with 1024 candidates
// 8.6 + 25.2 + 4.8.
#include <type_traits>

#include "lt_internal.h"
#include "lt_q8_device.h"
#include "lt_select.h"
#include "lt_paged.h"

using namespace lt;

namespace {

constexpr int kVfMaxV = 262144;
constexpr int kVfGroups = 4 * kSmThreads;           // groups of a row at most: four a thread
constexpr int kVfCand = 4 * kSmThreads;             // logits not below the bound that LDS holds
constexpr int kVfSpan = 8192;                       // logits of a workgroup of k_verify_maxima: 32 a thread, all asked for at once
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

// Calls f(pairs, valid) for the logits of the selected groups, U * PER of them a lane and every lane of a wave together;
// pairs order logits by rank, (order key << 32) | ~index.
template <bool VEC, class F>
__device__ __forceinline__ void vf_each(const VfArgs& A, const float* l, const int* grp, int count, F f) {
  constexpr int PER = VEC ? 4 : 1, U = VEC ? 4 : 8;
  const int lanes = A.group / PER;         // lanes of a group
  const int per = 64 / lanes;              // groups of a wave's load
  const int in = (threadIdx.x & (lanes - 1)) * PER, sub = (threadIdx.x & 63) / lanes;
  for (int g = (threadIdx.x >> 6) * per; g < count; g += kSmWaves * per * U) {
    float v[U * PER];
    int idx[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int gi = g + u * kSmWaves * per + sub;
      idx[u] = gi < count ? grp[gi] * A.group + in : A.V;
      if constexpr (VEC) {
        const float4 x = idx[u] < A.V ? *(const float4*)(l + idx[u]) : make_float4(0, 0, 0, 0);
        v[4 * u] = x.x;
        v[4 * u + 1] = x.y;
        v[4 * u + 2] = x.z;
        v[4 * u + 3] = x.w;
      } else {
        v[u] = idx[u] < A.V ? l[idx[u]] : 0.0f;
      }
    }
    u64 pair[U * PER];
    bool on[U * PER];
#pragma unroll
    for (int i = 0; i < U * PER; i++) {
      pair[i] = ((u64)order_key(v[i]) << 32) | (uint32_t)~(uint32_t)(idx[i / PER] + i % PER);
      on[i] = idx[i / PER] < A.V;
    }
    f(pair, on);
  }
}

// x of lane ^ S.
template <int S>
__device__ __forceinline__ uint32_t xor_lane(uint32_t x) {
  // quad_perm 1 0 3 2 / 2 3 0 1 / 3 2 1 0, row_half_mirror (lane ^ 7), row_mirror (lane ^ 15)
  auto dpp = [](uint32_t v, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, decltype(ctrl)::value, 0xF, 0xF, true);
  };
  if constexpr (S == 1) return dpp(x, std::integral_constant<int, 0xB1>{});
  else if constexpr (S == 2) return dpp(x, std::integral_constant<int, 0x4E>{});
  else if constexpr (S == 4) return dpp(dpp(x, std::integral_constant<int, 0x1B>{}), std::integral_constant<int, 0x141>{});
  else if constexpr (S == 8) return dpp(dpp(x, std::integral_constant<int, 0x141>{}), std::integral_constant<int, 0x140>{});
  else if constexpr (S == 16) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return threadIdx.x & 16 ? r.x : r.y;
  } else {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return threadIdx.x & 32 ? r.x : r.y;
  }
}

// One stage of a bitonic network over the lanes of a wave, larger first in descending blocks of `size`.
template <int S>
__device__ __forceinline__ u64 sort_stage(u64 x, int size) {
  const u64 y = (u64)xor_lane<S>((uint32_t)(x >> 32)) << 32 | xor_lane<S>((uint32_t)x);
  const bool first = ((threadIdx.x & size) == 0) == ((threadIdx.x & S) == 0);
  return (x > y) == first ? x : y;   // the pairs are distinct, padding apart
}

// The stages of one block size whose partners lie in the same wave.
__device__ __forceinline__ u64 sort_wave(u64 x, int size) {
  if (size >= 64) x = sort_stage<32>(x, size);
  if (size >= 32) x = sort_stage<16>(x, size);
  if (size >= 16) x = sort_stage<8>(x, size);
  if (size >= 8) x = sort_stage<4>(x, size);
  if (size >= 4) x = sort_stage<2>(x, size);
  return sort_stage<1>(x, size);
}

template <bool VEC>
__global__ __launch_bounds__(kSmThreads) void k_verify_rows(VfArgs A) {
  __shared__ SmShared S;
  __shared__ u64 s_key[kVfCand];
  __shared__ int s_grp[kVfGroups];
  __shared__ double s_sum[kSmWaves];
  __shared__ double s_c[kSmMaxK];
  __shared__ double s_px;
  __shared__ int s_n, s_count, s_groups;
  const int row = blockIdx.x, t = threadIdx.x;
  // the groups' maxima, asked for before it is known that the row takes part
  uint32_t key[4];
  bool live[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    live[j] = j * kSmThreads + t < A.groups;
    key[j] = live[j] ? A.ws.top[(size_t)row * A.groups + j * kSmThreads + t] : 0u;
  }
  int b, draft;
  const float* l = vf_row(A, row, &b, &draft);
  if (!l) return;
  const lt_sample_params* P = A.params + b;
  const int kc = sample_k(P, A.V);
  // the groups whose maximum is not below the kc-th largest's leading 16 bits, which is a bound for the kc-th largest
  // logit (all groups, if there are no more than kc)
  uint32_t bound = 0u;
  int count;
  {
    if (t == 0) s_count = s_groups = 0;
    if (A.groups > kc) {
      int rem;
      bound = radix_select<4, 2>(key, live, kc, S, &rem);
#pragma unroll
      for (int j = 0; j < 4; j++) live[j] = live[j] && key[j] >= bound;
    }
    u64 m[4];
    int sel = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      m[j] = __ballot(live[j]);
      sel += (int)__popcll(m[j]);
    }
    __syncthreads();   // the counters are zero
    int o = 0;
    if ((t & 63) == 0 && sel) o = atomicAdd(&s_groups, sel);
    o = __builtin_amdgcn_readfirstlane(o);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (live[j]) s_grp[o + (int)__popcll(m[j] & ((1ull << (t & 63)) - 1))] = j * kSmThreads + t;
      o += (int)__popcll(m[j]);
    }
    __syncthreads();
    count = s_groups;
  }
  // their logits at or above the bound, in any order (the sort settles it)
  auto gather = [&](u64 least) {
    vf_each<VEC>(A, l, s_grp, count, [&](auto& pair, auto& on) {
      constexpr int N = sizeof(on) / sizeof(on[0]);
      u64 m[N];
      int total = 0;
#pragma unroll
      for (int i = 0; i < N; i++) {
        m[i] = __ballot(on[i] && pair[i] >= least);
        total += (int)__popcll(m[i]);
      }
      if (!total) return;
      int at = 0;
      if ((t & 63) == 0) at = atomicAdd(&s_count, total);
      at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
      for (int i = 0; i < N; i++) {
        const int mine = at + (int)__popcll(m[i] & ((1ull << (t & 63)) - 1));
        if ((m[i] >> (t & 63) & 1) && mine < kVfCand) s_key[mine] = pair[i];
        at += (int)__popcll(m[i]);
      }
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
      vf_each<VEC>(A, l, s_grp, count, [&](auto& pair, auto& on) {
        constexpr int N = sizeof(on) / sizeof(on[0]);
        for (int i = 0; i < N; i++)
          if (on[i] && (pair[i] & mask) == prefix) atomicAdd(&S.hist[(int)(pair[i] >> shift) & 255], 1);
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
  // the weight of this thread's candidate, of k
  auto weight = [&](u64 pair, float l0, int k) {
    if (t >= k) return 0.0;
    if (k == 1) return 1.0;
    return exp(((double)key_logit((uint32_t)(pair >> 32)) - (double)l0) / (double)P->temperature);
  };
  int P2 = 1;
  u64 x = 0ull;   // padding: below every candidate
  if (M <= 64) {
    // one wave holds them all: no more waits of the workgroup
    if (t >= 64) return;
    x = t < M ? s_key[t] : 0ull;
    for (int size = 2; size <= 64; size <<= 1) x = sort_wave(x, size);
    const float l0 = key_logit((uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)));
    const int k = __builtin_isfinite(l0) ? kc : 1;
    const double w = weight(x, l0, k);
    double c = w;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(c, o, 64);
      if (t >= o) c += y;
    }
    const float topp = P->top_p;
    const u64 cut = topp < 1.0f ? __ballot(t < k && c >= (double)topp * __shfl(c, k - 1, 64)) : 0ull;
    const int n = cut ? __builtin_ctzll(cut) + 1 : k;
    const double total = __shfl(c, n - 1, 64);
    const int id = (int)~(uint32_t)x;
    const double p = w / total;
    if (t < n) {
      A.ws.p[(size_t)row * kSmMaxK + t] = p;
      A.ws.id[(size_t)row * kSmMaxK + t] = id;
    }
    const u64 at = __ballot(t < n && id == draft);
    const double px = at ? __shfl(p, __builtin_ctzll(at), 64) : 0.0;
    if (t == 0) {
      A.ws.n[row] = n;
      A.ws.px[row] = px;
    }
    return;
  }
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
  // bitonic network, larger first, one key a thread; partners in other waves trade through LDS, in two halves in turn
  {
    int half = 0;
    for (int size = 2; size <= P2; size <<= 1) {
      for (int stride = size >> 1; stride >= 64; stride >>= 1) {
        s_key[half + t] = x;
        __syncthreads();
        const u64 y = s_key[half + (t ^ stride)];
        half ^= kSmThreads;
        const bool first = ((t & size) == 0) == ((t & stride) == 0);
        x = (x > y) == first ? x : y;
      }
      x = sort_wave(x, size);
    }
  }
  __syncthreads();
  if (t == 0) {
    s_key[0] = x;
    s_px = 0.0;
  }
  __syncthreads();
  const float l0 = key_logit((uint32_t)(s_key[0] >> 32));
  const int k = __builtin_isfinite(l0) ? kc : 1;
  const double w = weight(x, l0, k);
  double total;
  const double c = scan_f64(w, s_sum, &total);
  if (t == 0) s_n = k;
  s_c[t] = c;
  __syncthreads();
  const float topp = P->top_p;
  if (topp < 1.0f) {
    const u64 hit = __ballot(t < k && c >= (double)topp * s_c[k - 1]);
    if (hit && (t & 63) == __builtin_ctzll(hit)) atomicMin(&s_n, t + 1);
  }
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
__device__ __forceinline__ int vf_count(int n) { return n < 0 ? 0 : n < kSmMaxK ? n : kSmMaxK; }

constexpr int kSeqThreads = 256, kSeqWaves = kSeqThreads / 64, kSeqPer = kSmMaxK / kSeqThreads;

// Inclusive prefix sums of four values a thread, in thread order; *total gets the sum.
__device__ __forceinline__ void scan4_f64(const double (&w)[kSeqPer], double (&c)[kSeqPer], double* wave_sum, double* total) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  c[0] = w[0];
#pragma unroll
  for (int j = 1; j < kSeqPer; j++) c[j] = c[j - 1] + w[j];
  double x = c[kSeqPer - 1];
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
  for (int v = 0; v < kSeqWaves; v++) {
    if (v < wv) before += wave_sum[v];
    all += wave_sum[v];
  }
  const double up = __shfl_up(x, 1, 64);
  before += lane ? up : 0.0;
#pragma unroll
  for (int j = 0; j < kSeqPer; j++) c[j] += before;
  *total = all;
}

__global__ __launch_bounds__(kSeqThreads) void k_verify_seqs(VfArgs A) {
  __shared__ double s_sum[kSeqWaves];
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
  const double u_last = uniform(rows - 1);
  __syncthreads();
  for (int i = t; i < rows - 1; i += kSeqThreads) {
    const double q = A.dlogits ? A.ws.px[A.T + r0 + i] : 1.0;
    if (!(uniform(i) * q < A.ws.px[r0 + i])) atomicMin(&s_first, i);
  }
  __syncthreads();
  const int first = s_first, r = r0 + first;
  const bool all = first == rows - 1, drafter = !all && A.dlogits;
  const int n = vf_count(A.ws.n[r]), nd = drafter ? vf_count(A.ws.n[A.T + r]) : 0;
  const int draft = all ? -1 : A.toks[r + 1];
  double p[kSeqPer], w[kSeqPer], c[kSeqPer];
  int id[kSeqPer];
#pragma unroll
  for (int j = 0; j < kSeqPer; j++) {
    const int i = t * kSeqPer + j;
    p[j] = i < n ? A.ws.p[(size_t)r * kSmMaxK + i] : 0.0;
    id[j] = i < n ? A.ws.id[(size_t)r * kSmMaxK + i] : -1;
    // without a drafter's logits Q has all its mass on the draft
    w[j] = !all && !drafter && id[j] == draft ? 0.0 : p[j];
  }
  if (drafter) {
    for (int i = t; i < nd; i += kSeqThreads) {
      s_q[i] = A.ws.p[(size_t)(A.T + r) * kSmMaxK + i];
      s_id[i] = A.ws.id[(size_t)(A.T + r) * kSmMaxK + i];
    }
    __syncthreads();
    int at[kSeqPer] = {-1, -1, -1, -1};
    for (int d = 0; d < nd; d++) {
      const int x = s_id[d];
#pragma unroll
      for (int j = 0; j < kSeqPer; j++) at[j] = x == id[j] ? d : at[j];
    }
#pragma unroll
    for (int j = 0; j < kSeqPer; j++)
      if (at[j] >= 0) w[j] = p[j] > s_q[at[j]] ? p[j] - s_q[at[j]] : 0.0;
  }
  double total;
  scan4_f64(w, c, s_sum, &total);
  if (!(total > 0.0)) scan4_f64(p, c, s_sum, &total);   // nothing is left of P: P itself
  if (t == 0) s_pick = n - 1;
  __syncthreads();
  // the sums do not fall: the first candidate past the goal is the first such lane's first
  int mine = kSeqPer;
#pragma unroll
  for (int j = kSeqPer - 1; j >= 0; j--)
    if (t * kSeqPer + j < n && c[j] > u_last * total) mine = j;
  const u64 hit = __ballot(mine < kSeqPer);
  if (hit && (t & 63) == __builtin_ctzll(hit)) atomicMin(&s_pick, t * kSeqPer + mine);
  __syncthreads();
  for (int i = t; i < rows; i += kSeqThreads)
    if (i != first) A.out_tok[r0 + i] = i < first ? A.toks[r0 + i + 1] : -1;
#pragma unroll
  for (int j = 0; j < kSeqPer; j++)
    if (t * kSeqPer + j == s_pick) A.out_tok[r] = id[j];
  if (t == 0) {
    A.n_out[b] = first + 1;
    if (A.len) A.len[b] += first + 1;
    if (!A.u) P->counter += (u64)rows;
  }
}

// Neighbours of a group: at most kVfGroups groups a row (four a thread), and as many as that allows, so that a group that
// is selected brings few logits with it.
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
  LT_REQUIRE(logits && toks && q_start && params && out_tok && n_out && (ws || T == 0), "lt_verify_drafts: null argument");
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
    const bool vec = V % 4 == 0 && lt_aligned(logits, 16) && lt_aligned(draft_logits, 16);
    if (vec) vf_maxima<true>(A, grid, ctx->stream);
    else vf_maxima<false>(A, grid, ctx->stream);
    if (int rc = lt_check_launch("k_verify_maxima")) return rc;
    if (vec) k_verify_rows<true><<<rows, kSmThreads, 0, ctx->stream>>>(A);
    else k_verify_rows<false><<<rows, kSmThreads, 0, ctx->stream>>>(A);
    if (int rc = lt_check_launch("k_verify_rows")) return rc;
  }
  k_verify_seqs<<<B, kSeqThreads, 0, ctx->stream>>>(A);
  return lt_check_launch("k_verify_seqs");
}

}  // extern "C"
