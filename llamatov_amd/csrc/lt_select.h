// lt_select.h -- selection by rank over a workgroup's logits: order-preserving keys, prefix sums, the
// radix select and the counter-based generator shared by the sampler (lt_sample.hip) and the verification of drafts (lt_verify.hip).
#pragma once

#include "lt_internal.h"

namespace lt {

constexpr int kSmThreads = 1024;
constexpr int kSmWaves = kSmThreads / 64;
constexpr int kSmMaxK = LT_SAMPLE_MAX_K;           // 1024 = kSmThreads

static_assert(kSmMaxK == kSmThreads, "one final candidate slot per thread");

// Order-preserving key of a logit: larger logit -> larger key; -0 and +0 share one key.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  if ((b << 1) == 0u) return 0x80000000u;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// Candidates of a draw over V logits: top_k within 1 .. kSmMaxK; greedy (1) when the temperature is
// not positive, or so small that 1/T is not finite (its weights would be exp(0 * inf) = NaN).
__device__ __forceinline__ int sample_k(const lt_sample_params* P, int V) {
  int k = P->top_k;
  k = k < 1 ? 1 : (k > kSmMaxK ? kSmMaxK : k);
  if (!(P->temperature > 0.0f) || !__builtin_isfinite(1.0f / P->temperature)) k = 1;
  return k < V ? k : V;
}

constexpr int kSmCopies = 16;    // pass-0 histogram copies (lane mod 16)
constexpr int kSmCopyStride = 257;   // rows 257 apart: equal digits of different copies in different banks

struct SmShared {
  int hist[256];
  int hist16[kSmCopies * kSmCopyStride];
  int wave_sum[kSmWaves];
  int sel_digit, sel_rem;
};

// Exclusive prefix sum of v over the workgroup's threads in thread order; *total gets the sum.
static __device__ int block_excl_scan(int v, SmShared& S, int* total) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) S.wave_sum[wv] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSmWaves; w++) {
    const int s = S.wave_sum[w];
    before += w < wv ? s : 0;
    all += s;
  }
  __syncthreads();   // wave_sum is reused by the next scan
  *total = all;
  return before + x - v;
}

// After the histogram of this pass is complete: the digit (largest first) at which the count
// of larger-or-equal digits reaches `rem`, and the rank left inside it.  Wave 0 only; lane j
// holds digits 255-4j .. 252-4j.
static __device__ void find_digit(SmShared& S, int rem) {
  const int lane = threadIdx.x & 63;
  int c[4];
#pragma unroll
  for (int q = 0; q < 4; q++) c[q] = S.hist[255 - 4 * lane - q];
  const int mine = c[0] + c[1] + c[2] + c[3];
  int x = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  int run = x - mine;   // elements with a larger digit than this lane's first
#pragma unroll
  for (int q = 0; q < 4; q++) {
    if (run < rem && run + c[q] >= rem) {
      S.sel_digit = 255 - 4 * lane - q;
      S.sel_rem = rem - run;
    }
    run += c[q];
  }
}

// Radix select over N keys per thread (those with live[j]): returns the key T of rank `rem`
// (1 = largest) among them and sets *rem_out to T's rank among the keys equal to T.  BYTES < 4: only the
// leading bytes of T are found and *rem_out is its rank among the keys that share them.
template <int N, int BYTES = 4>
__device__ uint32_t radix_select(const uint32_t (&key)[N], const bool (&live)[N], int rem, SmShared& S,
                                 int* rem_out) {
  uint32_t prefix = 0, mask = 0;
  // pass 0 (the top byte: mostly the exponent, so a few digits hold most keys) counts into
  // 16 copies of the histogram, one per lane mod 16, so lanes of one atomic instruction
  // with the same digit hit different banks; the copies are then summed (integer counts:
  // the same histogram)
#pragma unroll
  for (int i = threadIdx.x; i < kSmCopies * kSmCopyStride; i += kSmThreads) S.hist16[i] = 0;
  __syncthreads();
  {
    int* h = S.hist16 + (threadIdx.x & (kSmCopies - 1)) * kSmCopyStride;
#pragma unroll
    for (int j = 0; j < N; j++)
      if (live[j]) atomicAdd(&h[key[j] >> 24], 1);
  }
  __syncthreads();
  if (threadIdx.x < 256) {
    int c = 0;
#pragma unroll
    for (int q = 0; q < kSmCopies; q++) c += S.hist16[q * kSmCopyStride + threadIdx.x];
    S.hist[threadIdx.x] = c;
  }
#pragma unroll 1
  for (int pass = 0; pass < BYTES; pass++) {
    const int shift = 24 - 8 * pass;
    if (pass > 0) {
      if (threadIdx.x < 256) S.hist[threadIdx.x] = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < N; j++)
        if (live[j] && (key[j] & mask) == prefix) atomicAdd(&S.hist[(key[j] >> shift) & 255u], 1);
    }
    __syncthreads();
    if (threadIdx.x < 64) find_digit(S, rem);
    __syncthreads();
    prefix |= (uint32_t)S.sel_digit << shift;
    mask |= 255u << shift;
    rem = S.sel_rem;
  }
  *rem_out = rem;
  return prefix;
}

// Philox4x32-10 (Salmon et al., SC 2011).
__device__ __forceinline__ uint32_t philox_x(uint64_t counter, uint64_t seed) {
  uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0u, c3 = 0u;
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; r++) {
    if (r) {
      k0 += 0x9E3779B9u;
      k1 += 0xBB67AE85u;
    }
    const uint32_t lo0 = 0xD2511F53u * c0, hi0 = __umulhi(0xD2511F53u, c0);
    const uint32_t lo1 = 0xCD9E8D57u * c2, hi1 = __umulhi(0xCD9E8D57u, c2);
    const uint32_t n0 = hi1 ^ c1 ^ k0, n2 = hi0 ^ c3 ^ k1;
    c0 = n0;
    c1 = lo1;
    c2 = n2;
    c3 = lo0;
  }
  return c0;
}

}  // namespace lt
