// lt_paged.h -- what the launches over a packed batch of chunks share: the batch's rows, the paged cache.
#pragma once

#include "lt_internal.h"

// Makes the context's device current for the launches of one entry point and puts the caller's back.
struct LtDeviceGuard {
  int before = -1;
  explicit LtDeviceGuard(const lt_ctx* ctx) {
    if (hipGetDevice(&before) != hipSuccess || before == ctx->device) before = -1;
    else (void)hipSetDevice(ctx->device);
  }
  ~LtDeviceGuard() {
    if (before >= 0) (void)hipSetDevice(before);
  }
  LtDeviceGuard(const LtDeviceGuard&) = delete;
  LtDeviceGuard& operator=(const LtDeviceGuard&) = delete;
};

namespace lt {

// The sequence that packed row r belongs to (q_start[b] <= r < q_start[b + 1], q_start ascending), or -1.
// Every lane of the wave gives the same r.
__device__ __forceinline__ int seq_of_row(const int* __restrict__ q_start, int B, int r) {
  const int lane = threadIdx.x & 63;
  int b = 0;
  for (int c = 0; c < B; c += 64) {
    const int end = c + lane < B ? q_start[c + lane + 1] : 0x7FFFFFFF;
    const int n = __popcll(__ballot(end <= r));
    b += n;
    if (n < 64) break;
  }
  return b < B && q_start[b] <= r && r < q_start[b + 1] ? b : -1;
}

// One layer's cache as the kernels take it.
struct PagedKv {
  void* kc;
  void* vc;
  const int* table;
  int stride;     // table entries a sequence
  int n_pages;
  int shift;      // log2 of the page
  int nkv, hd;
};

// The page that position pos of sequence b lies in, or -1: past the table's row, or an id outside the pool.
__device__ __forceinline__ int page_of(const PagedKv& C, int b, int pos) {
  const int i = pos >> C.shift;
  if (pos < 0 || i >= C.stride) return -1;
  const int pg = C.table[(size_t)b * C.stride + i];
  return (unsigned)pg < (unsigned)C.n_pages ? pg : -1;
}

// First element of the row of KV head h at slot (pos mod page) of page pg.
__device__ __forceinline__ size_t paged_row(const PagedKv& C, int pg, int h, int pos) {
  return ((((size_t)pg * C.nkv + h) << C.shift) + (pos & ((1 << C.shift) - 1))) * C.hd;
}

}  // namespace lt

// The host's checks of a cache descriptor; 0 and *out filled, or an error with `fn`'s name.
int lt_paged_check(const char* fn, const lt_paged_kv* kv, int nh, lt::PagedKv* out);
