// lt_paged.hip -- the paged KV cache: RoPE and the append of a packed batch of chunks, and the lengths.
#include "lt_paged.h"
#include "lt_q8_device.h"

using namespace lt;

namespace {

// k_rope_append_batch's arithmetic (the same q rows and cache values) with row r the token r - q_start[b] of
// sequence b, at position len[b] + that, and its K and V rows at the page the table gives.  One workgroup a token takes
// the hd / 2 sines and cosines (binary64) once for all heads.  Bound by memory: 1960 tokens of 48 heads of 128 move 69 MB in
// 14.1 us (4.9 TB/s); one token 2.7 us.  qkv may be q_out, so neither pointer is __restrict__.
template <bool kF16>
__global__ __launch_bounds__(256) void k_rope_append_paged(const float* qkv, int row_stride, float* q_out,
                                                           int q_stride, const int* __restrict__ q_start,
                                                           const int* __restrict__ len, int B, int nh,
                                                           const float* __restrict__ freqs, PagedKv C, int* err) {
  __shared__ float s_sn[128], s_cs[128];
  const int r = blockIdx.x, hd = C.hd, half = hd >> 1, nkv = C.nkv;
  const int b = seq_of_row(q_start, B, r);
  if (b < 0) return;
  const int pos = (int)((uint32_t)len[b] + (uint32_t)(r - q_start[b]));   // past 2^31: negative, no page
  const int pg = page_of(C, b, pos);
  if (pg < 0 && err && threadIdx.x == 0) *err = 1;
  for (int j = threadIdx.x; j < half; j += 256) lt_sincosf((float)pos * freqs[j], &s_sn[j], &s_cs[j]);
  __syncthreads();
  const float* row = qkv + (size_t)r * row_stride;
  auto put = [&](void* c, size_t off, float v) {
    if (kF16) ((uint16_t*)c)[off] = lt_f2h(v);
    else ((float*)c)[off] = v;
  };
  for (int i = threadIdx.x; i < (nh + nkv) * half; i += 256) {
    const int hh = i / half, j = i - hh * half;
    const float x1 = row[(size_t)hh * hd + j], x2 = row[(size_t)hh * hd + j + half];
    const float o1 = fmaf(x1, s_cs[j], -(x2 * s_sn[j]));
    const float o2 = fmaf(x1, s_sn[j], x2 * s_cs[j]);
    if (hh < nh) {
      float* q = q_out + (size_t)r * q_stride + (size_t)hh * hd + j;
      q[0] = o1;
      q[half] = o2;
    } else if (pg >= 0) {
      const size_t off = paged_row(C, pg, hh - nh, pos) + j;
      put(C.kc, off, o1);
      put(C.kc, off + half, o2);
    }
  }
  if (pg < 0) return;
  for (int i = threadIdx.x; i < nkv * hd; i += 256) {
    const int h = i / hd, d = i - h * hd;
    put(C.vc, paged_row(C, pg, h, pos) + d, row[(size_t)(nh + nkv) * hd + i]);
  }
}

// each length advanced by its sequence's rows (clamped to maxt)
__global__ __launch_bounds__(256) void k_len_add_rows(int* __restrict__ len, const int* __restrict__ q_start, int B,
                                                      int maxt) {
  for (int b = threadIdx.x; b < B; b += 256) {
    const int L = len[b] + (q_start[b + 1] - q_start[b]);
    len[b] = L < maxt ? L : maxt;
  }
}

}  // namespace

int lt_paged_check(const char* fn, const lt_paged_kv* kv, int nh, PagedKv* out) {
  LT_REQUIRE(kv, "%s: null cache descriptor", fn);
  LT_REQUIRE(kv->kc && kv->vc && kv->table, "%s: null pool or table", fn);
  LT_REQUIRE(lt_aligned(kv->kc, 16) && lt_aligned(kv->vc, 16) && lt_aligned(kv->table, 4),
             "%s: pools 16-byte and table 4-byte aligned", fn);
  LT_REQUIRE(kv->page > 0 && (kv->page & (kv->page - 1)) == 0, "%s: page=%d (a power of two)", fn, kv->page);
  LT_REQUIRE(kv->n_pages > 0 && kv->table_stride > 0 && (long long)kv->table_stride * kv->page <= (1 << 30),
             "%s: n_pages=%d table_stride=%d page=%d (at most 2^30 positions a sequence)", fn, kv->n_pages,
             kv->table_stride, kv->page);
  LT_REQUIRE(kv->nkv > 0 && kv->hd > 0 && kv->hd % 8 == 0 && kv->hd <= 256,
             "%s: nkv=%d hd=%d (hd a multiple of 8, at most 256)", fn, kv->nkv, kv->hd);
  LT_REQUIRE(nh > 0 && nh % kv->nkv == 0 && nh <= 65535, "%s: nh=%d (a multiple of nkv=%d)", fn, nh, kv->nkv);
  LT_REQUIRE(kv->kv_dtype == LT_KV_F32 || kv->kv_dtype == LT_KV_F16, "%s: kv_dtype=%d", fn, kv->kv_dtype);
  *out = {kv->kc, kv->vc, kv->table, kv->table_stride, kv->n_pages, __builtin_ctz(kv->page), kv->nkv, kv->hd};
  return LT_OK;
}

extern "C" {

int lt_rope_append_paged(lt_ctx* ctx, const float* qkv, int row_stride, float* q_out, int q_stride, int T,
                         const int* q_start, const int* len, int B, int nh, const float* freqs,
                         const lt_paged_kv* kv, int* err) {
  const char* fn = "lt_rope_append_paged";
  LT_REQUIRE(qkv && q_out && q_start && len && freqs, "%s: null argument", fn);
  PagedKv C;
  if (int rc = lt_paged_check(fn, kv, nh, &C)) return rc;
  const long long width = (long long)(nh + 2 * C.nkv) * C.hd, qw = (long long)nh * C.hd;
  LT_REQUIRE(T >= 0 && B > 0 && row_stride >= width && q_stride >= qw,
             "%s: T=%d B=%d row_stride=%d (at least %lld) q_stride=%d (at least %lld)", fn, T, B, row_stride, width,
             q_stride, qw);
  LT_REQUIRE((const float*)q_out != qkv || q_stride == row_stride, "%s: in place takes q_stride == row_stride", fn);
  LT_REQUIRE(ctx, "%s: null ctx", fn);
  if (T == 0) return LT_OK;
  const LtDeviceGuard guard(ctx);
  auto kernel = kv->kv_dtype == LT_KV_F16 ? k_rope_append_paged<true> : k_rope_append_paged<false>;
  kernel<<<T, 256, 0, ctx->stream>>>(qkv, row_stride, q_out, q_stride, q_start, len, B, nh, freqs, C, err);
  return lt_check_launch("k_rope_append_paged");
}

int lt_len_add_rows(lt_ctx* ctx, int* len, const int* q_start, int B, int maxt) {
  LT_REQUIRE(len && q_start, "lt_len_add_rows: null argument");
  LT_REQUIRE(B > 0 && maxt > 0, "lt_len_add_rows: B=%d maxt=%d", B, maxt);
  LT_REQUIRE(ctx, "lt_len_add_rows: null ctx");
  const LtDeviceGuard guard(ctx);
  k_len_add_rows<<<1, 256, 0, ctx->stream>>>(len, q_start, B, maxt);
  return lt_check_launch("k_len_add_rows");
}

}  // extern "C"
