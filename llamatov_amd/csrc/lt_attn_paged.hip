// lt_attn_paged.hip -- attention of a packed batch of chunks over a paged KV cache.
//
// For one KV head, a sequence's chunk is n * rep query rows (rep = nh / nkv heads share the KV head): row r is token
// r / rep, head r % rep.  A workgroup takes a tile of those rows and a range of keys; key tiles go through LDS by
// direct loads while the tile before is computed, and the softmax runs over them in registers:
//   S^T = K Q^T       keys x rows, so that a lane holds one row's scores and row statistics stay in the lane's column
//   m, z, P           base-2 exponentials of the scores less a running reference
//   O^T += V^T P^T    P goes from the first product's result registers into the second's operand registers as it is
//                     (the key order inside a product is free, and V is read in the same order)
//
// An fp16 cache runs on the 16x16x32 fp16 matrix instruction.  Its products are exact and its sums fp32, and
// q and P are given to it as two binary16 terms each (x = hi + lo, |x - hi - lo| <= 2^-22 |x|), q scaled by a power of
// two to its row's size so that neither term is lost below binary16's range: two products a term instead of the 16 that
// the fp32 instruction would take.  An fp32 cache runs on the 16x16x4 fp32 instruction.
//
// Measured (fp16, 32 query heads over 8 of 128): one token over 32768 positions 23.8 us and the join 4.8 (134 MB, 5.6 TB/s;
// bound by memory); 64 sequences of 512 to 4096 positions 124 us (614 MB, 4.95 TB/s); 2048 tokens over 14336 797 to 852 us (515
// GFLOP, 1.26 PFLOP/s of the two-term products; matrix pipes busy 62% of the time at 1.93 GHz, vector instructions 47%); a
// short context 4.9 us (latency).  fp32, 14 heads over 2 of 64, 866 rows with a window of 512: 29.6 us and the join 9.2.
#include "lt_paged.h"
#include "lt_q8_device.h"

using namespace lt;

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;

constexpr float kLog2e = 1.4426950408889634f;
// P is held as 2^kPShift exp2(score - reference), the reference moved once a score passes it by kSlack.  For binary16
// terms at most 2^15, and a weight of 2^-32 of the largest still has a term; in fp32 at most 1, so that values near the
// type's largest do not overflow
constexpr float kSlack = 8.0f;
template <bool F16>
constexpr float kPShift = F16 ? 7.0f : -kSlack;
constexpr int kMaxSplits = 128, kCus = 256;

__device__ const u32x4 g_zero16 = {0, 0, 0, 0};   // what a row without a page reads

// x / d for any 32-bit x by a multiplication (Granlund and Montgomery, "Division by invariant integers using
// multiplication", PLDI 1994).
struct Div {
  uint32_t m, s1, s2;
};
inline Div make_div(uint32_t d) {
  int l = 0;
  while ((1ull << l) < d) l++;
  return {(uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1), (uint32_t)(l < 1 ? l : 1), (uint32_t)(l < 1 ? 0 : l - 1)};
}
__device__ __forceinline__ int div_by(const Div& D, int x) {
  const uint32_t hi = __umulhi((uint32_t)x, D.m);
  return (int)((((uint32_t)x - hi) >> D.s1) + hi >> D.s2);
}

struct AttnArgs {
  const float* q;
  int q_stride;
  const int* q_start;
  const int* len;
  int B, T, nh, rep;
  PagedKv C;
  float* out;
  float scale;       // |scale|; its sign goes into q
  float sign;
  int window;
  int* err;
  int vec;           // q rows are 16-byte aligned
  int chunk, nsplit; // keys a split, splits in the grid
  AttnWs ws;
  Div by_rep, by_chunk, by_nkv, by_nh;
};

// One tile of a sequence's rows and the keys it attends.
struct Tile {
  int q0;            // the sequence's first row in the batch
  int row0, rows;    // packed rows of the sequence from row0, and its count of them
  int past, cap;
  int lo, hi;        // keys any of its rows attends
  int kbeg;          // lo down to a multiple of the key tile
  int nact;          // splits that take part
};

__device__ __forceinline__ int key_lo(const AttnArgs& A, int past, int t) {
  const int p1 = past + t + 1;
  return A.window > 0 && p1 > A.window ? p1 - A.window : 0;
}
__device__ __forceinline__ int key_hi(int past, int cap, int t) {
  const int p1 = past + t + 1;
  return p1 < cap ? p1 : cap;
}

// Ints that no kernel of this file writes, for loads on the scalar side.
typedef const __attribute__((address_space(4))) int const_int;
__device__ __forceinline__ const_int* scalar_ints(const int* p) { return (const_int*)(uintptr_t)p; }

// Rows q_start[b] .. of sequence b, none where the two do not make sense.
__device__ __forceinline__ int rows_of(int s, int e, int T) { return s >= 0 && e > s && e <= T ? e - s : 0; }

__device__ __forceinline__ Tile tile_of(const AttnArgs& A, int q0, int q1, int L, int tile, int tm, int kt) {
  Tile X;
  X.q0 = q0;
  X.cap = A.C.stride << A.C.shift;
  X.past = L < 0 ? 0 : L < X.cap ? L : X.cap;
  X.row0 = tile * tm;
  X.rows = rows_of(q0, q1, A.T) * A.rep;
  const int last = X.row0 + tm < X.rows ? X.row0 + tm - 1 : X.rows - 1;
  X.lo = key_lo(A, X.past, div_by(A.by_rep, X.row0));
  X.hi = key_hi(X.past, X.cap, div_by(A.by_rep, last));
  X.kbeg = X.lo & ~(kt - 1);
  const int n = X.hi > X.kbeg ? div_by(A.by_chunk, X.hi - X.kbeg + A.chunk - 1) : 1;
  X.nact = n < A.nsplit ? n : A.nsplit;
  return X;
}

// Sequence and tile (the heaviest of a sequence first) of tile x of the batch; b = -1 past the last.
__device__ __forceinline__ void find_tile(const AttnArgs& A, int x, int tm, int* b, int* tile) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int c = 0; c < A.B; c += 64) {
    int n = 0;
    if (c + lane < A.B) {
      n = (rows_of(A.q_start[c + lane], A.q_start[c + lane + 1], A.T) * A.rep + tm - 1) / tm;   // tm: a constant
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(sum, o, 64);
      if (lane >= o) sum += y;
    }
    const uint64_t past = __ballot(base + sum > x);
    if (past) {
      const int f = __builtin_ctzll(past);
      const int nf = __builtin_amdgcn_readlane(n, f), sf = __builtin_amdgcn_readlane(sum, f);
      *b = c + f;
      *tile = nf - 1 - (x - base - (sf - nf));
      return;
    }
    base += __builtin_amdgcn_readlane(sum, 63);
  }
  *b = -1;
}

__device__ __forceinline__ float sum_over_groups(float a) {
  const uint32_t u = __float_as_uint(a);
  const u32x2 x = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t v = __float_as_uint(__uint_as_float(x.x) + __uint_as_float(x.y));
  const u32x2 y = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return __uint_as_float(y.x) + __uint_as_float(y.y);
}

// Matrix results complete before another basic block reads them (settle's reason in lt_q8_device.h): every
// accumulator is tied to a wait in the block that computed it.
template <int D, int N>
__device__ __forceinline__ void settle_all(f32x4 (&o)[D][N]) {
  static_assert(N == 1 || N == 2, "settle_all: accumulators");
#pragma unroll
  for (int d = 0; d + 2 <= D; d += 2) {
    if constexpr (N == 1) asm volatile("" : "+v"(o[d][0]), "+v"(o[d + 1][0]));
    else asm volatile("" : "+v"(o[d][0]), "+v"(o[d][1]), "+v"(o[d + 1][0]), "+v"(o[d + 1][1]));
  }
  if constexpr (N == 1) asm volatile("s_nop 15" : "+v"(o[D - 1][0]));
  else asm volatile("s_nop 15" : "+v"(o[D - 1][0]), "+v"(o[D - 1][1]));
}

// a less its binary16 rounding in the low (high) half of h, exactly.
__device__ __forceinline__ float rest_lo(uint32_t h, float a) {
  float r;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(a));
  return r;
}
__device__ __forceinline__ float rest_hi(uint32_t h, float a) {
  float r;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(a));
  return r;
}

// Two fp32 values as two binary16 terms each.
__device__ __forceinline__ void split2(float a, float b, uint32_t* hi, uint32_t* lo) {
  const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
  *hi = h;
  *lo = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){rest_lo(h, a), rest_hi(h, b)}, f16x2));
}

// Elements d .. d + 3 of packed row `row` of KV head h: the result, or the split's part of it.
__device__ __forceinline__ void put_row(const AttnArgs& A, const Tile& X, int h, int sp, int row, int d, f32x4 o,
                                        float m, float z) {
  const int t = div_by(A.by_rep, row), head = h * A.rep + (row - t * A.rep), hd = A.C.hd;
  const size_t r = (size_t)(X.q0 + t) * A.nh + head;
  if (X.nact == 1) {
    const bool any = key_hi(X.past, X.cap, t) > key_lo(A, X.past, t);
    const float inv = 1.0f / z;
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = any ? o[e] * inv : 0.0f;
    float* to = A.out + r * hd + d;
    if (A.vec) {
      *(f32x4*)to = o;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) to[e] = o[e];
    }
  } else {
    const size_t at = r * A.nsplit + sp;
    *(f32x4*)(A.ws.o + at * hd + d) = o;
    if (d == 0) {
      A.ws.m[at] = m;
      A.ws.z[at] = z;
    }
  }
}

// A tile's rows over keys k0 .. k1 - 1 by the formula itself, a wave a row: lane j scores key j of each 64, then sums
// the values' dimensions 4 j ..  Taken where the matrix products met what is not finite: a masked value of infinity times a
// weight of zero, or an infinity times two terms of different signs, is NaN there and nothing or an infinity here.
template <int TM, int WAVES, bool F16>
__device__ __forceinline__ void rows_one_by_one(const AttnArgs& A, const Tile& X, int b, int h, int k0, int k1, int sp) {
  const PagedKv& C = A.C;
  const int lane = threadIdx.x & 63, hd = C.hd;
  auto at = [](const void* c, size_t i) { return F16 ? lt_h2f(((const uint16_t*)c)[i]) : ((const float*)c)[i]; };
  for (int i = threadIdx.x >> 6; i < TM && X.row0 + i < X.rows; i += WAVES) {
    const int row = X.row0 + i, t = div_by(A.by_rep, row);
    const float* q = A.q + (size_t)(X.q0 + t) * A.q_stride + (size_t)(h * A.rep + row - t * A.rep) * hd;
    int lo = key_lo(A, X.past, t), end = key_hi(X.past, X.cap, t);
    lo = lo < k0 ? k0 : lo;
    end = end > k1 ? k1 : end;
    float m = -__builtin_inff(), z = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    for (int k = lo; k < end && !(z != z); k += 64) {   // a row with a NaN among its weights is NaN
      const int key = k + lane;
      const int pg = key < end ? page_of(C, b, key) : -1;
      float s = -__builtin_inff();
      if (key < end) {
        s = 0.0f;
        const size_t kr = pg >= 0 ? paged_row(C, pg, h, key) : 0;
#pragma unroll 1
        for (int d = 0; pg >= 0 && d < hd; d++) s = fmaf(q[d], at(C.kc, kr + d), s);
        s = s * (A.scale * A.sign * kLog2e);
      }
      float mt = s;
#pragma unroll
      for (int x = 32; x; x >>= 1) mt = fmaxf(mt, __shfl_xor(mt, x, 64));
      const float mn = fmaxf(m, mt), mu = mn == -__builtin_inff() ? 0.0f : mn;
      const float a = __builtin_amdgcn_exp2f(m - mu), p = __builtin_amdgcn_exp2f(s - mu + kPShift<F16>);
      float zt = p;
#pragma unroll
      for (int x = 32; x; x >>= 1) zt += __shfl_xor(zt, x, 64);
      z = fmaf(z, a, zt);
      m = mn;
      o *= a;
#pragma unroll 1
      for (int j = 0; j < 64 && k + j < end; j++) {
        const int pj = __shfl(pg, j, 64);
        const float w = __shfl(p, j, 64);
        if (pj < 0 || lane * 4 >= hd) continue;
        const size_t vr = paged_row(C, pj, h, k + j) + lane * 4;
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = fmaf(w, at(C.vc, vr + e), o[e]);
      }
    }
    if (z != z) o = (f32x4){z, z, z, z};
    if (lane * 4 < hd) put_row(A, X, h, sp, row, lane * 4, o, m, z);
  }
}

// HDP: head dim rounded up to 64, 128 or 256.  A wave takes NT tiles of 16 rows; RW waves take different rows and
// share their keys' LDS, KW groups of RW waves take different key tiles (of KT keys) of the same rows.
template <int HDP, int NT, int RW, int KW, int KT, bool F16>
struct Cfg {
  static constexpr int kWaves = RW * KW, kThreads = 64 * kWaves, kTM = 16 * NT * RW;
  static constexpr int kRowB = HDP * (F16 ? 2 : 4), kCpr = kRowB / 16, kTileB = KT * kRowB, kStageB = 2 * kTileB;
  static constexpr int kRing = KW * 2 * kStageB;
  static constexpr int kAccStride = HDP + 4;
  static constexpr int kMerge = KW > 1 ? kWaves * NT * 16 * (kAccStride + 2) * 4 : 0;
  static constexpr int kLds = kRing > kMerge ? kRing : kMerge;
  static constexpr int kLoads = KT * kCpr / (64 * RW);   // direct loads of a wave for K, and for V
  static_assert(KT * kCpr % (64 * RW) == 0 && kLds <= 160 * 1024, "configuration");
};

// LDS slot of 16-byte chunk c of key row r is c ^ swz(r): 16 rows' equal chunks then lie in different banks.
template <int CPR>
__device__ __forceinline__ int swz(int r) {
  return CPR >= 16 ? (r & 15) : ((r >> 1) & 7);
}

template <bool F16>
struct VFrag {
  typedef u32x2 T;
};
template <>
struct VFrag<false> {
  typedef uint32_t T;
};

__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Split sp of one tile of sequence b, KV head h; false where nothing was written because a result is not a number.
template <int HDP, int NT, int RW, int KW, int KT, bool F16>
__device__ __forceinline__ bool attend(const AttnArgs& A, const Tile& X, int b, int h, int sp, uint8_t* smem) {
  using G = Cfg<HDP, NT, RW, KW, KT, F16>;
  constexpr int CPR = G::kCpr, MT = KT / 16, DT = HDP / 16, KC = F16 ? HDP / 32 : HDP / 16;
  const PagedKv& C = A.C;
  const int lane = threadIdx.x & 63, n16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rw = wave % RW, kw = wave / RW;
  const int k0 = X.kbeg + sp * A.chunk;
  const int k1 = sp == X.nact - 1 ? X.hi : k0 + A.chunk;
  if (X.past + div_by(A.by_rep, X.rows - 1) >= X.cap && A.err && threadIdx.x == 0) *A.err = 1;

  // ---- key tiles into LDS -------------------------------------------------------------------------
  // A direct load takes 64 chunks of 16 bytes: kRpi rows of the tile, from one page unless pages are smaller than that.
  constexpr int kRpi = 64 / CPR;
  const uint32_t ring = (uint32_t)(uintptr_t)(lds_u8*)smem + kw * 2 * G::kStageB;
  const uint32_t row_b = C.hd * (F16 ? 2 : 4);
  const ptrdiff_t v_off = (ptrdiff_t)((uintptr_t)C.vc - (uintptr_t)C.kc);
  const_int* table = scalar_ints(C.table + (size_t)b * C.stride);
  const int slots = (1 << C.shift) - 1;
  // the pages of a tile's loads, read on the scalar side a tile ahead
  struct Pages {
    int id[G::kLoads];
  };
  auto look_up = [&](int k) {
    Pages P;
#pragma unroll
    for (int i = 0; i < G::kLoads; i++) {
      const int key = k + (i * RW + rw) * kRpi;
      P.id[i] = table[(key < k1 ? key : k1 - 1) >> C.shift];
    }
    return P;
  };
  auto load16 = [](uint32_t to, const uint8_t* base, uint32_t off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base)
                 : "memory", "m0");
  };
  auto load16_far = [](uint32_t to, const uint8_t* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory", "m0");
  };
  auto stage = [&](int k, const Pages& P, int buf) {
    int ln = lane;
    asm volatile("" : "+v"(ln));   // what follows from the lane is formed here, not kept over the loop
    const uint32_t to = ring + buf * G::kStageB + rw * 1024;
    bool fast = k >= X.lo && k + KT <= k1 && row_b == G::kRowB && slots + 1 >= kRpi;
#pragma unroll
    for (int i = 0; i < G::kLoads; i++) fast = fast && (uint32_t)P.id[i] < (uint32_t)C.n_pages;
    if (fast) {
#pragma unroll
      for (int i = 0; i < G::kLoads; i++) {
        const int r0 = (i * RW + rw) * kRpi;
        const uint8_t* kb = (const uint8_t*)C.kc +
                            ((((size_t)P.id[i] * C.nkv + h) << C.shift) + ((k + r0) & slots)) * G::kRowB;
        const uint32_t off = (ln / CPR) * G::kRowB + (((ln % CPR) ^ swz<CPR>(r0 + ln / CPR)) << 4);
        load16(to + i * RW * 1024, kb, off);
        load16(to + i * RW * 1024 + G::kTileB, kb + v_off, off);
      }
      return;
    }
    // rows past either end of the keys take the nearest one's (their weights are zero), chunks past hd and rows
    // without a page zeros
#pragma unroll
    for (int i = 0; i < G::kLoads; i++) {
      const int row = (i * RW + rw) * kRpi + ln / CPR, c = (ln % CPR) ^ swz<CPR>(row);
      int key = k + row;
      key = key >= k1 ? k1 - 1 : key;
      key = key < X.lo ? X.lo : key;
      const int pg = page_of(C, b, key);
      if (pg < 0 && A.err) *A.err = 1;
      const bool on = pg >= 0 && c * 16 < (int)row_b;
      const uint8_t* kp = (const uint8_t*)C.kc + ((((size_t)(on ? pg : 0) * C.nkv + h) << C.shift) + (key & slots)) * row_b + c * 16;
      load16_far(to + i * RW * 1024, on ? kp : (const uint8_t*)&g_zero16);
      load16_far(to + i * RW * 1024 + G::kTileB, on ? kp + v_off : (const uint8_t*)&g_zero16);
    }
  };
  const int ntiles = k1 > k0 ? (k1 - k0 + KT - 1) / KT : 0, iters = (ntiles + KW - 1) / KW;
  auto tile_key = [&](int it) { return k0 + (it * KW + kw) * KT; };
  // A wave that keeps its own tiles has two on their way; waves that share theirs meet once a tile and have one.
  constexpr bool kOwn = RW == 1;
  Pages next = {};
  if (iters > 0) {
    next = look_up(tile_key(0));
    stage(tile_key(0), next, 0);
    next = look_up(tile_key(1));
    if (kOwn && iters > 1) {
      stage(tile_key(1), next, 1);
      next = look_up(tile_key(2));
    }
  }

  // this lane's rows
  const int rw0 = X.row0 + rw * 16 * NT;
  int hi[NT], lo[NT];
  float f[NT];
  u32x4 qh[NT][KC], ql[F16 ? NT : 1][F16 ? KC : 1];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const int row = rw0 + nt * 16 + n16;
    const bool on = row < X.rows;
    const int t = div_by(A.by_rep, row);
    hi[nt] = on ? key_hi(X.past, X.cap, t) : 0;
    lo[nt] = on ? key_lo(A, X.past, t) : 0;
    const float* q = A.q + (size_t)(X.q0 + (on ? t : 0)) * A.q_stride + (size_t)(h * A.rep + (on ? row - t * A.rep : 0)) * C.hd;
    constexpr int W = F16 ? 8 : 4;   // values of a lane per step
    float v[KC][W];
#pragma unroll
    for (int c = 0; c < KC; c++) {
      const int d = (4 * c + g) * W;
      if (on && d < C.hd) {
        if (A.vec) {
#pragma unroll
          for (int j = 0; j < W; j += 4) *(float4*)&v[c][j] = *(const float4*)(q + d + j);
        } else {
#pragma unroll
          for (int j = 0; j < W; j++) v[c][j] = q[d + j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < W; j++) v[c][j] = 0.0f;
      }
    }
    if constexpr (F16) {
      // the row's largest value scaled to [2^14, 2^15)
      float mx = 0.0f;
#pragma unroll
      for (int c = 0; c < KC; c++)
#pragma unroll
        for (int j = 0; j < W; j++) mx = fmaxf(mx, fabsf(v[c][j]));
      int ex = (int)(__float_as_uint(max_over_groups(mx)) >> 23);
      ex = ex < 20 ? 20 : ex > 254 ? 254 : ex;
      const float up = __uint_as_float((uint32_t)(127 + 14 + 127 - ex) << 23) * A.sign;
      f[nt] = A.scale * kLog2e * __uint_as_float((uint32_t)(ex - 14) << 23);
#pragma unroll
      for (int c = 0; c < KC; c++)
#pragma unroll
        for (int j = 0; j < W; j += 2) {
          uint32_t a, e;
          split2(v[c][j] * up, v[c][j + 1] * up, &a, &e);
          qh[nt][c][j / 2] = a;
          ql[nt][c][j / 2] = e;
        }
    } else {
      f[nt] = A.scale * kLog2e;
#pragma unroll
      for (int c = 0; c < KC; c++)
#pragma unroll
        for (int j = 0; j < W; j++) qh[nt][c][j] = __float_as_uint(v[c][j] * A.sign);
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; nt++) f[nt] = fmaxf(f[nt], 0x1.0p-126f);   // a scale of zero: scores of -inf stay that
  // the wave's rows as a whole
  const int wrows = rw0 + 16 * NT < X.rows ? 16 * NT : X.rows - rw0;
  const int tw0 = div_by(A.by_rep, rw0), tw1 = div_by(A.by_rep, rw0 + (wrows > 0 ? wrows : 1) - 1);
  const int whi0 = key_hi(X.past, X.cap, tw0), whi1 = wrows > 0 ? key_hi(X.past, X.cap, tw1) : 0;
  const int wlo0 = key_lo(A, X.past, tw0), wlo1 = key_lo(A, X.past, tw1);

  // ---- one key tile -------------------------------------------------------------------------------
  f32x4 acc[DT][NT];
  float mref[NT], z[NT];
  const uint32_t ka0 = ring + n16 * G::kRowB + ((g ^ swz<CPR>(n16)) << 4);                        // step c: ^ (c << 6)
  const int vr = 4 * g + (n16 >> 2);
  const uint32_t va0 = ring + G::kTileB +
                       (F16 ? vr * G::kRowB + ((((n16 >> 1) & 1) ^ swz<CPR>(vr)) << 4) + (n16 & 1) * 8   // dim tile d: ^ (d << 5)
                            : 4 * g * G::kRowB + (n16 & 3) * 4);
  auto lds = [](uint32_t a) { return (lds_u8*)(uintptr_t)a; };
  // V^T's operand of dim tile d: fp16, keys 4 g .. 4 g + 3 of key tile j of dimension n16 (a transposing read);
  // fp32, key 4 g + j % 4 of key tile j / 4
  auto v_frag = [&](uint32_t va, int d, int j) -> typename VFrag<F16>::T {
    if constexpr (F16) {
      typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
      return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)lds((va ^ (d << 5)) + j * 16 * G::kRowB)));
    } else {
      const int i = j & 3;
      return *(const __attribute__((address_space(3))) uint32_t*)lds(
          va + (((4 * d + (n16 >> 2)) ^ swz<CPR>(4 * g + i)) << 4) + i * G::kRowB + (j >> 2) * 16 * G::kRowB);
    }
  };

  auto compute = [&](int k, int buf, bool masked) {
    uint32_t ka = ka0 + buf * G::kStageB, va = va0 + buf * G::kStageB;
    asm volatile("" : "+v"(ka), "+v"(va));   // the addresses of the steps are formed here, not kept over the loop
    // waves that share tiles pass their phases together: the workgroup whose products are waiting goes first
    if (!kOwn) __builtin_amdgcn_s_setprio(2);
    auto k_frag = [&](int c, int m) {
      return *(const __attribute__((address_space(3))) u32x4*)lds((ka ^ (c << 6)) + m * 16 * G::kRowB);
    };
    // A wave of its own has nothing to fill its waits with: it reads the whole tile first (its registers allow it).
    u32x4 kf[kOwn ? KC : 1][MT];
    typename VFrag<F16>::T vf[kOwn ? DT : 1][MT * (F16 ? 1 : 4)];
    if constexpr (kOwn) {
#pragma unroll
      for (int c = 0; c < KC; c++)
#pragma unroll
        for (int m = 0; m < MT; m++) kf[c][m] = k_frag(c, m);
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int j = 0; j < MT * (F16 ? 1 : 4); j++) vf[d][j] = v_frag(va, d, j);
      __builtin_amdgcn_sched_barrier(0);
    }
    f32x4 s[MT][NT], s2[F16 && kOwn ? MT : 1][NT];   // s2: the second term's sums, a chain of their own
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        s[m][nt] = (f32x4){0, 0, 0, 0};
        if constexpr (F16 && kOwn) s2[m][nt] = (f32x4){0, 0, 0, 0};
      }
#pragma unroll
    for (int c = 0; c < KC; c++)
#pragma unroll
      for (int m = 0; m < MT; m++) {
        const u32x4 a = kOwn ? kf[kOwn ? c : 0][m] : k_frag(c, m);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          if constexpr (F16) {
            f32x4& t = kOwn ? s2[kOwn ? m : 0][nt] : s[m][nt];
            s[m][nt] = mma16(a, qh[nt][c], s[m][nt]);
            t = mma16(a, ql[nt][c], t);
          } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
              s[m][nt] = mma(__uint_as_float(a[j]), __uint_as_float(qh[nt][c][j]), s[m][nt]);
          }
        }
      }
    if constexpr (F16 && kOwn) {
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) s[m][nt] += s2[m][nt];
    }
    settle_all(s);
    if (!kOwn) __builtin_amdgcn_s_setprio(0);
    if (masked) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        const int first = k + 4 * g - lo[nt];
        const uint32_t width = hi[nt] - lo[nt];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            s[m][nt][i] = (uint32_t)(first + 16 * m + i) < width ? s[m][nt][i] : -__builtin_inff();
      }
    }
    // this lane's largest scores; the reference moves only when one passes it by kSlack
    float mt[NT];
    bool moved = false;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      mt[nt] = -__builtin_inff();
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) mt[nt] = fmaxf(mt[nt], s[m][nt][i]);
      mt[nt] *= f[nt];
      moved |= mt[nt] > mref[nt] + kSlack;
    }
    if (__any(moved)) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        const float mn = fmaxf(mref[nt], max_over_groups(mt[nt]));
        const float al = mn == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(mref[nt] - mn);
        mref[nt] = mn;
        z[nt] *= al;
#pragma unroll
        for (int d = 0; d < DT; d++) acc[d][nt] *= al;
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const float bias = kPShift<F16> - (mref[nt] == -__builtin_inff() ? 0.0f : mref[nt]);
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          s[m][nt][i] = __builtin_amdgcn_exp2f(fmaf(s[m][nt][i], f[nt], bias));
          z[nt] += s[m][nt][i];
        }
    }
    if constexpr (F16) {
      u32x4 ph[MT / 2][NT], pl[MT / 2][NT];
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            uint32_t a, e;
            split2(s[m][nt][i], s[m][nt][i + 1], &a, &e);
            ph[m / 2][nt][(m & 1) * 2 + i / 2] = a;
            pl[m / 2][nt][(m & 1) * 2 + i / 2] = e;
          }
      if (!kOwn) __builtin_amdgcn_s_setprio(1);
      auto v_pair = [&](int d, int kk) {
        const u32x2 w0 = kOwn ? vf[kOwn ? d : 0][2 * kk] : v_frag(va, d, 2 * kk);
        const u32x2 w1 = kOwn ? vf[kOwn ? d : 0][2 * kk + 1] : v_frag(va, d, 2 * kk + 1);
        return (u32x4){w0.x, w0.y, w1.x, w1.y};
      };
      if constexpr (kOwn) {   // an accumulator's two products far apart
#pragma unroll
        for (int kk = 0; kk < MT / 2; kk++)
#pragma unroll
          for (int term = 0; term < 2; term++)
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
              for (int nt = 0; nt < NT; nt++)
                acc[d][nt] = mma16(v_pair(d, kk), term ? pl[kk][nt] : ph[kk][nt], acc[d][nt]);
      } else {
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
          for (int kk = 0; kk < MT / 2; kk++) {
            const u32x4 av = v_pair(d, kk);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              acc[d][nt] = mma16(av, ph[kk][nt], acc[d][nt]);
              acc[d][nt] = mma16(av, pl[kk][nt], acc[d][nt]);
            }
          }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
          for (int m = 0; m < MT; m++) {
            const uint32_t w = kOwn ? vf[kOwn ? d : 0][m * 4 + i] : v_frag(va, d, m * 4 + i);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) acc[d][nt] = mma(__uint_as_float(w), s[m][nt][i], acc[d][nt]);
          }
    }
    settle_all(acc);
    if (!kOwn) __builtin_amdgcn_s_setprio(0);
  };

  // ---- the split's tiles ---------------------------------------------------------------------------
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    mref[nt] = -__builtin_inff();
    z[nt] = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; d++) acc[d][nt] = (f32x4){0, 0, 0, 0};
  }
  for (int it = 0; it < iters; it++) {
    const int k = tile_key(it);
    const bool on = k < k1 && k < whi1 && k + KT > wlo0, masked = k < wlo1 || k + KT > whi0;
    if constexpr (kOwn) {
      // all but the loads of the tile after this one have come
      if (it + 1 < iters) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * G::kLoads) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (on) compute(k, it & 1, masked);
      if (it + 2 < iters) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // what was read of this buffer has left it
        stage(tile_key(it + 2), next, it & 1);
        next = look_up(tile_key(it + 3));
      }
    } else {
      // this tile has come, and what was read of the one before it has left the buffer that is filled next
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __syncthreads();
      if (it + 1 < iters) {
        stage(tile_key(it + 1), next, (it + 1) & 1);
        next = look_up(tile_key(it + 2));
      }
      if (on) compute(k, it & 1, masked);
    }
  }
  // What is not finite and was wrongly met -- a value of infinity times the zero weight of a masked key, an infinity
  // times two terms of different signs -- is a NaN in the results; the sum is one also where infinities of both signs meet.
  float sum = 0.0f;
#pragma unroll
  for (int d = 0; d < DT; d++)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 4; e++) sum += acc[d][nt][e];
  if (__syncthreads_or(sum != sum)) return false;

  // ---- the groups of keys joined, and the result ---------------------------------------------------
#pragma unroll
  for (int nt = 0; nt < NT; nt++) z[nt] = sum_over_groups(z[nt]);
  auto put = [&](int row, int d, f32x4 o, float m, float zz) { put_row(A, X, h, sp, row, d, o, m, zz); };
  if constexpr (KW == 1) {
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int row = rw0 + nt * 16 + n16;
      if (row < X.rows)
#pragma unroll
        for (int d = 0; d < DT; d++)
          if (16 * d + 4 * g < C.hd) put(row, 16 * d + 4 * g, acc[d][nt], mref[nt], z[nt]);
    }
  } else {
    // [key group][row][HDP + 4] sums, then [key group][row] references and sums of weights
    constexpr int R = RW * NT * 16;
    float* so = (float*)smem;
    float* sm = so + KW * R * G::kAccStride;
    float* sz = sm + KW * R;
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int r = kw * R + (rw * NT + nt) * 16 + n16;
#pragma unroll
      for (int d = 0; d < DT; d++) *(f32x4*)(so + r * G::kAccStride + 16 * d + 4 * g) = acc[d][nt];
      if (g == 0) {
        sm[r] = mref[nt];
        sz[r] = z[nt];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * (HDP / 4); i += G::kThreads) {
      const int r = i / (HDP / 4), d = i % (HDP / 4) * 4;
      if (X.row0 + r >= X.rows || d >= C.hd) continue;
      float m = -__builtin_inff(), zz = 0.0f;
      f32x4 o = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < KW; w++) m = fmaxf(m, sm[w * R + r]);
#pragma unroll
      for (int w = 0; w < KW; w++) {
        const float mw = sm[w * R + r], a = mw == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(mw - m);
        zz = fmaf(sz[w * R + r], a, zz);
        const f32x4 x = *(const f32x4*)(so + (w * R + r) * G::kAccStride + d);
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = fmaf(x[e], a, o[e]);
      }
      put(X.row0 + r, d, o, m, zz);
    }
  }
  return true;
}

// PER_SEQ: workgroup x takes sequence x, whose rows are one tile where max_q is right (and any others one by one);
// else tile x of the batch.
template <int HDP, int NT, int RW, int KW, int KT, bool F16, int WPE, bool PER_SEQ>
__global__ __launch_bounds__(64 * RW * KW, WPE) void k_attn_paged(AttnArgs A) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];   // a row's chunks change by xor
  constexpr int TM = 16 * NT * RW;
  const int x = div_by(A.by_nkv, blockIdx.x), h = blockIdx.x - x * A.C.nkv, sp = blockIdx.y;
  const_int* qs = scalar_ints(A.q_start);
  int b = x, tile = 0;
  if constexpr (!PER_SEQ) {
    find_tile(A, x, TM, &b, &tile);
    if (b < 0) return;
  }
  const int q0 = qs[b], q1 = qs[b + 1], L = scalar_ints(A.len)[b];
  Tile X = tile_of(A, q0, q1, L, tile, TM, KT);
  if (X.rows == 0) return;
  bool done = sp >= X.nact || attend<HDP, NT, RW, KW, KT, F16>(A, X, b, h, sp, smem);
  for (;;) {
    if (!done)
      rows_one_by_one<TM, RW * KW, F16>(A, X, b, h, X.kbeg + sp * A.chunk,
                                        sp == X.nact - 1 ? X.hi : X.kbeg + (sp + 1) * A.chunk, sp);
    if (!PER_SEQ || ++tile * TM >= X.rows) break;
    X = tile_of(A, q0, q1, L, tile, TM, KT);
    done = sp >= X.nact;
  }
}

// The splits of a row and head joined; rows with one split are in `out` already.  An item (row and head) takes
// `groups` groups of hd / 4 lanes, at least a wave: group i sums splits i, i + groups, .. in ascending order, then the
// groups are joined in ascending order through LDS (the order depends on the sizes alone).
__global__ __launch_bounds__(256) void k_attn_paged_join(AttnArgs A, int tm, int kt, int lanes, int groups) {
  __shared__ __attribute__((aligned(16))) float so[256 * 4];
  __shared__ float sm[256], sz[256];
  const int hd = A.C.hd, per = lanes * groups;
  const int sub = threadIdx.x / per, in = threadIdx.x % per, grp = in / lanes, d = in % lanes * 4;
  const uint32_t item = blockIdx.x * (256 / per) + sub;   // T * nh < 2^31
  const int r = __builtin_amdgcn_readfirstlane(div_by(A.by_nh, (int)item));
  const int head = __builtin_amdgcn_readfirstlane((int)item) - r * A.nh;
  const size_t row = (size_t)r * A.nh + head, at = row * A.nsplit;
  // four splits of this group from s on; the first four are asked for before it is known how many took part
  float ms[4], zs[4];
  f32x4 x[4];
  const bool mine = r < A.T && d < hd;
  auto load = [&](int s) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int sj = s + j * groups;
      const bool in = mine && sj < A.nsplit;
      ms[j] = in ? A.ws.m[at + sj] : 0.0f;
      zs[j] = in ? A.ws.z[at + sj] : 0.0f;
      x[j] = in ? *(const f32x4*)(A.ws.o + (at + sj) * hd + d) : (f32x4){0, 0, 0, 0};
    }
  };
  load(grp);
  const int b = r < A.T ? seq_of_row(A.q_start, A.B, r) : -1;
  Tile X = {};
  int t = 0;
  if (b >= 0) {
    const int q0 = A.q_start[b];
    t = r - q0;
    X = tile_of(A, q0, A.q_start[b + 1], A.len[b], (t * A.rep + (head - div_by(A.by_rep, head) * A.rep)) / tm, tm, kt);
  }
  const bool on = b >= 0 && X.rows > 0 && X.nact > 1;
  float m = -__builtin_inff(), z = 0.0f;
  f32x4 o = {0, 0, 0, 0};
  if (on && d < hd) {
    for (int s = grp; s < X.nact;) {
      float mn = m;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (s + j * groups >= X.nact) ms[j] = -__builtin_inff();
        mn = fmaxf(mn, ms[j]);
      }
      const float a0 = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
      z *= a0;
      o *= a0;
      m = mn;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (s + j * groups >= X.nact) continue;   // what lies there was not written
        const float a = ms[j] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ms[j] - mn);
        z = fmaf(zs[j], a, z);
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = fmaf(x[j][e], a, o[e]);
      }
      s += 4 * groups;
      if (s < X.nact) load(s);
    }
  }
  *(f32x4*)(so + threadIdx.x * 4) = o;
  sm[threadIdx.x] = m;
  sz[threadIdx.x] = z;
  __syncthreads();
  if (!on || grp != 0 || d >= hd) return;
  float M = -__builtin_inff();
  for (int i = 0; i < groups; i++) M = fmaxf(M, sm[threadIdx.x + i * lanes]);
  z = 0.0f;
  o = (f32x4){0, 0, 0, 0};
  for (int i = 0; i < groups; i++) {
    const int w = threadIdx.x + i * lanes;
    const float a = sm[w] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(sm[w] - M);
    z = fmaf(sz[w], a, z);
    const f32x4 x = *(const f32x4*)(so + w * 4);
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = fmaf(x[e], a, o[e]);
  }
  const bool any = key_hi(X.past, X.cap, t) > key_lo(A, X.past, t);
  const float inv = 1.0f / z;
#pragma unroll
  for (int e = 0; e < 4; e++) A.out[row * hd + d + e] = any ? o[e] * inv : 0.0f;
}

// ---- the launch ------------------------------------------------------------------------------------
enum Form { kDecode16, kDecode32, kRows64, kRows128 };

struct Plan {
  Form form;
  int tm, kt;        // rows of a tile, keys of a key tile
  bool per_seq;      // a workgroup a sequence: all of its rows are one tile if max_q is right
  int tiles;         // workgroups along the batch
  bool halves;       // workgroups of half the waves, two a CU
  int chunk, nsplit;
  int most;          // splits of any window: what the workspace is sized for
};

// Key tiles: 32 keys (fp16) or 16 (fp32) where a wave keeps its own, 64 where four share them.
int form_kt(Form f, int hd, bool f16) {
  if (!f16) return 16;
  return f == kRows128 && hd <= 128 ? 64 : 32;
}

Plan plan_form(Form form, int T, int B, int nh, const PagedKv& C, bool f16, int max_len, int window) {
  Plan P;
  const int rep = nh / C.nkv;
  P.form = form;
  P.per_seq = form == kDecode16 || form == kDecode32;
  P.tm = form == kDecode16 ? 16 : form == kDecode32 ? 32 : form == kRows64 || C.hd > 128 ? 64 : 128;
  P.kt = form_kt(form, C.hd, f16);
  const int seqs = B < T ? B : T;
  const long long full = (long long)T * rep / P.tm;
  P.tiles = P.per_seq ? B : (int)(full + seqs);
  const long long cap = (long long)C.stride << C.shift;
  long long len = max_len > 0 ? max_len : 4096;
  if (len > cap) len = cap;
  const long long est = (full > seqs ? full : seqs) * C.nkv;       // workgroups of one split
  const long long least = P.per_seq ? 256 : 128, unit = P.per_seq ? 128 : 64;   // keys; unit: the key tiles of all groups
  long long span = len;                                             // keys of one tile's rows
  if (window > 0 && span > (long long)window + P.tm / rep + 2) span = (long long)window + P.tm / rep + 2;
  auto set = [&](long long want) {
    long long chunk = (span + want - 1) / want;
    if (chunk < least) chunk = least;
    P.chunk = (int)((chunk + unit - 1) / unit * unit);
    P.nsplit = (int)((span + P.chunk - 1) / P.chunk);
  };
  // Splits.  Tiles of 128 rows, to two workgroups a CU, which is what registers allow: four chunks over 6000 at 512 / 1024 /
  // 1536 workgroups 171 / 186 / 224 us.  Tiles of 64 rows, where the CUs are not all taken, to two a CU (11 x 96 tokens over
  // 3640 at 3 / 1 splits 37 / 44 us); where they are, the join costs more than it gives (8 x 64 over 500 at 2 / 1 splits 29
  // / 20).
  long long most = form == kRows128 ? (2 * kCus + est - 1) / est : form == kRows64 && est >= kCus ? 1 : 2 * kCus / est;
  most = most < 1 ? 1 : most > kMaxSplits ? kMaxSplits : most;
  set(most);
  if (P.per_seq) {
    // Few rows: one workgroup a CU (its ring fills LDS), so that what counts is rounds of workgroups.  In keys: those of a
    // split and about 200 for a workgroup's beginning and end each round, and 300 for the join.  One token over 32768
    // at 32 / 64 / 43 splits (256, 512, 344 workgroups) 32 / 36 / 38 us.
    long long best = 0, pick = 1;
    for (long long w = 1; w <= most; w++) {
      set(w);
      const long long cost = (est * P.nsplit + kCus - 1) / kCus * (P.chunk + 200) + (P.nsplit > 1 ? 300 : 0);
      if (w == 1 || cost < best) {
        best = cost;
        pick = w;
      }
      if (P.chunk <= least) break;   // no shorter split
    }
    set(pick);
  }
  // Up to 32 rows, four groups of waves a workgroup while each workgroup has a CU of its own, else two, so that one
  // workgroup's products go beside another's waits (four / two: 8 x 5 tokens over 700 14.4 / 15.1 us, one of 5 over 30000 26.8
  // / 28.5; 64 x 5 over 4096 148 / 129, 20 x 8 over 5727 81 / 67)
  P.halves = form == kDecode32 && est * P.nsplit > kCus;
  P.most = (int)((len + least - 1) / least < most ? (len + least - 1) / least : most);
  return P;
}

// Rows of a sequence's KV head, at most: to 16 a wave's own tile, four waves on different keys; to 32 two waves' (eight drafts
// of 5 x 4 rows 14.7 us, with 32 rows a wave 17.5); past that workgroups that share their keys.  Of those, 64 rows with
// 16 a wave make more workgroups and need fewer splits, 128 with 32 a wave read less of LDS a product, which pays once a
// workgroup has kLongKeys keys to go through (64 / 128 rows: 2 x 500 tokens over 2000, 700 keys a workgroup, 54 / 87 us;
// 4 x 509 over 6000, 3300 keys, 153 / 159; 512 over 14336, 3700 keys, 224 / 211; 2048 over 14336 864 / 792).  The fp32
// instruction is slow enough for the narrow form throughout (2 x 500 over 2000 241 / 250).
constexpr int kLongKeys = 3500;
Plan make_plan(int T, int B, int nh, const PagedKv& C, bool f16, int max_q, int max_len, int window) {
  if (max_q <= 0 || max_q > T) max_q = T;
  const long long rows = (long long)max_q * (nh / C.nkv);
  auto form = [&](Form f) { return plan_form(f, T, B, nh, C, f16, max_len, window); };
  if (rows <= 16) return form(kDecode16);
  if (C.hd > 128) return form(kRows128);
  if (rows <= 32) return form(kDecode32);
  if (rows <= 64 || !f16) return form(kRows64);
  const Plan wide = form(kRows128);
  if (wide.chunk >= kLongKeys) return wide;
  Plan P = form(kRows64);
  P.most = wide.most > P.most ? wide.most : P.most;   // another window may take the other form
  return P;
}

template <int HDP, bool F16>
int launch(lt_ctx* ctx, const AttnArgs& A, const Plan& P) {
  const dim3 grid((unsigned)P.tiles * A.C.nkv, P.nsplit);
  auto go = [&](auto kernel, int threads, int lds) {
    kernel<<<grid, threads, lds, ctx->stream>>>(A);
    return lt_check_launch("k_attn_paged");
  };
  constexpr int KT = F16 ? 32 : 16, KT2 = F16 && HDP <= 128 ? 64 : KT, KW = HDP <= 128 ? 4 : 2, NT = HDP <= 128 ? 2 : 1;
  switch (P.form) {
    case kDecode16:
      return go(k_attn_paged<HDP, 1, 1, KW, KT, F16, 1, true>, 64 * KW, Cfg<HDP, 1, 1, KW, KT, F16>::kLds);
    case kDecode32:
      if constexpr (HDP <= 128) {
        if (P.halves) return go(k_attn_paged<HDP, 1, 2, 2, KT, F16, 1, true>, 256, Cfg<HDP, 1, 2, 2, KT, F16>::kLds);
        return go(k_attn_paged<HDP, 1, 2, 4, KT, F16, 1, true>, 512, Cfg<HDP, 1, 2, 4, KT, F16>::kLds);
      }
      break;
    case kRows64:
      if constexpr (HDP <= 128) return go(k_attn_paged<HDP, 1, 4, 2, KT, F16, 1, false>, 512, Cfg<HDP, 1, 4, 2, KT, F16>::kLds);
      break;
    case kRows128:
      return go(k_attn_paged<HDP, NT, 4, 1, KT2, F16, 2, false>, 256, Cfg<HDP, NT, 4, 1, KT2, F16>::kLds);
  }
  return lt_fail(LT_EINVAL, "lt_attn_paged: no kernel");
}

}  // namespace

extern "C" {

size_t lt_attn_paged_workspace_size(int T, int B, int nh, const lt_paged_kv* kv, int max_q, int max_len) {
  PagedKv C;
  if (T <= 0 || T > (1 << 24) || B <= 0 || lt_paged_check("lt_attn_paged_workspace_size", kv, nh, &C)) return 0;
  const Plan P = make_plan(T, B, nh, C, kv->kv_dtype == LT_KV_F16, max_q, max_len, 0);
  return P.most == 1 ? 0 : lt_attn_ws_bytes(T * nh, C.hd, P.most);
}

int lt_attn_paged(lt_ctx* ctx, const float* q, int q_stride, int T, const int* q_start, const int* len, int B, int nh,
                  const lt_paged_kv* kv, float* out, float scale, int window, int max_q, int max_len, void* ws,
                  size_t ws_bytes, int* err) {
  const char* fn = "lt_attn_paged";
  LT_REQUIRE(q && out && q_start && len, "%s: null argument", fn);
  PagedKv C;
  if (int rc = lt_paged_check(fn, kv, nh, &C)) return rc;
  LT_REQUIRE(T >= 0 && B > 0 && q_stride >= (long long)nh * C.hd, "%s: T=%d B=%d q_stride=%d (at least %d)", fn, T, B,
             q_stride, nh * C.hd);
  LT_REQUIRE(window >= 0 && max_q >= 0 && max_len >= 0, "%s: window=%d max_q=%d max_len=%d", fn, window, max_q, max_len);
  LT_REQUIRE(T <= (1 << 24) && (long long)T * nh < (1ll << 31), "%s: T=%d rows of nh=%d heads", fn, T, nh);
  const bool f16 = kv->kv_dtype == LT_KV_F16;
  Plan P = {};
  if (T > 0) {
    P = make_plan(T, B, nh, C, f16, max_q, max_len, window);
    LT_REQUIRE((long long)P.tiles * C.nkv < (1ll << 31), "%s: T=%d B=%d nkv=%d", fn, T, B, C.nkv);
  }
  if (P.nsplit > 1) {
    const size_t need = lt_attn_ws_bytes(T * nh, C.hd, P.nsplit);
    LT_REQUIRE(ws, "%s: null workspace", fn);
    LT_REQUIRE(lt_aligned(ws, 16), "%s: workspace 16-byte aligned", fn);
    if (ws_bytes < need) return lt_fail(LT_ENOMEM, "%s: workspace %zu < %zu bytes", fn, ws_bytes, need);
  }
  LT_REQUIRE(ctx, "%s: null ctx", fn);
  if (T == 0) return LT_OK;
  const LtDeviceGuard guard(ctx);
  AttnArgs A = {q, q_stride, q_start, len, B, T, nh, nh / C.nkv, C, out, scale < 0 ? -scale : scale, scale < 0 ? -1.0f : 1.0f,
                window, err, lt_aligned(q, 16) && q_stride % 4 == 0 && lt_aligned(out, 16), P.chunk, P.nsplit, {},
                make_div(nh / C.nkv), make_div(P.chunk ? P.chunk : 1), make_div(C.nkv), make_div(nh)};
  if (P.nsplit > 1) A.ws = lt_attn_ws_layout(ws, T * nh, C.hd, P.nsplit);
  int rc;
  if (C.hd <= 64) rc = f16 ? launch<64, true>(ctx, A, P) : launch<64, false>(ctx, A, P);
  else if (C.hd <= 128) rc = f16 ? launch<128, true>(ctx, A, P) : launch<128, false>(ctx, A, P);
  else rc = f16 ? launch<256, true>(ctx, A, P) : launch<256, false>(ctx, A, P);
  if (rc || P.nsplit == 1) return rc;
  // lanes for the head dim; groups for the splits, to a wave at least and a workgroup at most
  int lanes = 1, groups = 1;
  while (lanes * 4 < C.hd) lanes *= 2;
  while (groups < P.nsplit && lanes * groups < 256) groups *= 2;
  while (lanes * groups < 64) groups *= 2;
  const long long items = (long long)T * nh, per = 256 / (lanes * groups);
  k_attn_paged_join<<<(unsigned)((items + per - 1) / per), 256, 0, ctx->stream>>>(A, P.tm, P.kt, lanes, groups);
  return lt_check_launch("k_attn_paged_join");
}

}  // extern "C"
