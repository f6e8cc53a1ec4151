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
// P is held as 2^7 exp2(score - reference), the reference moved once a score passes it by 8: at most 2^15, and a weight
// of 2^-32 of the largest still has a term
constexpr float kPShift = 7.0f, kSlack = 8.0f;
constexpr int kMaxSplits = 128;

__device__ const u32x4 g_zero16 = {0, 0, 0, 0};   // what a row without a page reads

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
};

// One tile of a sequence's rows and the keys it attends.
struct Tile {
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

__device__ __forceinline__ Tile tile_of(const AttnArgs& A, int b, int tile, int tm, int kt) {
  Tile X;
  X.cap = A.C.stride << A.C.shift;
  const int L = A.len[b];
  X.past = L < 0 ? 0 : L < X.cap ? L : X.cap;
  X.row0 = tile * tm;
  X.rows = (A.q_start[b + 1] - A.q_start[b]) * A.rep;
  const int last = X.row0 + tm < X.rows ? X.row0 + tm - 1 : X.rows - 1;
  X.lo = key_lo(A, X.past, X.row0 / A.rep);
  X.hi = key_hi(X.past, X.cap, last / A.rep);
  X.kbeg = X.lo & ~(kt - 1);
  const int n = X.hi > X.kbeg ? (X.hi - X.kbeg + A.chunk - 1) / A.chunk : 1;
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
      const int s = A.q_start[c + lane], e = A.q_start[c + lane + 1];
      n = s >= 0 && e > s && e <= A.T ? ((e - s) * A.rep + tm - 1) / tm : 0;
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
  static_assert(D % 4 == 0 && (N == 1 || N == 2), "settle_all: accumulators");
#pragma unroll
  for (int d = 0; d < D; d += 4) {
    if constexpr (N == 1)
      asm volatile("s_nop 15" : "+v"(o[d][0]), "+v"(o[d + 1][0]), "+v"(o[d + 2][0]), "+v"(o[d + 3][0]));
    else
      asm volatile("s_nop 15"
                   : "+v"(o[d][0]), "+v"(o[d][1]), "+v"(o[d + 1][0]), "+v"(o[d + 1][1]), "+v"(o[d + 2][0]),
                     "+v"(o[d + 2][1]), "+v"(o[d + 3][0]), "+v"(o[d + 3][1]));
  }
}

// Two fp32 values as two binary16 terms each.
__device__ __forceinline__ void split2(float a, float b, uint32_t* hi, uint32_t* lo) {
  const f16x2 h = __builtin_convertvector((f32x2){a, b}, f16x2);
  *hi = __builtin_bit_cast(uint32_t, h);
  *lo = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a - (float)h.x, b - (float)h.y}, f16x2));
}

// The same for a query, whose terms also multiply keys of infinity: both terms have q's sign and are zero only
// where q is, so that their products with one add up to what q's own is (the least binary16 in place of a zero: 2^-38
// of the row's largest).
__device__ __forceinline__ uint16_t same_sign(float x, float q) {
  const uint16_t h = __builtin_bit_cast(uint16_t, (_Float16)x);
  return (h & 0x7FFFu) == 0 && q != 0.0f ? (uint16_t)((__float_as_uint(q) >> 16 & 0x8000u) | 1u) : h;
}
__device__ __forceinline__ void split2_q(float a, float b, uint32_t* hi, uint32_t* lo) {
  const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(a, b));   // toward zero: the rest keeps the sign
  *hi = same_sign((float)h.x, a) | (uint32_t)same_sign((float)h.y, b) << 16;
  *lo = same_sign(a - (float)h.x, a) | (uint32_t)same_sign(b - (float)h.y, b) << 16;
}

// The binary16 halves of w that are not finite become zero; true when there were any.
__device__ __forceinline__ bool drop_nonfinite(uint32_t* w) {
  const bool l = (*w & 0x7C00u) == 0x7C00u, h = (*w & 0x7C000000u) == 0x7C000000u;
  *w &= (l ? 0xFFFF0000u : 0xFFFFFFFFu) & (h ? 0x0000FFFFu : 0xFFFFFFFFu);
  return l || h;
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

template <int HDP, int NT, int RW, int KW, int KT, bool F16, int WPE>
__global__ __launch_bounds__(64 * RW * KW, WPE) void k_attn_paged(AttnArgs A) {
  using G = Cfg<HDP, NT, RW, KW, KT, F16>;
  constexpr int CPR = G::kCpr, MT = KT / 16, DT = HDP / 16, KC = F16 ? HDP / 32 : HDP / 16;
  extern __shared__ __attribute__((aligned(256))) uint8_t smem[];
  const PagedKv& C = A.C;
  const int lane = threadIdx.x & 63, n16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rw = wave % RW, kw = wave / RW;
  const int h = blockIdx.x % C.nkv, sp = blockIdx.y;
  int b, tile;
  find_tile(A, blockIdx.x / C.nkv, G::kTM, &b, &tile);
  if (b < 0) return;
  const Tile X = tile_of(A, b, tile, G::kTM, KT);
  if (sp >= X.nact) return;
  const int k0 = X.kbeg + sp * A.chunk;
  const int k1 = sp == X.nact - 1 ? X.hi : k0 + A.chunk;
  if (X.past + (X.rows - 1) / A.rep >= X.cap && A.err && threadIdx.x == 0) *A.err = 1;

  // this lane's rows
  const int rw0 = X.row0 + rw * 16 * NT;
  const int q0 = A.q_start[b];
  int hi[NT], lo[NT];
  float f[NT];
  u32x4 qh[NT][KC], ql[F16 ? NT : 1][F16 ? KC : 1];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const int row = rw0 + nt * 16 + n16;
    const bool on = row < X.rows;
    const int t = row / A.rep;
    hi[nt] = on ? key_hi(X.past, X.cap, t) : 0;
    lo[nt] = on ? key_lo(A, X.past, t) : 0;
    const float* q = A.q + (size_t)(q0 + (on ? t : 0)) * A.q_stride + (size_t)(h * A.rep + (on ? row % A.rep : 0)) * C.hd;
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
          split2_q(v[c][j] * up, v[c][j + 1] * up, &a, &e);
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
  // the wave's rows as a whole
  const int wrows = rw0 + 16 * NT < X.rows ? 16 * NT : X.rows - rw0;
  const int tw0 = rw0 / A.rep, tw1 = (rw0 + wrows - 1) / A.rep;
  const int whi0 = key_hi(X.past, X.cap, tw0), whi1 = wrows > 0 ? key_hi(X.past, X.cap, tw1) : 0;
  const int wlo0 = key_lo(A, X.past, tw0), wlo1 = key_lo(A, X.past, tw1);

  // ---- key tiles into LDS -------------------------------------------------------------------------
  const uint32_t ring = (uint32_t)(uintptr_t)(lds_u8*)smem + kw * 2 * G::kStageB;
  const size_t row_b = (size_t)C.hd * (F16 ? 2 : 4);
  // byte offset of the pool row of key k + lane (lanes below KT), or -1: no row, or a page outside the pool
  auto look_up = [&](int k) -> long long {
    const int key = k + lane;
    if (lane >= KT || key < X.lo || key >= k1) return -1;
    const int pg = page_of(C, b, key);
    if (pg < 0) {
      if (A.err) *A.err = 1;
      return -1;
    }
    return (long long)((((size_t)pg * C.nkv + h) << C.shift) + (key & ((1 << C.shift) - 1))) * row_b;
  };
  auto stage = [&](long long off, int buf) {
#pragma unroll
    for (int i = 0; i < G::kLoads; i++) {
      const int first = (i * RW + rw) * 64, slot = first + lane;
      const int row = slot / CPR, c = (slot % CPR) ^ swz<CPR>(row);
      const long long o = __shfl(off, row, 64);
      const bool on = o >= 0 && (size_t)c * 16 < row_b;
      const uint8_t* kp = on ? (const uint8_t*)C.kc + o + c * 16 : (const uint8_t*)&g_zero16;
      const uint8_t* vp = on ? (const uint8_t*)C.vc + o + c * 16 : (const uint8_t*)&g_zero16;
      const uint32_t to = ring + buf * G::kStageB + first * 16;
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(kp) : "memory", "m0");
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to + G::kTileB), "v"(vp)
                   : "memory", "m0");
    }
  };

  // ---- one key tile -------------------------------------------------------------------------------
  f32x4 acc[DT][NT];
  float mref[NT], z[NT];
  const uint32_t ka0 = n16 * G::kRowB + ((g ^ swz<CPR>(n16)) << 4);             // step c: ^ (c << 6)
  const int vr = 4 * g + (n16 >> 2);
  const uint32_t va0 = vr * G::kRowB + ((((n16 >> 1) & 1) ^ swz<CPR>(vr)) << 4) + (n16 & 1) * 8;   // fp16: ^ (d << 5)
  auto lds = [](uint32_t a) { return (lds_u8*)(uintptr_t)a; };

  auto compute = [&](int k, int buf, auto masked) {
    constexpr bool M = decltype(masked)::value;
    const uint32_t kb = ring + buf * G::kStageB, vb = kb + G::kTileB;
    f32x4 s[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int nt = 0; nt < NT; nt++) s[m][nt] = (f32x4){0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < KC; c++)
#pragma unroll
      for (int m = 0; m < MT; m++) {
        const u32x4 a = *(const __attribute__((address_space(3))) u32x4*)lds(kb + m * 16 * G::kRowB + (ka0 ^ (c << 6)));
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          if constexpr (F16) {
            const f16x8 ah = __builtin_bit_cast(f16x8, a);
            s[m][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, __builtin_bit_cast(f16x8, qh[nt][c]), s[m][nt], 0, 0, 0);
            s[m][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, __builtin_bit_cast(f16x8, ql[nt][c]), s[m][nt], 0, 0, 0);
          } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
              s[m][nt] = mma(__uint_as_float(a[j]), __uint_as_float(qh[nt][c][j]), s[m][nt]);
          }
        }
      }
    // scores in base-2 units, their maxima, the reference
    float mt[NT];
    bool moved = false;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      mt[nt] = -__builtin_inff();
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float x = s[m][nt][i] * f[nt];
          if constexpr (M) {
            const int key = k + 16 * m + 4 * g + i;
            x = key < hi[nt] && key >= lo[nt] ? x : -__builtin_inff();
          }
          s[m][nt][i] = x;
          mt[nt] = fmaxf(mt[nt], x);
        }
      mt[nt] = max_over_groups(mt[nt]);
      moved |= mt[nt] > mref[nt] + kSlack;
    }
    if (__any(moved)) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        const float mn = fmaxf(mref[nt], mt[nt]);
        const float al = mn == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(mref[nt] - mn);
        mref[nt] = mn;
        z[nt] *= al;
#pragma unroll
        for (int d = 0; d < DT; d++) acc[d][nt] *= al;
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const float bias = kPShift - (mref[nt] == -__builtin_inff() ? 0.0f : mref[nt]);
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          s[m][nt][i] = __builtin_amdgcn_exp2f(s[m][nt][i] + bias);
          z[nt] += s[m][nt][i];
        }
    }
    bool bad = false;   // a masked tile's V values that are not finite are left to put_nonfinite
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
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int kk = 0; kk < MT / 2; kk++) {
          const uint32_t at = vb + kk * 32 * G::kRowB + (va0 ^ (d << 5));
          typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
          const i16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)lds(at));
          const i16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)lds(at + 16 * G::kRowB));
          const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
          uint32_t w[4] = {w0.x, w0.y, w1.x, w1.y};
          if constexpr (M) {
#pragma unroll
            for (int j = 0; j < 4; j++) bad |= drop_nonfinite(&w[j]);
          }
          const f16x8 av = __builtin_bit_cast(f16x8, (u32x4){w[0], w[1], w[2], w[3]});
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            acc[d][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, __builtin_bit_cast(f16x8, ph[kk][nt]), acc[d][nt], 0, 0, 0);
            acc[d][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, __builtin_bit_cast(f16x8, pl[kk][nt]), acc[d][nt], 0, 0, 0);
          }
        }
    } else {
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int r = 4 * g + i;
          const uint32_t rb = vb + (m * 16 + r) * G::kRowB + (n16 & 3) * 4;
#pragma unroll
          for (int d = 0; d < DT; d++) {
            const uint32_t at = rb + (((4 * d + (n16 >> 2)) ^ swz<CPR>(r)) << 4);
            uint32_t w = *(const __attribute__((address_space(3))) uint32_t*)lds(at);
            if constexpr (M) {
              if ((w & 0x7F800000u) == 0x7F800000u) {
                w = 0;
                bad = true;
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++) acc[d][nt] = mma(__uint_as_float(w), s[m][nt][i], acc[d][nt]);
          }
        }
    }
    settle_all(acc);
    if constexpr (M) {
      if (__any(bad)) {
        // the values that are not finite, key by key, for the rows that attend the key
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll 1
            for (int gg = 0; gg < 4; gg++) {
              const int r = 4 * gg + i, key = k + 16 * m + r;
              float p[NT];
              bool on[NT];
#pragma unroll
              for (int nt = 0; nt < NT; nt++) {
                p[nt] = __shfl(s[m][nt][i], gg * 16 + n16, 64);
                on[nt] = key < hi[nt] && key >= lo[nt];
              }
              const uint32_t rb = vb + (m * 16 + r) * G::kRowB;
#pragma unroll
              for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                  float v;
                  if constexpr (F16) {
                    const int c = 2 * d + (g >> 1);
                    v = lt_h2f(*(const __attribute__((address_space(3))) uint16_t*)lds(
                        rb + ((c ^ swz<CPR>(r)) << 4) + (g & 1) * 8 + e * 2));
                  } else {
                    v = *(const __attribute__((address_space(3))) float*)lds(rb + (((4 * d + g) ^ swz<CPR>(r)) << 4) + e * 4);
                  }
                  if (!__builtin_isfinite(v)) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
                      if (on[nt]) acc[d][nt][e] = fmaf(p[nt], v, acc[d][nt][e]);
                  }
                }
            }
      }
    }
  };

  // ---- the split's tiles: while one is computed, the next is on its way ----------------------------
  const int ntiles = k1 > k0 ? (k1 - k0 + KT - 1) / KT : 0, iters = (ntiles + KW - 1) / KW;
  auto tile_key = [&](int it) { return k0 + (it * KW + kw) * KT; };
  // A value of infinity that is attended meets a weight's two terms one by one, and the second may be zero or
  // negative: a NaN in the result sends the workgroup over its tiles again with such values taken apart everywhere.
  bool careful = false;
  for (;;) {
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      mref[nt] = -__builtin_inff();
      z[nt] = 0.0f;
#pragma unroll
      for (int d = 0; d < DT; d++) acc[d][nt] = (f32x4){0, 0, 0, 0};
    }
    if (iters > 0) {
      stage(look_up(tile_key(0)), 0);
      long long off = look_up(tile_key(1));
      for (int it = 0; it < iters; it++) {
        // this tile has come, and what was read of the one before it has left the buffer that is filled next
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if constexpr (RW > 1) __syncthreads();
        if (it + 1 < iters) {
          stage(off, (it + 1) & 1);
          off = look_up(tile_key(it + 2));
        }
        const int k = tile_key(it);
        if (k < k1 && k < whi1 && k + KT > wlo0) {
          if (careful || k < wlo1 || k + KT > whi0) compute(k, it & 1, std::true_type{});
          else compute(k, it & 1, std::false_type{});
        }
      }
    }
    if (careful) break;
    float sum = 0.0f;   // NaN where any of them is, or where infinities of both signs meet
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) sum += acc[d][nt][e];
    if (!F16 || !__syncthreads_or(sum != sum)) break;
    careful = true;
  }

  // ---- the groups of keys joined, and the result ---------------------------------------------------
#pragma unroll
  for (int nt = 0; nt < NT; nt++) z[nt] = sum_over_groups(z[nt]);
  const bool final = X.nact == 1;
  auto put = [&](int row, int d, f32x4 o, float m, float zz) {   // d < hd, a multiple of 4
    const int t = row / A.rep, head = h * A.rep + row % A.rep;
    const size_t r = (size_t)(q0 + t) * A.nh + head;
    if (final) {
      const bool any = key_hi(X.past, X.cap, t) > key_lo(A, X.past, t);
      const float inv = 1.0f / zz;
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] = any ? o[e] * inv : 0.0f;
      float* to = A.out + r * C.hd + d;
      if (A.vec) *(f32x4*)to = o;
      else
#pragma unroll
        for (int e = 0; e < 4; e++) to[e] = o[e];
    } else {
      const size_t at = r * A.nsplit + sp;
      *(f32x4*)(A.ws.o + at * C.hd + d) = o;
      if (d == 0) {
        A.ws.m[at] = m;
        A.ws.z[at] = zz;
      }
    }
  };
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
}

// The splits of one row and head joined in ascending order; rows with one split are in `out` already.
__global__ __launch_bounds__(64) void k_attn_paged_join(AttnArgs A, int tm, int kt) {
  const int r = blockIdx.x, head = blockIdx.y, lane = threadIdx.x, hd = A.C.hd;
  const int b = seq_of_row(A.q_start, A.B, r);
  if (b < 0) return;
  const int t = r - A.q_start[b];
  const Tile X = tile_of(A, b, (t * A.rep + head % A.rep) / tm, tm, kt);
  if (X.nact == 1) return;
  const size_t row = (size_t)r * A.nh + head, at = row * A.nsplit;
  float m = -__builtin_inff();
  for (int s = lane; s < X.nact; s += 64) m = fmaxf(m, A.ws.m[at + s]);
  for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
  const bool any = key_hi(X.past, X.cap, t) > key_lo(A, X.past, t);
  for (int d = lane * 4; d < hd; d += 256) {
    float z = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    for (int s = 0; s < X.nact; s++) {
      const float ms = A.ws.m[at + s], a = ms == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ms - m);
      z = fmaf(A.ws.z[at + s], a, z);
      const f32x4 x = *(const f32x4*)(A.ws.o + (at + s) * hd + d);
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] = fmaf(x[e], a, o[e]);
    }
    const float inv = 1.0f / z;
#pragma unroll
    for (int e = 0; e < 4; e++) A.out[row * hd + d + e] = any ? o[e] * inv : 0.0f;
  }
}

// ---- the launch ------------------------------------------------------------------------------------
enum Form { kDecode16, kDecode32, kRows64, kRows128 };

struct Plan {
  Form form;
  int tm, kt;        // rows of a tile, keys of a key tile
  int tiles;         // at most
  int chunk, nsplit;
  int most;          // splits of any window: what the workspace is sized for
};

// Key tiles: 32 keys (fp16) or 16 (fp32) a wave or four of them, 64 where four share rows of 64.
int form_kt(Form f, int hd, bool f16) {
  if (!f16) return 16;
  return f == kRows128 && hd <= 64 ? 64 : 32;
}

Plan make_plan(int T, int B, int nh, const PagedKv& C, bool f16, int max_q, int max_len, int window) {
  Plan P;
  const int rep = nh / C.nkv;
  if (max_q <= 0 || max_q > T) max_q = T;
  const long long rows = (long long)max_q * rep;
  const bool wide = C.hd > 128;
  P.form = rows <= 16 ? kDecode16 : wide ? kRows128 : rows <= 32 ? kDecode32 : rows <= 64 ? kRows64 : kRows128;
  P.tm = P.form == kDecode16 ? 16 : P.form == kDecode32 ? 32 : P.form == kRows64 || wide ? 64 : 128;
  P.kt = form_kt(P.form, C.hd, f16);
  const int seqs = B < T ? B : T;
  const long long full = (long long)T * rep / P.tm;
  P.tiles = (int)(full + seqs);
  // splits: enough workgroups for the CUs, of at least 256 keys
  const long long cap = (long long)C.stride << C.shift;
  long long len = max_len > 0 ? max_len : 4096;
  if (len > cap) len = cap;
  if (window > 0 && len > (long long)window + max_q) len = (long long)window + max_q;
  const long long est = (full > seqs ? full : seqs) * C.nkv;
  long long want = (512 + est - 1) / est;
  if (want > kMaxSplits) want = kMaxSplits;
  long long chunk = (len + want - 1) / want;
  if (chunk < 256) chunk = 256;
  P.chunk = (int)((chunk + 255) / 256 * 256);
  P.nsplit = (int)((len + P.chunk - 1) / P.chunk);
  P.most = (int)((len + 255) / 256 < want ? (len + 255) / 256 : want);
  return P;
}

template <int HDP, bool F16>
int launch(lt_ctx* ctx, const AttnArgs& A, const Plan& P) {
  const dim3 grid((unsigned)P.tiles * A.C.nkv, P.nsplit);
  auto go = [&](auto kernel, int threads, int lds) {
    kernel<<<grid, threads, lds, ctx->stream>>>(A);
    return lt_check_launch("k_attn_paged");
  };
  constexpr int KT = F16 ? 32 : 16, KT2 = F16 && HDP <= 64 ? 64 : KT, KW = HDP <= 128 ? 4 : 2, NT = HDP <= 128 ? 2 : 1;
  switch (P.form) {
    case kDecode16:
      return go(k_attn_paged<HDP, 1, 1, KW, KT, F16, 1>, 64 * KW, Cfg<HDP, 1, 1, KW, KT, F16>::kLds);
    case kDecode32:
      if constexpr (HDP <= 128) return go(k_attn_paged<HDP, 2, 1, 4, KT, F16, 1>, 256, Cfg<HDP, 2, 1, 4, KT, F16>::kLds);
      break;
    case kRows64:
      if constexpr (HDP <= 128) return go(k_attn_paged<HDP, 2, 2, 2, KT, F16, 1>, 256, Cfg<HDP, 2, 2, 2, KT, F16>::kLds);
      break;
    case kRows128:
      return go(k_attn_paged<HDP, NT, 4, 1, KT2, F16, 2>, 256, Cfg<HDP, NT, 4, 1, KT2, F16>::kLds);
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
                window, err, lt_aligned(q, 16) && q_stride % 4 == 0 && lt_aligned(out, 16), P.chunk, P.nsplit, {}};
  if (P.nsplit > 1) A.ws = lt_attn_ws_layout(ws, T * nh, C.hd, P.nsplit);
  int rc;
  if (C.hd <= 64) rc = f16 ? launch<64, true>(ctx, A, P) : launch<64, false>(ctx, A, P);
  else if (C.hd <= 128) rc = f16 ? launch<128, true>(ctx, A, P) : launch<128, false>(ctx, A, P);
  else rc = f16 ? launch<256, true>(ctx, A, P) : launch<256, false>(ctx, A, P);
  if (rc || P.nsplit == 1) return rc;
  k_attn_paged_join<<<dim3(T, nh), 64, 0, ctx->stream>>>(A, P.tm, P.kt);
  return lt_check_launch("k_attn_paged_join");
}

}  // extern "C"
