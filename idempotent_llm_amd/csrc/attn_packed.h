// The blocks of the packed attention (attn_packed.hip, gfx950).
#pragma once

#include "attn_tiles.h"

namespace {

constexpr int PACKED_MAX_S = 131071;    // int32 accumulators: 128 * 128 * S < 2^31
constexpr int PACKED_MAX_ROWS = 65536;  // rows of a batch
constexpr int FEW_SLOTS = 2048;         // slots of a few-row unit in a block of eight waves
constexpr int FEW_ONE_SLOTS = 512;      // and beside tiles

// Passes
constexpr int PH_MAX = 1, PH_DEN = 2, PH_PV = 4, PH_ALL = 7;

struct PackedArgs {
  const int8_t* q8;     // [N][n_q][128]
  const int64_t* tpos;  // [N][n_q]
  KVPages kv;
  int n_pages;
  const int32_t* cu;    // [B + 1]
  const int32_t* past;  // [B]
  int N, B, S, max_new, n_q, n_kv;
  int lg;        // log2 of the query heads per kv head
  // A few-row unit's rows of scores start at row b few_rows, or, where all token rows
  // have fewer (few_rows 0), at its first token's
  int few_rows, score_rows;
  int units, chunk, nch;
  int step;      // blocks per kv head
  int32_t* scores;  // few-row units: [n_kv][score_rows][nch * chunk]
  int32_t* smax;    // [units][n_kv][nch][64]: maxima of the visible scores
  int64_t* sden;    // the same of partial denominators
  int32_t* part;    // [nch][N][n_q * 128] contexts (null: one chunk, straight to out)
  int64_t* out;     // [N][n_q * 128]
  int32_t* err;
};

// Never a score: |q . k| <= 2^21
constexpr int32_t NO_SCORE = INT32_MIN;

// What a block works on: a chunk of a unit, for a kv head
struct Work {
  bool few;   // the row has at most 16 query rows
  bool bad;   // the row's slots are past the launch's bound
  int b, tile, unit, kvh, c;
  int tok0, T, past;  // the row's first token row, its tokens and filled slots
  int len;            // slots that its tokens see (past + T, bounded)
};

// Last slot that token t of a row at `past` sees
__device__ __forceinline__ int row_limit(const PackedArgs& a, int past, int t) {
  const i64 l = (i64)::max(past, 0) + t;
  return (int)imin(l, (i64)a.S - 1);
}

// threadIdx.x as a value of its own: what follows from it is made anew for each item
// of a block, not held in registers across them
__device__ __forceinline__ int thread_now() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// Inclusive sum over the lanes: within rows of 16 (row shifts by 1, 2, 4, 8),
// then the rows' totals (broadcasts of lanes 15 and 31)
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
}

// Every LDS read of the wave done (before a barrier that frees what it read)
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(0xC07F); }

// The rows' work, found by every wave for itself: lane l holds row b0 + l of 64.
// A row's items are its units times its chunks.
struct Rows {
  int tok0, T, past, over, units, nc;  // the lane's row
  int items, units_to, items_to;       // its items; units and items up to and with it
  __device__ __forceinline__ void load(const PackedArgs& a, int b0) {
    const int b = b0 + (int)(threadIdx.x & 63), bc = ::min(b, a.B - 1);
    past = a.past[bc];
    const int c0 = ::min(::max(a.cu[bc], 0), a.N), c1 = ::min(::max(a.cu[bc + 1], c0), a.N);
    tok0 = c0;
    over = b < a.B && c1 - c0 > a.max_new;
    T = b < a.B ? ::min(c1 - c0, a.max_new) : 0;
    const i64 R = (i64)T << a.lg;
    units = R <= 16 ? (T > 0 ? 1 : 0) : ::min((int)((R + 63) >> 6), a.units);
    nc = (row_limit(a, past, T - 1) + a.chunk) / a.chunk;
    items = units * nc;
    units_to = wave_scan(units);
    items_to = wave_scan(items);
  }
};

// Items from the last row's last unit on (the tiles of a prompt that see most go
// first), kv heads fastest (with 8 of them a head's blocks share an XCD, so its L2
// holds their K and V). A block takes item j, j + a.step, ...
// Rows that overlap (a cu that is not ascending) can ask for more than a.units: items
// past a.units nch are dropped (so no sum passes 2^31), and units past a.units (outside()).
struct Finder {
  int total;  // items
  int ntok;   // token rows of all rows
  // r: the first 64 rows (all of most batches)
  __device__ __forceinline__ Finder(const PackedArgs& a, Rows& r) {
    ntok = ::min(::max(a.cu[a.B], 0), a.N);
    r.load(a, 0);
    const int most = a.units * a.nch;  // at most 2^24
    total = ::min(__builtin_amdgcn_readlane(r.items_to, 63), most);
    u64 over = __ballot(r.over != 0);
    for (int b0 = 64; b0 < a.B; b0 += 64) {
      Rows x;
      x.load(a, b0);
      total = ::min(total + __builtin_amdgcn_readlane(x.items_to, 63), most);
      over |= __ballot(x.over != 0);
    }
    // rows of more tokens than the bound (which may have no item)
    if (DI_UNLIKELY(over != 0) && blockIdx.x == 0 && threadIdx.x == 0 && a.err)
      atomicOr(a.err, DI_ERR_SLOTS);
  }
  // item j of kv head kvh; x: the first 64 rows
  __device__ __forceinline__ Work find(const PackedArgs& a, Rows x, int kvh, int j) const {
    Work w{};
    w.kvh = kvh;
    const int item = total - 1 - j;
    int items = 0, units = 0, b0 = 0;
    for (;;) {
      const int tot = __builtin_amdgcn_readlane(x.items_to, 63);
      if (item < items + tot || b0 + 64 >= a.B) break;
      items += tot;
      units += __builtin_amdgcn_readlane(x.units_to, 63);
      b0 += 64;
      x.load(a, b0);
    }
    const int l = __ffsll((unsigned long long)__ballot(items + x.items_to > item)) - 1;
    auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
    const int nc = of(x.nc), at = item - items - (of(x.items_to) - of(x.items));
    w.b = b0 + l;
    w.tile = at / nc;
    w.c = at - w.tile * nc;
    w.unit = units + of(x.units_to) - of(x.units) + w.tile;
    w.tok0 = of(x.tok0);
    w.T = of(x.T);
    const int past = of(x.past);
    w.bad = past < 0 || (i64)past + w.T > (i64)a.S;
    w.past = ::max(past, 0);
    w.len = row_limit(a, w.past, w.T - 1) + 1;
    w.few = (w.T << a.lg) <= 16;
    return w;
  }
};

// Slots outside the launch's bound: DI_ERR_SLOTS, once a row
__device__ __forceinline__ void report_row(const PackedArgs& a, const Work& w) {
  if (w.bad && w.tile == 0 && w.kvh == 0 && w.c == 0 && threadIdx.x == 0 && a.err)
    atomicOr(a.err, DI_ERR_SLOTS);
}

// A unit that the launch has no room for (rows that overlap)
__device__ __forceinline__ bool outside(const PackedArgs& a, const Work& w) {
  if (DI_LIKELY(w.unit < a.units)) return false;
  if (threadIdx.x == 0 && a.err) atomicOr(a.err, DI_ERR_SLOTS);
  return true;
}

// Token rows behind the last row's: zeros, shared among the blocks
__device__ __forceinline__ void zero_tail(const PackedArgs& a, int ntok, int kvh, int j) {
  const int cols = 128 << a.lg;
  for (int tok = ntok + j; tok < a.N; tok += a.step) {
    int64_t* o = a.out + ((i64)tok * a.n_kv + kvh) * cols;
    for (int i = threadIdx.x; i < cols; i += 256) o[i] = 0;
  }
}

// The page of row b's slots [128 j, 128 j + 128): -1 when not mapped
__device__ __forceinline__ int packed_page(const PackedArgs& a, int b, int j) {
  const int pg = j < a.kv.width ? a.kv.table[(i64)b * a.kv.width + j] : -1;
  return pg < a.n_pages ? pg : -1;
}

// ---- DI-Exp and probabilities of a query row
//
// For tpos < 2^17 (a wave's rows decide together; else the integer forms):
// with n = m - s >= 0, t = tpos, sp = t - n, the exponential is
// e = ((q + 1) t + sp) >> (q + 1) = ((q + 2) t - n) >> (q + 1), q = n div t
// (intops.h, dexp_est): what is shifted is 2 t - n mod t, above t and at most
// 2 t < 2^18. The scores' accumulators start from 0x4B400000 + t - m, so that they
// arrive as the bits of the float 1.5 2^23 + sp (|sp| < 2^22: |n| <= 2^22), whose
// low 22 bits the multiply-add and the AND leave. Then
//   x = clamp01(b - sp a), a = fl(1 / 31 t), b = fl((1.5 + 0.5 / t) / 31):
//     31 x is (n + 0.5) / t + 0.5 within 2^-18.3 where that is below 31 (a, b and
//     the fma are off by at most half a step, on values up to 32 / 31), and a
//     quotient (n + 0.5) / t + 0.5 is at least 0.5 / t >= 2^-18 from the next half-integer,
//   so fma(x, 31, 2^23) rounds to 2^23 + q + 1, q + 1 in its low bits.
// From 31 on the shift is 31 and (31 t + sp) in 22 bits, whatever its sign,
// shifts to the 0 that e is there. Of these operations the fmas, the
// subtraction, the AND and the shift issue in two cycles a wave, the multiply-add
// in four: 17 cycles against 26 through doubles (conversions, and the minimum of
// the shift).
//
// p = floor((e 2^14 + floor(den / 2)) / den) is e 2^14 / den rounded to nearest,
// halves up (for odd den there are none). In double, r = fl(2^14 / den) (1 + 2^-50)
// and fma(e, r, 2^52 + 128) rounds e r once, to an integer: a half goes up, since
// r exceeds 2^14 / den by 2^-51 of it at least, and another value is 1 / (2 den) from the
// next half, more than the 2^14 2^-49 that r adds, as den <= S t < 2^34. The low word
// is p + 128: its second byte H and its first L give p = 256 H + (L - 128), and
// L - 128 as a byte is L ^ 0x80, so the bytes are two int8 operands.
struct RowExp {
  float a, b;
  uint32_t t;
  int32_t c0;  // the accumulators' start
};
constexpr i64 FAST_T = (i64)1 << 17;

__device__ __forceinline__ RowExp make_rowexp(i64 t, int32_t mx) {
  RowExp E;
  const double d = (double)t;
  E.a = (float)(1.0 / (31.0 * d));
  E.b = (float)((1.5 + 0.5 / d) / 31.0);
  E.t = (uint32_t)t;
  E.c0 = (int32_t)(0x4B400000u + (uint32_t)t - (uint32_t)mx);
  return E;
}
__device__ __forceinline__ uint32_t row_exp(int32_t F, const RowExp& E) {
  const float sp = __builtin_bit_cast(float, F) - 12582912.0f;
  const float x = __builtin_amdgcn_fmed3f(__builtin_fmaf(sp, -E.a, E.b), 0.0f, 1.0f);
  const uint32_t y = __builtin_bit_cast(uint32_t, __builtin_fmaf(x, 31.0f, 8388608.0f));
  return (mad_u24(y, E.t, (uint32_t)F) & 0x3FFFFFu) >> (y & 31u);
}
// Of 16 scores, eight at a time, step by step: each step waits for the one before,
// so eight chains run side by side
__device__ __forceinline__ void row_exps(const v4i (&st)[4], const RowExp& E, uint32_t (&e)[16]) {
#pragma unroll
  for (int h = 0; h < 16; h += 8) {
    int32_t F[8];
    float x[8];
    uint32_t m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) F[i] = st[(h + i) >> 2][i & 3];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_bit_cast(float, F[i]) - 12582912.0f;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] = __builtin_amdgcn_fmed3f(__builtin_fmaf(x[i], -E.a, E.b), 0.0f, 1.0f);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_fmaf(x[i], 31.0f, 8388608.0f);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      m[i] = mad_u24(__builtin_bit_cast(uint32_t, x[i]), E.t, (uint32_t)F[i]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] &= 0x3FFFFFu;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[h + i] = m[i] >> (__builtin_bit_cast(uint32_t, x[i]) & 31u);
  }
}

__device__ __forceinline__ double make_rowp(i64 den) {
  const double r = 16384.0 / (double)den;
  return fma(r, 0x1p-50, r);
}
// The P operands of 16 exponentials
__device__ __forceinline__ void pack4(const uint32_t (&w)[4], int& hi, int& lo);
__device__ __forceinline__ void row_probs(const uint32_t (&e)[16], double r, v4i& phi, v4i& plo) {
#pragma unroll
  for (int h = 0; h < 16; h += 8) {
    double d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = (double)e[h + i];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = fma(d[i], r, 0x1p52 + 128.0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__builtin_bit_cast(u64, d[4 * q + i]);
      int a, b;
      pack4(w, a, b);
      phi[(h >> 2) + q] = a;
      plo[(h >> 2) + q] = b;
    }
  }
}
// Four words p + 128 as the operands' bytes
__device__ __forceinline__ void pack4(const uint32_t (&w)[4], int& hi, int& lo) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u);  // L0 L1 H0 H1
  const uint32_t b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  lo = (int)(__builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u);
  hi = (int)__builtin_amdgcn_perm(b, a, 0x07060302u);
}

// Any tpos (from 2^17 on, a few instructions a value do not matter): q as in
// dexp_est, whose bound holds for every t >= 1 with n <= 2^22 (from t = 2^23 on n / t
// is at most a half), the rest in 64 bits. The sums that wrap wrap as the
// reference's do.
__device__ __forceinline__ i64 slow_exp(int32_t st, int32_t mx, i64 t) {
  const uint32_t n = (uint32_t)(mx - st);
  const uint32_t q1 = (uint32_t)fma((double)n, 1.0 / (double)t, 1.0 + 0x1p-26);
  const u64 m = (u64)q1 * (u64)t + (u64)t - n;
  return q1 < 64u ? (i64)(m >> q1) : 0;
}
__device__ __forceinline__ uint32_t slow_p128(i64 e, i64 den) {
  return (uint32_t)to_i32(rhad(shl(e, 14), den)) + 128u;
}

// 16 values of a lane that a loop reads and writes at a number of its own: a
// vector, or LDS (a wave's [16][64] words)
typedef int v16i __attribute__((ext_vector_type(16)));
struct InRegs {
  v16i x;
  __device__ __forceinline__ int get(int i) const { return x[i]; }
  __device__ __forceinline__ void put(int i, int v) { x[i] = v; }
};
struct InLds {
  int32_t* p;
  __device__ __forceinline__ int get(int i) const { return p[i * 64 + (threadIdx.x & 63)]; }
  __device__ __forceinline__ void put(int i, int v) { p[i * 64 + (threadIdx.x & 63)] = v; }
};
// In the integer forms, a score after the other: the sum of 16 exponentials, and
// their P operands (small code and few registers, for what is hardly ever met)
template <class Mem>
__device__ __forceinline__ i64 slow_den(const v4i (&st)[4], int32_t off, uint32_t bits, int32_t mx,
                                        i64 tpos, Mem m) {
#pragma unroll
  for (int i = 0; i < 16; ++i) m.put(i, st[i >> 2][i & 3] - off);
  i64 den = 0;
#pragma unroll 1
  for (int i = 0; i < 16; ++i)
    if ((bits >> i) & 1u) den = wadd(den, slow_exp(m.get(i), mx, tpos));
  return den;
}
template <class Mem>
__device__ __forceinline__ void slow_probs(const v4i (&st)[4], int32_t off, uint32_t bits,
                                           int32_t mx, i64 tpos, i64 den, v4i& phi, v4i& plo,
                                           Mem m) {
#pragma unroll
  for (int i = 0; i < 16; ++i) m.put(i, st[i >> 2][i & 3] - off);
#pragma unroll 1
  for (int i = 0; i < 16; ++i)
    m.put(i, (bits >> i) & 1u ? (int)slow_p128(slow_exp(m.get(i), mx, tpos), den) : 128);
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const uint32_t w4[4] = {(uint32_t)m.get(4 * b), (uint32_t)m.get(4 * b + 1),
                            (uint32_t)m.get(4 * b + 2), (uint32_t)m.get(4 * b + 3)};
    int a, c;
    pack4(w4, a, c);
    phi[b] = a;
    plo[b] = c;
  }
}

__device__ __forceinline__ int max16(int v) {  // over the lanes of one query row
  v = ::max(v, __shfl_xor(v, 16));
  return ::max(v, __shfl_xor(v, 32));
}

// ------------------------------------------------------------- few-row units
//
// One row, at most 16 query rows (token t and head g: row t G + g). S^T = K . Q^T
// on v_mfma_i32_16x16x64_i8 with K's rows straight from the cache: MFMA row i of
// block blk is slot 16 (i / 4) + 4 blk + i % 4 of a 64-slot tile, so that lane (qi, g4)
// of a wave receives query row qi's scores of the 16 slots 16 g4 .. + 15, which are
// its bytes of the P operand. Each byte of K and V is read once; what bounds it
// is HBM, or, for short rows, one chain of loads and three block reductions. The
// arithmetic of the query rows that are not there (14 of 16 at one token and two
// heads) is 5 cycles a slot and CU against the 31 that its 256 bytes take. Up to 8
// query rows (R8), a lane works for row qi % 8: the P operand has the high bytes in
// rows 0 to 7 and the low bytes in rows 8 to 15, one MFMA and half the accumulators.

template <int NW>
struct FewLds {
  int32_t mx[NW][16];
  int64_t den[NW][16];
  int32_t ctx[16][128];
  int32_t slow[NW][16 * 64];
};

struct FewRow {
  bool on;     // the lane's query row is there
  int limit;   // the last slot it sees (-1: none)
  i64 tpos;
  v4i q0, q1;
};

template <bool R8>
__device__ __forceinline__ FewRow few_row(const PackedArgs& a, const Work& w) {
  const int lane = thread_now() & 63, qi = R8 ? lane & 7 : lane & 15, g4 = lane >> 4;
  FewRow r;
  const int t = qi >> a.lg, g = qi & ((1 << a.lg) - 1);
  r.on = qi < (w.T << a.lg);
  const i64 row = (i64)(w.tok0 + (r.on ? t : 0)) * a.n_q + (w.kvh << a.lg) + g;
  r.limit = r.on ? row_limit(a, w.past, t) : -1;
  const i64 tp = a.tpos[row];
  const v4i q0 = *(const v4i*)(a.q8 + row * 128 + g4 * 16);
  const v4i q1 = *(const v4i*)(a.q8 + row * 128 + 64 + g4 * 16);
  r.tpos = r.on ? tp : 1;
  const v4i z = v4i{0, 0, 0, 0};
  r.q0 = r.on ? q0 : z;
  r.q1 = r.on ? q1 : z;
  return r;
}

// K operands of the 64-slot half hf of a page (a page that is not there reads page 0)
__device__ __forceinline__ void few_k(const PackedArgs& a, int pg, int kvh, int hf, v4i (&k)[8]) {
  const int lane = thread_now() & 63, qi = lane & 15, g4 = lane >> 4;
  const int8_t* p = a.kv.krow(::max(pg, 0), kvh, hf * 64 + 16 * (qi >> 2) + (qi & 3)) + g4 * 16;
#pragma unroll
  for (int blk = 0; blk < 4; ++blk) {
    k[2 * blk] = *(const v4i*)(p + blk * 512);
    k[2 * blk + 1] = *(const v4i*)(p + blk * 512 + 64);
  }
}
// V operands: channel 16 j + qi, slots 16 g4 .. + 15 of the half
template <int J0 = 0, int J1 = 8>
__device__ __forceinline__ void few_v(const PackedArgs& a, int pg, int kvh, int hf, v4i (&v)[8]) {
  const int lane = thread_now() & 63, qi = lane & 15, g4 = lane >> 4;
  const int8_t* p = a.kv.vchan(::max(pg, 0), kvh, qi) + hf * 64 + g4 * 16;
#pragma unroll
  for (int j = J0; j < J1; ++j) v[j] = *(const v4i*)(p + j * 16 * DI_PAGE);
}
__device__ __forceinline__ void few_scores(const v4i (&k)[8], const FewRow& r, v4i (&st)[4]) {
  const v4i z = v4i{0, 0, 0, 0};
#pragma unroll
  for (int blk = 0; blk < 4; ++blk) st[blk] = mfma16(k[2 * blk], r.q0, z);
#pragma unroll
  for (int blk = 0; blk < 4; ++blk) st[blk] = mfma16(k[2 * blk + 1], r.q1, st[blk]);
}
// bit i: the lane's query row sees slot s0 + i, i < 16
__device__ __forceinline__ uint32_t seen16(int limit, int s0) {
  const int e = limit - s0;
  return e >= 15 ? 0xFFFFu : (e < 0 ? 0u : (2u << e) - 1u);
}

// sum p v of a tile into the accumulators
__device__ __forceinline__ void pv16(const v4i& phi, const v4i& plo, const v4i (&v)[8], v4i (&hi)[8],
                                     v4i (&lo)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    hi[j] = mfma16(phi, v[j], hi[j]);
    lo[j] = mfma16(plo, v[j], lo[j]);
  }
}
template <bool R8>
struct FewAcc {
  v4i hi[8], lo[R8 ? 1 : 8];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < 8; ++j) hi[j] = v4i{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < (R8 ? 1 : 8); ++j) lo[j] = v4i{0, 0, 0, 0};
  }
  // channel blocks [J0, J1)
  template <int J0 = 0, int J1 = 8>
  __device__ __forceinline__ void add(const v4i& phi, const v4i& plo, const v4i (&v)[8]) {
    if constexpr (R8) {
      const v4i p = (threadIdx.x & 8) ? plo : phi;
#pragma unroll
      for (int j = J0; j < J1; ++j) hi[j] = mfma16(p, v[j], hi[j]);
    } else {
#pragma unroll
      for (int j = J0; j < J1; ++j) {
        hi[j] = mfma16(phi, v[j], hi[j]);
        lo[j] = mfma16(plo, v[j], lo[j]);
      }
    }
  }
};

// The tile's operands from its 16 scores a lane (raw; `bits` of them are seen)
__device__ __forceinline__ void few_probs(const v4i (&st)[4], uint32_t bits, bool fast,
                                          const RowExp& E, double rp, int32_t mx, i64 tpos, i64 den,
                                          v4i& phi, v4i& plo, InLds m) {
  if (DI_UNLIKELY(!fast)) {
    slow_probs(st, 0, bits, mx, tpos, den, phi, plo, m);
    return;
  }
  v4i f[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) f[b] = st[b] + E.c0;
  uint32_t e[16];
  row_exps(f, E, e);
#pragma unroll
  for (int i = 0; i < 16; ++i) e[i] = (bits >> i) & 1u ? e[i] : 0u;
  row_probs(e, rp, phi, plo);
}
__device__ __forceinline__ i64 few_den(const v4i (&st)[4], uint32_t bits, bool fast, const RowExp& E,
                                       int32_t mx, i64 tpos, InLds m) {
  if (DI_UNLIKELY(!fast)) return slow_den(st, 0, bits, mx, tpos, m);
  v4i f[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) f[b] = st[b] + E.c0;
  uint32_t e[16], sum = 0;
  row_exps(f, E, e);
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += (bits >> i) & 1u ? e[i] : 0u;
  return sum;
}

// The waves' contexts (accumulators of operand row 4 g4 + r, channel 16 j + qi)
// added up in LDS, then written: to out, to a chunk's part, or (where the launch has
// only few-row units) added to out, which the first pass cleared: integers, so in
// any order
template <int NW, bool R8>
__device__ __forceinline__ void few_store(const PackedArgs& a, const Work& w, FewLds<NW>& lds,
                                          const FewAcc<R8>& c, bool any) {
  const int lane = thread_now() & 63, qi = lane & 15, g4 = lane >> 4;
  const int R = w.T << a.lg;
  if (any) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = R8 ? (4 * g4 + r) & 7 : 4 * g4 + r;
        int x;
        if constexpr (R8) x = g4 < 2 ? c.hi[j][r] * 256 : c.hi[j][r];
        else x = c.hi[j][r] * 256 + c.lo[j][r];
        if (row < R) atomicAdd(&lds.ctx[row][16 * j + qi], x);
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * 128; i += NW * 64) {
    const int row = i >> 7, t = row >> a.lg, g = row & ((1 << a.lg) - 1);
    const i64 at = ((i64)(w.tok0 + t) * a.n_q + (w.kvh << a.lg) + g) * 128 + (i & 127);
    const int x = lds.ctx[row][i & 127];
    if (a.part) a.part[(i64)w.c * a.N * a.n_q * 128 + at] = x;
    else if (a.nch > 1) atomicAdd((unsigned long long*)&a.out[at], (unsigned long long)(i64)x);
    else a.out[at] = x;
  }
}

// A whole row of at most 64 NW NT slots: tile i of wave v is tile i NW + v
template <int NW, int NT, bool R8>
__device__ __forceinline__ void few_one(const PackedArgs& a, const Work& w, FewLds<NW>& lds) {
  const int lane = threadIdx.x & 63, qi = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int ntiles = (w.len + 63) / 64;
  int pg[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int it = i * NW + wave;
    pg[i] = it < ntiles ? packed_page(a, w.b, it >> 1) : -1;
  }
  const FewRow row = few_row<R8>(a, w);
  for (int i = threadIdx.x; i < 16 * 128; i += NW * 64) ((int32_t*)lds.ctx)[i] = 0;
  v4i st[NT][4];
  {
    v4i k[NT][8];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      pg[i] = __builtin_amdgcn_readfirstlane(pg[i]);
      if (i * NW + wave < ntiles) few_k(a, pg[i], w.kvh, (i * NW + wave) & 1, k[i]);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
      if (i * NW + wave < ntiles) few_scores(k[i], row, st[i]);
  }
  // the first V operands load under the reductions
  v4i v0[8];
  if (wave < ntiles) few_v(a, pg[0], w.kvh, wave & 1, v0);
  auto bits = [&](int i) {
    const int it = i * NW + wave;
    return it < ntiles && pg[i] >= 0 ? seen16(row.limit, it * 64 + 16 * g4) : 0u;
  };
  int mx = NO_SCORE;
#pragma unroll
  for (int i = 0; i < NT; ++i)
    if (i * NW + wave < ntiles) {
      const uint32_t bb = bits(i);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if ((bb >> e) & 1u) mx = ::max(mx, st[i][e >> 2][e & 3]);
    }
  mx = max16(mx);
  if (g4 == 0) lds.mx[wave][qi] = mx;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < NW; ++v) mx = ::max(mx, lds.mx[v][qi]);
  if (mx == NO_SCORE) mx = 0;  // nothing seen: max := 0, every p = 0
  const bool fast = __ballot(row.tpos >= FAST_T) == 0;
  const RowExp E = make_rowexp(row.tpos, mx);
  i64 den = 0;
#pragma unroll
  for (int i = 0; i < NT; ++i)
    if (i * NW + wave < ntiles) den = wadd(den, few_den(st[i], bits(i), fast, E, mx, row.tpos, {lds.slow[wave]}));
  den = group4_sum(den);
  if (g4 == 0) lds.den[wave][qi] = den;
  __syncthreads();
  den = 0;
#pragma unroll
  for (int v = 0; v < NW; ++v) den = wadd(den, lds.den[v][qi]);
  den = imax(den, 1);
  const double rp = make_rowp(den);
  FewAcc<R8> acc;
  acc.clear();
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int it = i * NW + wave;
    if (it < ntiles) {
      v4i v[8], phi, plo;
      if (i > 0) few_v(a, pg[i], w.kvh, it & 1, v);
      few_probs(st[i], bits(i), fast, E, rp, mx, row.tpos, den, phi, plo, {lds.slow[wave]});
      acc.add(phi, plo, i > 0 ? v : v0);
    }
  }
  few_store<NW, R8>(a, w, lds, acc, wave < ntiles);
}

// The place of a unit's chunk in smax and sden
__device__ __forceinline__ i64 cell(const PackedArgs& a, const Work& w, int c) {
  return (((i64)w.unit * a.n_kv + w.kvh) * a.nch + c) * 64;
}
// Over a row's chunks [0, nc): the maximum and, with DEN, the denominator of query
// row i of the unit (lanes that share i take chunks in turn)
template <bool DEN>
__device__ __forceinline__ void over_chunks(const PackedArgs& a, const Work& w, int nc, int i,
                                            int32_t* mx, i64* den) {
  const int g4 = (threadIdx.x & 63) >> 4;
  int m = NO_SCORE;
  i64 d = 0;
  for (int c0 = 0; c0 < nc; c0 += 16) {
    int x[4];
    i64 y[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = ::min(c0 + 4 * u + g4, nc - 1);
      const i64 at = cell(a, w, c) + i;
      x[u] = a.smax[at];
      if (DEN) y[u] = a.sden[at];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      m = ::max(m, x[u]);
      if (DEN && c0 + 4 * u + g4 < nc) d = wadd(d, y[u]);
    }
  }
  m = max16(m);
  *mx = m == NO_SCORE ? 0 : m;
  if (DEN) *den = imax(group4_sum(d), 1);
}

// One pass over chunk w.c of a few-row unit, NW waves
template <int PH, int NW, bool R8>
__device__ __forceinline__ void few_phase(const PackedArgs& a, const Work& w, FewLds<NW>& lds) {
  const int tid = thread_now(), lane = tid & 63, qi = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lo_s = w.c * a.chunk, hi_s = ::min(w.len, lo_s + a.chunk);
  if (lo_s >= hi_s) return;
  const int R = w.T << a.lg, nc = (w.len + a.chunk - 1) / a.chunk;
  const i64 pitch = (i64)a.nch * a.chunk;
  const i64 row0 = a.few_rows ? (i64)w.b * a.few_rows : (i64)w.tok0 << a.lg;
  int32_t* const sc = a.scores + ((i64)w.kvh * a.score_rows + row0) * pitch;
  const int t0 = lo_s / 64, t1 = (hi_s + 63) / 64;
  if constexpr (PH == PH_MAX) {
    if (w.c == 0 && !a.part && a.nch > 1)
      for (int i = threadIdx.x; i < R * 128; i += NW * 64)
        a.out[((i64)(w.tok0 + (i >> 7 >> a.lg)) * a.n_q + (w.kvh << a.lg) +
               ((i >> 7) & ((1 << a.lg) - 1))) * 128 + (i & 127)] = 0;
    const FewRow row = few_row<false>(a, w);
    int mx = NO_SCORE;
    // two tiles of K in flight a wave
    for (int it = t0 + wave; it < t1; it += 2 * NW) {
      v4i k[2][8];
      int pg[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
        pg[u] = __builtin_amdgcn_readfirstlane(it + NW * u < t1 ? packed_page(a, w.b, (it + NW * u) >> 1) : -1);
#pragma unroll
      for (int u = 0; u < 2; ++u) few_k(a, pg[u], w.kvh, (it + NW * u) & 1, k[u]);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int x = it + NW * u;
        if (x < t1) {
          v4i st[4];
          few_scores(k[u], row, st);
          const uint32_t bb = pg[u] >= 0 ? seen16(row.limit, x * 64 + 16 * g4) : 0u;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            int& s = ((int*)&st[e >> 2])[e & 3];
            s = (bb >> e) & 1u ? s : NO_SCORE;
            mx = ::max(mx, s);
          }
          if (row.on) {
            v4i* o = (v4i*)(sc + qi * pitch + x * 64 + 16 * g4);
#pragma unroll
            for (int blk = 0; blk < 4; ++blk) o[blk] = st[blk];
          }
        }
      }
    }
    mx = max16(mx);
    if (g4 == 0) lds.mx[wave][qi] = mx;
    __syncthreads();
    if (threadIdx.x < 16) {
#pragma unroll
      for (int v = 0; v < NW; ++v) mx = ::max(mx, lds.mx[v][qi]);
      a.smax[cell(a, w, w.c) + qi] = mx;
    }
  } else if constexpr (PH == PH_DEN) {
    // a query row a wave, four slots a lane and load (chunks end on whole tiles)
    for (int r = wave; r < R; r += NW) {
      int m = NO_SCORE;
      for (int c = lane; c < nc; c += 64) m = ::max(m, a.smax[cell(a, w, c) + r]);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) m = ::max(m, __shfl_xor(m, d));
      const int mx = m == NO_SCORE ? 0 : m;
      const int t = r >> a.lg, g = r & ((1 << a.lg) - 1);
      const i64 tpos = a.tpos[(i64)(w.tok0 + t) * a.n_q + (w.kvh << a.lg) + g];
      const bool fast = tpos < FAST_T;  // (one row: uniform)
      const RowExp E = make_rowexp(fast ? tpos : 1, mx);
      const int32_t* src = sc + r * pitch;
      i64 den = 0;
      for (int s0 = lo_s + 4 * lane; s0 < t1 * 64; s0 += 1024) {
        v4i x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = *(const v4i*)(src + (s0 + 256 * u < t1 * 64 ? s0 + 256 * u : s0));
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (s0 + 256 * u < t1 * 64) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int v = x[u][i];
              if (fast) {
                const uint32_t e = row_exp(v + E.c0, E);
                den += v == NO_SCORE ? 0u : e;
              } else if (v != NO_SCORE) {
                den = wadd(den, slow_exp(v, mx, tpos));
              }
            }
          }
      }
      den = wave_sum(den);
      if (lane == 0) a.sden[cell(a, w, w.c) + r] = den;
    }
  } else {
    const FewRow row = few_row<R8>(a, w);
    const int ri = R8 ? qi & 7 : qi;  // the lane's query row
    const int32_t* src = sc + (row.on ? ri : 0) * pitch + 16 * g4;
    for (int i = threadIdx.x; i < 16 * 128; i += NW * 64) ((int32_t*)lds.ctx)[i] = 0;
    int32_t mx;
    i64 den;
    over_chunks<true>(a, w, nc, ri, &mx, &den);
    if (!row.on) {
      mx = 0;
      den = 1;
    }
    const bool fast = __ballot(row.tpos >= FAST_T) == 0;
    const RowExp E = make_rowexp(row.tpos, mx);
    const double rp = make_rowp(den);
    FewAcc<R8> acc;
    acc.clear();
    __syncthreads();  // ctx is zero
    for (int it = t0 + wave; it < t1; it += NW) {
      v4i v[8], st[4];
      const int pg = __builtin_amdgcn_readfirstlane(packed_page(a, w.b, it >> 1));
#pragma unroll
      for (int blk = 0; blk < 4; ++blk) st[blk] = *(const v4i*)(src + it * 64 + 4 * blk);
      // (half of V waits until the scores' registers are free)
      few_v<0, 4>(a, pg, w.kvh, it & 1, v);
      uint32_t bb = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) bb |= (st[e >> 2][e & 3] != NO_SCORE ? 1u : 0u) << e;
      v4i phi, plo;
      few_probs(st, row.on ? bb : 0u, fast, E, rp, mx, row.tpos, den, phi, plo, {lds.slow[wave]});
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (R8) {
        few_v<4, 8>(a, pg, w.kvh, it & 1, v);
        acc.add(phi, plo, v);
      } else {
        acc.template add<0, 4>(phi, plo, v);
        few_v<4, 8>(a, pg, w.kvh, it & 1, v);
        acc.template add<4, 8>(phi, plo, v);
      }
    }
    few_store<NW, R8>(a, w, lds, acc, true);
  }
}

// ------------------------------------------------------------- 64 query rows
//
// Four waves of 16 query rows (row i: token i / G, head i % G of the kv head, so K
// and V are read once for the kv head's query heads). Keys reach LDS by
// direct-to-LDS loads into a ring of three 16 KB steps: a page of K in the first two
// passes, half a page of K and V in the third; one barrier a step, 16-byte chunks
// swizzled against bank conflicts.
//
// What bounds it is issue. Alone on a SIMD a wave takes some 240, 670 and 1520
// cycles for a half page's three passes, two side by side 170, 460 and 1050, so a
// prompt of 2500 tokens (632 tiles of up to 40 half pages, 68 us) is bound by its last
// tiles' own chains; its loads alone take 30 us. Three blocks a CU (168 registers a lane,
// none spilled: scratch memory cost a launch 8 us by itself, and two waves more a
// SIMD at 128 registers did not make up for it).

constexpr int TL_HALF = 8 * 1024;   // 64 slot rows of K, or 64 slots of V's 128 channels
constexpr int TL_PAGE = 16 * 1024;  // a page of K, or of V

constexpr int TL_STEPS = 3;

union TileLds {
  __attribute__((aligned(1024))) int8_t ring[TL_STEPS * TL_PAGE];
  FewLds<4> few;
};

// Physical chunk = logical ^ swizzle, so that the operand reads below take LDS's
// full rate (eight lanes at a time over 128 bytes). K (rows of 8 chunks): bits 0, 1
// and 4 of the row. Half pages of V (channel rows of 4 chunks): bits 1 and 2 of the
// channel.
__device__ __forceinline__ int tl_kswz(int row) { return (row & 3) | ((row >> 2) & 4); }
__device__ __forceinline__ int tl_vswz(int d) { return (d >> 1) & 3; }

// The page ids of a row's pages from p on, 64 of them in the lanes of a register,
// the next 64 when they come up
struct PageIds {
  int v, base;
  __device__ __forceinline__ void load(const PackedArgs& a, int b, int p) {
    base = p;
    v = packed_page(a, b, p + (int)(threadIdx.x & 63));
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt 0: here, not at every use
  }
  __device__ __forceinline__ int get(const PackedArgs& a, int b, int p) {
    if (DI_UNLIKELY(p - base >= 64 || p < base)) load(a, b, p);
    return __builtin_amdgcn_readlane(v, p - base);
  }
};

template <int PH>
__device__ __forceinline__ void tile_body(const PackedArgs& a, const Work& w, TileLds& lds) {
  const int tid = thread_now(), lane = tid & 63, qi = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = w.T << a.lg;             // the row's query rows
  const int r0 = w.tile * 64;            // the tile's first
  const int rl = ::min(r0 + 63, R - 1);  // and last
  // the tile's slots, and the chunk's of those
  const int end = row_limit(a, w.past, rl >> a.lg) + 1;
  const int lo_s = PH == PH_ALL ? 0 : w.c * a.chunk;
  const int hi_s = PH == PH_ALL ? end : ::min(end, lo_s + a.chunk);
  if (lo_s >= hi_s) return;
  const int p0 = lo_s / DI_PAGE, np = (hi_s + DI_PAGE - 1) / DI_PAGE - p0;
  PageIds ids;
  ids.load(a, w.b, p0);
  const int wr0 = r0 + wave * 16;            // the wave's first query row
  const bool work = wr0 < R;               // (waves without one only load)
  const int qr = ::min(wr0 + qi, R - 1);   // the lane's (rows past the last: the last, not stored)
  const int limit = row_limit(a, w.past, qr >> a.lg);
  const int wlim = row_limit(a, w.past, ::min(wr0, R - 1) >> a.lg);        // the wave's smallest
  const int wmax = row_limit(a, w.past, ::min(wr0 + 15, R - 1) >> a.lg);   // and largest limit
  // the half pages that the wave sees: [0, nsee)
  const int nsee = work && wmax >= lo_s ? (wmax - p0 * DI_PAGE) / 64 + 1 : 0;

  u64 there = 0;  // of the last 64 pages asked for, those that are mapped
  auto page_of = [&](int i) {
    const int pg = ids.get(a, w.b, p0 + i);
    const u64 bit = 1ull << (i & 63);
    there = pg < 0 ? there & ~bit : there | bit;
    return pg;
  };
  // (a page that is not there: a view of no bytes, whose loads read 0)
  auto view = [&](const int8_t* pool, int pg) {
    return __builtin_amdgcn_make_buffer_rsrc(
        (void*)(pool + ((i64)::max(pg, 0) * a.n_kv + w.kvh) * TL_PAGE), (short)0,
        pg < 0 ? 0 : TL_PAGE, 0x00020000);
  };
  auto k_off = [&](int row) { return row * 128 + ((lane & 7) ^ tl_kswz(row)) * 16; };
  // a page of K to `to`: each load of a wave brings 8 rows, 1 KB
  auto issue_k = [&](int i, int8_t* to) {
    const auto rs = view(a.kv.k, page_of(i));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = wave * 4 + j;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(to + at * 1024), 16,
                                               k_off(at * 8 + (lane >> 3)), 0, 0, 0);
    }
  };
  // half hf of page i, K then V, to `to`: of each, a wave's two loads bring 1 KB, 8
  // rows of K or 16 channels of V
  auto issue_kv = [&](int i, int hf, int8_t* to) {
    const int pg = page_of(i);
    const auto ks = view(a.kv.k, pg), vs = view(a.kv.v, pg);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int at = wave * 2 + j, d = at * 16 + (lane >> 2);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ks, (lds_ptr_t)(to + at * 1024), 16,
                                               k_off(at * 8 + (lane >> 3)), hf * TL_HALF, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vs, (lds_ptr_t)(to + TL_HALF + at * 1024), 16,
                                               d * DI_PAGE + ((lane & 3) ^ tl_vswz(d)) * 16,
                                               hf * 64, 0, 0);
    }
  };
  const i64 qrow = (i64)(w.tok0 + (qr >> a.lg)) * a.n_q + (w.kvh << a.lg) + (qr & ((1 << a.lg) - 1));
  const v4i qf0 = *(const v4i*)(a.q8 + qrow * 128 + g * 16);
  const v4i qf1 = *(const v4i*)(a.q8 + qrow * 128 + 64 + g * 16);
  const i64 tpos = a.tpos[qrow];
  // one page stays for all three passes
  const bool resident = PH == PH_ALL && np == 1;
  if (resident)
    for (int h = 0; h < 2; ++h) issue_kv(0, h, lds.ring + h * TL_PAGE);
  wait_vmcnt<0>();  // (queries, before the ring's loads count)
  if (resident) __syncthreads();
  const int kr = 16 * (qi >> 2) + (qi & 3);
  const int k0 = kr * 128 + ((g ^ tl_kswz(kr)) << 4);
  const int k1 = kr * 128 + (((g + 4) ^ tl_kswz(kr)) << 4);
  // half page i is there, and some query row of the wave sees it
  auto seen = [&](int i) { return i < nsee && ((there >> ((i >> 1) & 63)) & 1) != 0; };
  // its K operands (its K rows at p), and the wave's scores from accumulators z
  auto load_k = [&](const int8_t* p, v4i (&kf)[8]) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      kf[2 * b] = *(const v4i*)(p + k0 + b * 512);
      kf[2 * b + 1] = *(const v4i*)(p + k1 + b * 512);
    }
  };
  auto scores = [&](const v4i (&kf)[8], const v4i z, v4i (&st)[4]) {
#pragma unroll
    for (int b = 0; b < 4; ++b) st[b] = mfma16(kf[2 * b], qf0, z);
#pragma unroll
    for (int b = 0; b < 4; ++b) st[b] = mfma16(kf[2 * b + 1], qf1, st[b]);
  };
  // n steps of four loads a wave: issue(i, where). A wave waits for its own loads of
  // a step (they complete in order), then a barrier publishes every wave's
  // part and frees what the next issue overwrites; body(i, where) with it in LDS.
  auto pass = [&](int n, auto&& issue, auto&& body) {
    wait_lds();
    __builtin_amdgcn_s_barrier();  // the pass before is done with the ring
#pragma unroll
    for (int i = 0; i < TL_STEPS - 1; ++i)
      if (i < n) issue(i, lds.ring + i * TL_PAGE);
    int at = 0;  // the place of step i
    for (int i = 0; i < n; ++i) {
      if (i + 1 < n) wait_vmcnt<4>();
      else wait_vmcnt<0>();
      wait_lds();
      __builtin_amdgcn_s_barrier();
      if (i + TL_STEPS - 1 < n)
        issue(i + TL_STEPS - 1, lds.ring + (at == 0 ? TL_STEPS - 1 : at - 1) * TL_PAGE);
      body(i, lds.ring + at * TL_PAGE);
      at = at + 1 == TL_STEPS ? 0 : at + 1;
    }
  };
  auto first_slot = [&](int i) { return p0 * DI_PAGE + i * 64; };
  auto k_pass = [&](const v4i z, auto&& fn) {
    auto one = [&](int i, const int8_t* p) {
      if (!seen(i)) return;
      v4i kf[8], st[4];
      load_k(p, kf);
      scores(kf, z, st);
      fn(st, first_slot(i));
    };
    if (resident) {
      for (int i = 0; i < 2; ++i) one(i, lds.ring + i * TL_PAGE);
    } else {
      pass(np, issue_k, [&](int i, const int8_t* p) {
#pragma unroll
        for (int h = 0; h < 2; ++h) one(2 * i + h, p + h * TL_HALF);
      });
    }
  };

  int32_t mx = NO_SCORE;
  if constexpr ((PH & PH_MAX) != 0) {
    k_pass(v4i{0, 0, 0, 0}, [&](const v4i (&st)[4], int s0) {
      if (s0 + 63 <= wlim) {
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = ::max(mx, st[e >> 2][e & 3]);
      } else {
        const uint32_t bits = seen16(limit, s0 + 16 * g);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if ((bits >> e) & 1u) mx = ::max(mx, st[e >> 2][e & 3]);
      }
    });
    mx = max16(mx);
    if constexpr (PH == PH_MAX) {
      if (work && g == 0) a.smax[cell(a, w, w.c) + wave * 16 + qi] = mx;
      return;
    }
    if (mx == NO_SCORE) mx = 0;  // nothing seen: max := 0, every p = 0
  }
  const int nc = (end + a.chunk - 1) / a.chunk;
  i64 den = 0;
  if constexpr (PH == PH_DEN) over_chunks<false>(a, w, nc, qr - r0, &mx, &den);
  if constexpr (PH == PH_PV) over_chunks<true>(a, w, nc, qr - r0, &mx, &den);

  const bool fast = __ballot(tpos >= FAST_T) == 0;
  const RowExp E = make_rowexp(fast ? tpos : 1, mx);
  // the accumulators of the slow forms start from 0
  const int32_t c0 = fast ? E.c0 : 0;
  const v4i cinit = v4i{c0, c0, c0, c0};
  if constexpr ((PH & PH_DEN) != 0) {
    den = 0;
    // (the slow forms in a loop of their own: what they hold does not weigh on the other)
    if (DI_LIKELY(fast)) {
      k_pass(cinit, [&](const v4i (&st)[4], int s0) {
        uint32_t e[16], sum = 0;
        row_exps(st, E, e);
        if (s0 + 63 <= wlim) {
#pragma unroll
          for (int i = 0; i < 16; ++i) sum += e[i];
        } else {
          const uint32_t bits = seen16(limit, s0 + 16 * g);
#pragma unroll
          for (int i = 0; i < 16; ++i) sum += (bits >> i) & 1u ? e[i] : 0u;
        }
        den += sum;
      });
    } else {
      k_pass(cinit, [&](const v4i (&st)[4], int s0) {
        den = wadd(den, slow_den(st, 0, seen16(limit, s0 + 16 * g), mx, tpos, InRegs{}));
      });
    }
    den = group4_sum(den);
    if constexpr (PH == PH_DEN) {
      if (work && g == 0) a.sden[cell(a, w, w.c) + wave * 16 + qi] = den;
      return;
    }
    den = imax(den, 1);
  }
  const double rp = make_rowp(den);
  v4i ohi[8], olo[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) ohi[j] = olo[j] = v4i{0, 0, 0, 0};
  // V operand of a half page: channel 16 j + qi, slots 16 g .. + 15 (the swizzle of
  // channel 16 j + qi does not depend on j)
  const int v0 = TL_HALF + qi * 64 + ((g ^ tl_vswz(qi)) << 4);
  auto kv_pass = [&](auto&& probs) {
    auto add = [&](int i, const int8_t* p, const v4i (&st)[4]) {
      v4i phi, plo, vf[8];
      probs(st, first_slot(i), phi, plo);
#pragma unroll
      for (int j = 0; j < 8; ++j) vf[j] = *(const v4i*)(p + v0 + j * 1024);
      pv16(phi, plo, vf, ohi, olo);
    };
    auto one = [&](int i, const int8_t* p) {
      if (!seen(i)) return;
      v4i kf[8], st[4];
      load_k(p, kf);
      scores(kf, cinit, st);
      add(i, p, st);
    };
    if (resident) {
      for (int i = 0; i < 2; ++i) one(i, lds.ring + i * TL_PAGE);
    } else {
      pass(2 * np, [&](int i, int8_t* to) { issue_kv(i >> 1, i & 1, to); }, one);
    }
  };
  if (DI_LIKELY(fast)) {
    kv_pass([&](const v4i (&st)[4], int s0, v4i& phi, v4i& plo) {
      uint32_t e[16];
      row_exps(st, E, e);
      if (s0 + 63 > wlim) {
        const uint32_t bits = seen16(limit, s0 + 16 * g);
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = (bits >> i) & 1u ? e[i] : 0u;
      }
      row_probs(e, rp, phi, plo);
    });
  } else {
    kv_pass([&](const v4i (&st)[4], int s0, v4i& phi, v4i& plo) {
      slow_probs(st, 0, seen16(limit, s0 + 16 * g), mx, tpos, den, phi, plo, InRegs{});
    });
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) ohi[j] = ohi[j] * 256 + olo[j];
  if (!work) return;
  // lane (qi, g): query rows 4 g + r of the wave, channel 16 j + qi
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = wr0 + 4 * g + r;
    if (row < R) {
      const i64 at = ((i64)(w.tok0 + (row >> a.lg)) * a.n_q + (w.kvh << a.lg) +
                      (row & ((1 << a.lg) - 1))) * 128 + qi;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (a.part) a.part[(i64)w.c * a.N * a.n_q * 128 + at + 16 * j] = ohi[j][r];
        else a.out[at + 16 * j] = ohi[j][r];
      }
    }
  }
}

}  // namespace
