// Decode attention of a batch whose rows share their first pages (gfx950). No
// counterpart in the reference; every row's integers are those of
// detllm_attn_decode over its own page table.
//
// Attention of one row reads K and V once for the G query heads of a kv head;
// rows behind one prefix read the same bytes B times. Here the prefix is read
// once for all M = B * G queries of a kv head, which also fill the 16 columns of
// the MFMA tiles that one row leaves mostly empty.
//
// DI-Exp is not multiplicative, so partial softmaxes cannot be rescaled and
// joined: a row's true maximum comes first, then its denominator, then p. Four
// launches: the maxima of each part of a row (k_shared_stat<NG, false>), the
// exponentials' sums of each part (<NG, true>), p and P.V of the prefix
// (k_shared_pv: one int32 partial context per chunk), and a row's own slots with
// the sum of its partials (k_shared_out). The scores are computed again in each:
// a slot's K row is 128 bytes for all queries, its scores 4 bytes for each.
// |partial context| <= 128 sum p <= 128 * 2^15 (a p rounds to at most twice its
// value), so int32 holds it.
//
// Query m of a kv head is head m % G of row m / G. Lane layout of the scores as
// in attn_prefill.h: S^T = K . Q^T, a lane holds one query (column qi = lane % 16)
// and 16 slots (16 g + 4 blk + r, g = lane / 16) of a 64-slot tile.
//
// 64 rows behind 8192 slots, 200 of their own, 16 / 8 heads: 50 us (maxima 11,
// sums 12, P.V of the prefix 16, the rest 12), 145 in the per-row form; the 46 MB
// take 10 us and the products 2. What is left is the launches' own chains (the
// first load, the parts' join and the block's end: 4 to 7 us each with one slot
// per row), so fewer and larger parts or another number of blocks change
// nothing: 256, 512 and 1024 blocks of maxima 11.0, 11.2, 11.3 us.
//
// Few rows or short prefixes do not pay for four launches and take
// attention.hip's kernels, the prefix's pages looked up in row 0.

#include "attn_plan.h"
#include "attn_prefill.h"
#include "attn_window.h"

namespace {

struct SharedArgs {
  const int8_t* q8;      // [B][n_q][128]
  const int64_t* tpos;   // [B][n_q]
  KVPages kv;
  const uint8_t* valid;  // [B][valid_stride]
  int64_t* out;          // [B][n_q * 128]
  int32_t* cmax;         // [n_kv][parts][M] maxima (INT32_MIN: no visible slot)
  i64* den;              // [n_kv][parts][M] sums of exponentials
  int32_t* ctx;          // [n_kv][parts2][M][128] partial contexts of the prefix
  const int64_t* s_dev;
  int32_t* err;
  i64 valid_stride;
  int B, S, P, n_q, n_kv;
  int gs, M;                       // G = 1 << gs
  int chunk, nchunks, qblocks;     // stat: slots per block (a multiple of 64)
  int pages2, nchunks2, qblocks2;  // pv: pages per block
  int parts, parts2;               // nchunks + 1 (the row's own slots), pv's

  __device__ __forceinline__ i64 query(int kvh, int m) const {
    return (i64)(m >> gs) * n_q + (kvh << gs) + (m & ((1 << gs) - 1));
  }
  __device__ __forceinline__ int scanned(bool report) const {
    if (!s_dev) return S;
    const i64 sd = *s_dev;
    if (report && sd > (i64)S && err) atomicOr(err, DI_ERR_SLOTS);
    return (int)imax(0, imin((i64)S, sd));
  }
};

// A lane's constants of the estimated DI-Exp and p: attn_prefill.h's PfFast
__device__ __forceinline__ PfFast shared_fast(i64 tpos, int mx, i64 den) {
  PfFast F;
  F.E = make_expest(tpos);
  F.kx = dexp_sp_const(F.E);
  F.cx = (int32_t)(F.E.t - (uint32_t)mx);
  F.D = make_divest(den, 16384.0);
  return F;
}

// The 16 flags of slots sl .. sl + 15 below S as loaded (flags16), and the bits
// of those that are set (flags16_bits): a group that would pass S is loaded to
// end there, and fewer than 16 slots in all come one by one.
__device__ __forceinline__ void flags16(const uint8_t* vrow, int sl, int S, uint32_t (&f)[4]) {
  if (S >= 16) {
    __builtin_memcpy(f, vrow + min(sl, S - 16), 16);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f[q] = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int s = sl + 4 * q + r;
        f[q] |= (s < S && vrow[max(min(s, S - 1), 0)] != 0 ? 1u : 0u) << (8 * r);
      }
    }
  }
}
__device__ __forceinline__ uint32_t flags16_bits(const uint32_t (&f)[4], int sl, int S) {
  const uint32_t m = flag_bits(f);
  const int past = S >= 16 ? max(sl + 16 - S, 0) : 0;
  return past < 16 ? m >> past : 0u;
}

// The maxima and (DEN) denominators of the block's queries m0 .. m0 + NQ - 1 (those
// below mend) over all parts, read by the 256 threads together, up to eight
// parts of a query in flight each: a lane on its own would wait for one part
// after the other. To mx / den (shared memory, NQ each), ready for the block.
template <int NQ, bool DEN>
__device__ __forceinline__ void shared_parts(const SharedArgs& a, int kvh, int m0, int mend,
                                             int32_t (&buf)[256], i64 (&dbuf)[DEN ? 256 : 1]) {
  constexpr int K = 256 / NQ, U = 8;
  const int q = threadIdx.x % NQ, k0 = threadIdx.x / NQ;
  const int m = min(m0 + q, mend - 1);
  const int32_t* cm = a.cmax + (i64)kvh * a.parts * a.M + m;
  const i64* dn = a.den + (i64)kvh * a.parts * a.M + m;
  int mx = INT32_MIN;
  i64 den = 0;
  for (int k = k0; k < a.parts; k += U * K) {
    int32_t x[U];
    i64 y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const i64 at = (i64)min(k + u * K, a.parts - 1) * a.M;
      x[u] = cm[at];
      if (DEN) y[u] = dn[at];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mx = max(mx, x[u]);  // (a part read twice changes no maximum)
      if (DEN) den = wadd(den, k + u * K < a.parts ? y[u] : 0);
    }
  }
  buf[threadIdx.x] = mx;
  if (DEN) dbuf[threadIdx.x] = den;
  __syncthreads();
  mx = INT32_MIN;
  den = 0;
#pragma unroll
  for (int w = 0; w < K; ++w) {
    mx = max(mx, buf[w * NQ + q]);
    if (DEN) den = wadd(den, dbuf[w * NQ + q]);
  }
  __syncthreads();
  if (k0 == 0) {
    buf[q] = mx == INT32_MIN ? 0 : mx;  // no visible slot: every p = 0
    if (DEN) dbuf[q] = imax(den, 1);
  }
  __syncthreads();
}

// Maxima or sums of exponentials of NG groups of 16 queries from m0 on, over the
// tiles [tile0, tend) (64 slots each) of row trow's pages, for part `part`. Each
// wave takes every fourth tile, a K row read once for its NG groups; the
// queries and their constants are read back from LDS, so that a wave needs about
// 100 registers and four blocks share a CU.
constexpr int STAT_QROW = 144;  // bytes between queries in LDS: 16 lanes on 64 banks
template <int NG>
struct StatLds {
  __attribute__((aligned(16))) int8_t q[16 * NG * STAT_QROW];
  double rt[16 * NG], kx[16 * NG];  // of the estimated DI-Exp
  uint32_t t[16 * NG];
  i64 tpos[16 * NG];
  i64 red[4 * 16 * NG];
  int32_t mx[256];
};
template <int NG, bool DEN>
__device__ __forceinline__ void shared_stat(const SharedArgs& a, int S, int kvh, int m0, int mend,
                                            int trow, int tile0, int tend, int part, char* lds) {
  StatLds<NG>& L = *(StatLds<NG>*)lds;
  const int tid = threadIdx.x, lane = tid & 63, qi = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int first = tile0 + wave;
  const int ntiles = first < tend ? (tend - first + 3) / 4 : 0;
  const int kr = 16 * (qi >> 2) + (qi & 3);
  int pgv = 0;  // pages of the wave's next 64 tiles, a lane each
  auto load_pages = [&](int i0) {
    const int t = first + (i0 + lane) * 4;
    pgv = a.kv.page(trow, (i64)(t < tend ? t : tile0) * 64);
  };
  if (ntiles > 0) load_pages(0);
  // the queries to LDS, 8 threads each
#pragma unroll
  for (int i = tid; i < 16 * NG * 8; i += 256) {
    const int m = min(m0 + (i >> 3), mend - 1);
    *(v4i*)(L.q + (i >> 3) * STAT_QROW + (i & 7) * 16) =
        *(const v4i*)(a.q8 + a.query(kvh, m) * 128 + (i & 7) * 16);
  }
  const uint8_t* vrow[NG];
#pragma unroll
  for (int n = 0; n < NG; ++n)
    vrow[n] = a.valid + (i64)(min(m0 + 16 * n + qi, mend - 1) >> a.gs) * a.valid_stride;
  v4i k[8];
  uint32_t f[NG][4];
  bool ok = false;  // the tile's page is mapped
  auto load = [&](int i) {
    const int s0 = (first + i * 4) * 64, pg = __builtin_amdgcn_readlane(pgv, i & 63);
    const int8_t* kb = a.kv.krow(pg < 0 ? 0 : pg, kvh, (s0 & (DI_PAGE - 1)) + kr) + g * 16;
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) {
      k[2 * blk] = *(const v4i*)(kb + blk * 512);
      k[2 * blk + 1] = *(const v4i*)(kb + blk * 512 + 64);
    }
#pragma unroll
    for (int n = 0; n < NG; ++n) flags16(vrow[n], s0 + 16 * g, S, f[n]);
    ok = pg >= 0;
  };
  if (ntiles > 0) load(0);
  bool fexp = true;  // block-uniform: every constant below 2^23
  if (DEN) {
    i64 none[1];
    i64 tp = 1;
    if (tid < 16 * NG) tp = a.tpos[a.query(kvh, min(m0 + tid, mend - 1))];
    shared_parts<16 * NG, false>(a, kvh, m0, mend, L.mx, none);
    if (tid < 16 * NG) {
      const ExpEst E = make_expest(tp);
      L.rt[tid] = E.rt;
      L.kx[tid] = dexp_sp_const(E);
      L.t[tid] = E.t;
      L.tpos[tid] = tp;
    }
    fexp = __syncthreads_and(tp < (i64)PF_SMALL_T) != 0;
  } else {
    __syncthreads();
  }
  int mx[NG];
  i64 den[NG];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    mx[n] = INT32_MIN;
    den[n] = 0;
  }
  for (int i = 0; i < ntiles; ++i) {
    const int sl = (first + i * 4) * 64 + 16 * g;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int q = 16 * n + qi;
      __builtin_amdgcn_sched_barrier(0);  // (else all groups' queries are read at once)
      const v4i qf0 = *(const v4i*)(L.q + q * STAT_QROW + g * 16);
      const v4i qf1 = *(const v4i*)(L.q + q * STAT_QROW + 64 + g * 16);
      // (where the estimate runs, scores arrive as st + t - mx)
      ExpEst E{0.0, 0};
      double kx = 0.0;
      int off = 0;
      if (DEN) {
        E.rt = L.rt[q];
        E.t = L.t[q];
        kx = L.kx[q];
        off = fexp ? (int)(E.t - (uint32_t)L.mx[q]) : 0;
      }
      const v4i z = v4i{off, off, off, off};
      v4i st[4];
#pragma unroll
      for (int blk = 0; blk < 4; ++blk) st[blk] = mfma16(k[2 * blk], qf0, z);
#pragma unroll
      for (int blk = 0; blk < 4; ++blk) st[blk] = mfma16(k[2 * blk + 1], qf1, st[blk]);
      const uint32_t bits = ok ? flags16_bits(f[n], sl, S) : 0u;
      if (!DEN) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          mx[n] = max(mx[n], (bits >> r) & 1u ? st[r >> 2][r & 3] : INT32_MIN);
      } else if (DI_LIKELY(fexp)) {
        uint32_t sum = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool vis = (bits >> r) & 1u;
          const uint32_t e = dexp_est_sp(vis ? st[r >> 2][r & 3] : (int32_t)E.t, E, kx);
          sum += vis ? e : 0u;
        }
        den[n] += sum;
      } else {
        const ExpR Et = make_exp(L.tpos[q]);
        const int m = L.mx[q];
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if ((bits >> r) & 1u)
            den[n] = wadd(den[n], di_exp_neg((u64)(uint32_t)(m - st[r >> 2][r & 3]), Et));
      }
    }
    if (i + 1 < ntiles) {
      if (((i + 1) & 63) == 0) load_pages(i + 1);
      load(i + 1);
    }
  }
  // over the lanes of a query, then over the waves
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    i64 v;
    if (DEN) {
      v = group4_sum(den[n]);
    } else {
      const int x = max(mx[n], __shfl_xor(mx[n], 16));
      v = max(x, __shfl_xor(x, 32));
    }
    if (g == 0) L.red[(wave * NG + n) * 16 + qi] = v;
  }
  __syncthreads();
  if (tid < 16 * NG && m0 + tid < mend) {
    i64 v = L.red[tid];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const i64 o = L.red[w * NG * 16 + tid];
      v = DEN ? wadd(v, o) : imax(v, o);
    }
    const i64 at = ((i64)kvh * a.parts + part) * a.M + m0 + tid;
    if (DEN) a.den[at] = v;
    else a.cmax[at] = (int32_t)v;
  }
}

// Blocks of the prefix (chunk, query block, kv head), then one per (row, kv
// head) for the row's own slots.
template <int NG, bool DEN>
__global__ __launch_bounds__(256, DEN ? 4 : 3) void k_shared_stat(SharedArgs a) {
  keep_hidden_args();
  __shared__ __attribute__((aligned(16))) char lds[sizeof(StatLds<NG>)];
  const int S = a.scanned(false);
  const int npre = a.nchunks * a.qblocks * a.n_kv;
  const int bid = blockIdx.x;
  if (bid < npre) {
    const int c = bid / (a.qblocks * a.n_kv), r = bid % (a.qblocks * a.n_kv);
    const int end = min(min((c + 1) * a.chunk, a.P), S);
    shared_stat<NG, DEN>(a, S, r % a.n_kv, r / a.n_kv * 16 * NG, a.M, 0, c * (a.chunk / 64),
                         (end + 63) / 64, c, lds);
  } else {
    const int r = bid - npre, b = r / a.n_kv;
    shared_stat<1, DEN>(a, S, r % a.n_kv, b << a.gs, (b + 1) << a.gs, b, a.P / 64, (S + 63) / 64,
                        a.nchunks, lds);
  }
}

// What a lane needs to make p of its query
struct SharedRow {
  i64 tpos, den;
  int mx;
  int32_t off;  // scores arrive as st + off
  bool fdiv;    // wave-uniform: the estimates hold
  PfFast F;
};
__device__ __forceinline__ SharedRow shared_row(i64 tpos, int mx, i64 den) {
  SharedRow R;
  R.tpos = tpos;
  R.mx = mx;
  R.den = den;
  R.fdiv = __ballot(R.tpos >= (i64)PF_SMALL_T || R.den >= PF_SMALL_DEN) == 0;
  R.F = shared_fast(R.tpos, R.mx, R.den);
  R.off = R.fdiv ? R.F.cx : 0;
  return R;
}

// p of a lane's 16 slots as the two operands of P.V
__device__ __forceinline__ void shared_p(const SharedRow& R, const v4i (&st)[4], uint32_t bits,
                                         v4i& phi, v4i& plo) {
  auto put = [&](int blk, const uint32_t (&p)[4]) {
    int whi, wlo;
    pf_pack(p, whi, wlo);
    phi[blk] = whi;
    plo[blk] = wlo;
  };
  if (DI_LIKELY(R.fdiv)) {
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) {
      uint32_t p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool vis = (bits >> (4 * blk + r)) & 1u;
        const uint32_t e = dexp_est_sp(vis ? st[blk][r] : (int32_t)R.F.E.t, R.F.E, R.F.kx);
        p[r] = rhad_est((double)(vis ? e : 0u), R.F.D);
      }
      put(blk, p);
    }
  } else {
    const ExpR Et = make_exp(R.tpos);
    const Recip Rd = make_recip(R.den);
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) {
      uint32_t p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = 0;
        if ((bits >> (4 * blk + r)) & 1u) {
          const i64 e = di_exp_neg((u64)(uint32_t)(R.mx - st[blk][r]), Et);
          p[r] = (uint32_t)to_i32(rhad_r(shl(e, 14), Rd));
        }
      }
      put(blk, p);
    }
  }
}

// P.V of the prefix. Block: one kv head, pages2 pages, QW groups of 16 queries;
// its 4 waves are the QW groups times SW = 4 / QW shares of the 64-slot tiles.
// K and V pages go through LDS as in attn_prefill.h, two pages deep; the
// validity bits of the block's rows and pages are made first.
constexpr int SH_MAXP = 8;  // pages per block at most (the bits' LDS), so the partial
                            // contexts grow with rows x prefix: 268 MB of scratch for
                            // 64 rows of 64 / 8 heads behind 130944 slots
template <int QW>
__global__ __launch_bounds__(256, 2) void k_shared_pv(SharedArgs a) {
  keep_hidden_args();
  constexpr int SW = 4 / QW, NC = 8 / QW, STAGE = PF_KBYTES + PF_VBYTES;
  __shared__ __attribute__((aligned(1024))) int8_t ring[2 * STAGE];
  __shared__ uint16_t bits16[16 * QW][SH_MAXP * 8];
  __shared__ int32_t csum[SW][128], buf[256];
  __shared__ i64 dbuf[256];
  const int tid = threadIdx.x, lane = tid & 63, qi = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave % QW, sub = wave / QW;
  const int c = blockIdx.x / (a.qblocks2 * a.n_kv), rr = blockIdx.x % (a.qblocks2 * a.n_kv);
  const int kvh = rr % a.n_kv, mb = rr / a.n_kv * 16 * QW;
  const int S = a.scanned(false);
  const int p0 = c * a.pages2, np = min(a.pages2, a.P / DI_PAGE - p0);
  const int pgv = lane < np ? a.kv.page(0, (i64)(p0 + lane) * DI_PAGE) : -1;
  int koff[4], voff4[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = (wave * 4 + j) * 8 + (lane >> 3);
    koff[j] = row * 128 + ((lane & 7) ^ pf_kswz(row)) * 16;
    voff4[j] = row * DI_PAGE + ((lane & 7) ^ pf_vswz(row)) * 16;
  }
  auto issue = [&](int i) {
    const int pg = __builtin_amdgcn_readlane(pgv, i);
    int8_t* st = ring + (i & 1) * STAGE;
    const int nrec = pg < 0 ? 0 : DI_PAGE * 128;  // (a page that is not mapped reads 0)
    const __amdgpu_buffer_rsrc_t krs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)a.kv.krow(pg < 0 ? 0 : pg, kvh, 0), (short)0, nrec, 0x00020000);
    const __amdgpu_buffer_rsrc_t vrs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)a.kv.vchan(pg < 0 ? 0 : pg, kvh, 0), (short)0, nrec, 0x00020000);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(krs, (lds_ptr_t)(st + (wave * 4 + j) * 1024), 16,
                                               koff[j], 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          vrs, (lds_ptr_t)(st + PF_KBYTES + (wave * 4 + j) * 1024), 16, voff4[j], 0, 0, 0);
  };
  issue(0);
  // validity bits: row r of the block's (its first is mb / G), 16 slots each
  {
    const int r0 = mb >> a.gs, nrows = min(((16 * QW - 1) >> a.gs) + 1, a.B - r0), ng = np * 8;
    for (int i = tid; i < nrows * ng; i += 256) {
      const int r = i / ng, q = i % ng;
      uint32_t f[4];
      const int sl = p0 * DI_PAGE + 16 * q;
      flags16(a.valid + (i64)(r0 + r) * a.valid_stride, sl, S, f);
      bits16[r][q] = (uint16_t)flags16_bits(f, sl, S);
    }
  }
  const int m = mb + grp * 16 + qi;
  const bool tok = m < a.M;
  const i64 gq = a.query(kvh, tok ? m : mb);
  const v4i qf0 = *(const v4i*)(a.q8 + gq * 128 + g * 16);
  const v4i qf1 = *(const v4i*)(a.q8 + gq * 128 + 64 + g * 16);
  const i64 tpos = a.tpos[gq];
  shared_parts<16 * QW, true>(a, kvh, mb, a.M, buf, dbuf);  // (its barriers publish the bits)
  const SharedRow R = shared_row(tpos, buf[grp * 16 + qi], dbuf[grp * 16 + qi]);
  const v4i z = v4i{R.off, R.off, R.off, R.off};
  const int brow = tok ? (m >> a.gs) - (mb >> a.gs) : 0;
  const int kr = 16 * (qi >> 2) + (qi & 3);
  const int koff0 = kr * 128 + ((g ^ pf_kswz(kr)) << 4);
  const int koff1 = kr * 128 + (((g + 4) ^ pf_kswz(kr)) << 4);
  v4i ohi[8], olo[8], ocs[NC];
#pragma unroll
  for (int j = 0; j < 8; ++j) ohi[j] = olo[j] = v4i{0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < NC; ++j) ocs[j] = v4i{0, 0, 0, 0};
  const v4i ones = v4i{0x01010101, 0x01010101, 0x01010101, 0x01010101};
  for (int i = 0; i < np; ++i) {
    const bool mapped = __builtin_amdgcn_readlane(pgv, i) >= 0;
    // this wave's loads of the page are done and its LDS reads of the last one;
    // after the barrier every wave's are, and the other stage is free
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_s_barrier();
    if (i + 1 < np) issue(i + 1);
    const int8_t* stg = ring + (i & 1) * STAGE;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      if (SW == 2 && sub != hf) continue;
      if (SW == 4 && ((2 * i + hf) & 3) != sub) continue;
      v4i st[4], k[8], vf[8];
#pragma unroll
      for (int blk = 0; blk < 4; ++blk) {
        k[2 * blk] = *(const v4i*)(stg + hf * 64 * 128 + koff0 + blk * 512);
        k[2 * blk + 1] = *(const v4i*)(stg + hf * 64 * 128 + koff1 + blk * 512);
      }
#pragma unroll
      for (int blk = 0; blk < 4; ++blk) st[blk] = mfma16(k[2 * blk], qf0, z);
#pragma unroll
      for (int blk = 0; blk < 4; ++blk) st[blk] = mfma16(k[2 * blk + 1], qf1, st[blk]);
      const uint32_t bits = mapped && tok ? bits16[brow][i * 8 + hf * 4 + g] : 0u;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        vf[j] = *(const v4i*)(stg + PF_KBYTES + (16 * j + qi) * 128 +
                              (((4 * hf + g) ^ pf_vswz(qi)) << 4));
      v4i phi, plo;
      shared_p(R, st, bits, phi, plo);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ohi[j] = mfma16(phi, vf[j], ohi[j]);
        olo[j] = mfma16(plo, vf[j], olo[j]);
      }
      // the waves that share the tile make the column sums of V in parts
#pragma unroll
      for (int w = 0; w < QW; ++w)
        if (grp == w) {  // wave-uniform
#pragma unroll
          for (int j = 0; j < NC; ++j) ocs[j] = mfma16(ones, vf[w * NC + j], ocs[j]);
        }
    }
  }
  if (g == 0) {
#pragma unroll
    for (int j = 0; j < NC; ++j) csum[sub][(grp * NC + j) * 16 + qi] = ocs[j][0];
  }
  __syncthreads();
  // lane holds O[query 4 g + r][channel 16 j + qi]
  int32_t* o = a.ctx + (((i64)kvh * a.parts2 + c * SW + sub) * a.M + mb + grp * 16 + 4 * g) * 128 + qi;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int32_t cs = csum[sub][16 * j + qi];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (mb + grp * 16 + 4 * g + r < a.M)
        o[r * 128 + 16 * j] = (ohi[j][r] + 64 * cs) * 128 + olo[j][r];  // (modulo 2^32)
  }
}

// The row's own slots (4 waves, every fourth tile each), and the prefix's
// partial contexts added. Block per (kv head, row).
__global__ __launch_bounds__(256, 2) void k_shared_out(SharedArgs a) {
  keep_hidden_args();
  __shared__ int32_t sums[4][8 * 128], buf[256];
  __shared__ i64 dbuf[256];
  const int tid = threadIdx.x, lane = tid & 63, qi = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % a.n_kv, b = blockIdx.x / a.n_kv, G = 1 << a.gs, m0 = b << a.gs;
  const int S = a.scanned(blockIdx.x == 0 && tid == 0);
  const int first = a.P / 64 + wave, tend = (S + 63) / 64;
  const int ntiles = first < tend ? (tend - first + 3) / 4 : 0;
  const int kr = 16 * (qi >> 2) + (qi & 3);
  const bool tok = qi < G;
  const i64 gq = a.query(kvh, m0 + (tok ? qi : 0));
  const uint8_t* vrow = a.valid + (i64)b * a.valid_stride;
  int pgv = 0;
  auto load_pages = [&](int i0) {
    const int t = first + (i0 + lane) * 4;
    pgv = a.kv.page(b, (i64)(t < tend ? t : first) * 64);
  };
  v4i k[8], vf[8];
  uint32_t f[4];
  int pg = 0;
  auto load_k = [&](int i) {
    pg = __builtin_amdgcn_readlane(pgv, i & 63);
    const int s0 = (first + i * 4) * 64;
    const int8_t* kb = a.kv.krow(pg < 0 ? 0 : pg, kvh, (s0 & (DI_PAGE - 1)) + kr) + g * 16;
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) {
      k[2 * blk] = *(const v4i*)(kb + blk * 512);
      k[2 * blk + 1] = *(const v4i*)(kb + blk * 512 + 64);
    }
    flags16(vrow, s0 + 16 * g, S, f);
  };
  auto load_v = [&](int i) {
    const int s0 = (first + i * 4) * 64;
    const int8_t* vb = a.kv.vchan(pg < 0 ? 0 : pg, kvh, qi) + (s0 & (DI_PAGE - 1)) + 16 * g;
#pragma unroll
    for (int j = 0; j < 8; ++j) vf[j] = *(const v4i*)(vb + j * 16 * DI_PAGE);
  };
  if (ntiles > 0) {
    load_pages(0);
    load_k(0);
    load_v(0);
  }
  const v4i qf0 = *(const v4i*)(a.q8 + gq * 128 + g * 16);
  const v4i qf1 = *(const v4i*)(a.q8 + gq * 128 + 64 + g * 16);
  const i64 tpos = a.tpos[gq];
  // this thread's outputs of the prefix: element tid + 256 e of [G][128]
  int32_t pre[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (256 * e < G * 128) {
      const int32_t* cx =
          a.ctx + ((i64)kvh * a.parts2 * a.M + m0) * 128 + min(tid + 256 * e, G * 128 - 1);
      for (int p = 0; p < a.parts2; p += 8) {
        int32_t x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = cx[(i64)min(p + u, a.parts2 - 1) * a.M * 128];
#pragma unroll
        for (int u = 0; u < 8; ++u) pre[e] += p + u < a.parts2 ? x[u] : 0;
      }
    }
  shared_parts<16, true>(a, kvh, m0, m0 + G, buf, dbuf);
  const SharedRow R = shared_row(tpos, buf[qi], dbuf[qi]);
  const v4i z = v4i{R.off, R.off, R.off, R.off};
  v4i ohi[8], olo[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) ohi[j] = olo[j] = v4i{0, 0, 0, 0};
  const v4i ones = v4i{0x01010101, 0x01010101, 0x01010101, 0x01010101};
  for (int i = 0; i < ntiles; ++i) {
    v4i st[4];
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) st[blk] = mfma16(k[2 * blk], qf0, z);
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) st[blk] = mfma16(k[2 * blk + 1], qf1, st[blk]);
    const int sl = (first + i * 4) * 64 + 16 * g;
    const uint32_t bits = pg >= 0 && tok ? flags16_bits(f, sl, S) : 0u;
    v4i phi, plo;
    shared_p(R, st, bits, phi, plo);
    if (qi == 15) phi = ones;  // no query: the row makes V's column sums
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ohi[j] = mfma16(phi, vf[j], ohi[j]);
      olo[j] = mfma16(plo, vf[j], olo[j]);
    }
    if (i + 1 < ntiles) {
      if (((i + 1) & 63) == 0) load_pages(i + 1);
      load_k(i + 1);
      load_v(i + 1);
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int32_t cs = __shfl(ohi[j][3], 48 + qi);  // row 15
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (4 * g + r < G)
        sums[wave][(4 * g + r) * 128 + 16 * j + qi] = (ohi[j][r] + 64 * cs) * 128 + olo[j][r];
  }
  __syncthreads();
  int64_t* o = a.out + ((i64)b * a.n_q + (kvh << a.gs)) * 128;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int i = tid + 256 * e;
    if (i < G * 128) o[i] = pre[e] + sums[0][i] + sums[1][i] + sums[2][i] + sums[3][i];
  }
}

// ---- the per-row form: attention.hip's kernels, the first P slots' pages row 0's
struct SharedView {
  static constexpr bool kWhole = true;
  int P;
  __device__ __forceinline__ int slot(int s) const { return s; }
  __device__ __forceinline__ int page(const KVPages& kv, int b, int s) const {
    return kv.page(s < P ? 0 : b, s);
  }
  __device__ __forceinline__ bool sees(int) const { return true; }
};
template <int G>
__global__ __launch_bounds__(512) void k_shared_one(DecodeArgs a, int P) {
  keep_hidden_args();
  extern __shared__ __attribute__((aligned(16))) int32_t sh_scores[];
  __shared__ int32_t pg_lds[DEC_MAX_PAGES];
  const int kvh = blockIdx.x, b = blockIdx.y;
  const i64 q0 = (i64)b * a.n_q + kvh * G;
  const SharedView v{P};
  bool over;
  const int S = scanned_slots(a, a.tpos, &over);
  const int npages = (a.S + DI_PAGE - 1) / DI_PAGE;
  for (int i = threadIdx.x; i < npages; i += 512) pg_lds[i] = v.page(a.kv, b, i * DI_PAGE);
  if (npages == 0 && threadIdx.x == 0) pg_lds[0] = -1;  // S = 0: loads read page 0
  __syncthreads();
  decode_body<G, VPRE, false, false, 8>(a, S, kvh, b, a.q8 + q0 * 128, a.tpos + q0, sh_scores, pg_lds);
  report_slots(a, over, kvh == 0);
}
template <int G>
__global__ __launch_bounds__(256) void k_shared_scores(SplitArgs sa, int P) {
  keep_hidden_args();
  split_scores_chunk<G, SharedView>(sa, blockIdx.x, blockIdx.y, blockIdx.z, SharedView{P});
}
template <int G>
__global__ __launch_bounds__(256) void k_shared_split_pv(SplitArgs sa, int P) {
  keep_hidden_args();
  split_pv_chunk<G, SharedView>(sa, blockIdx.x, blockIdx.y, blockIdx.z, SharedView{P});
}

// Whether the four launches pay: they cost 19 us with few rows and 25 with 17
// and more (the queries then fill blocks of four groups), whatever the prefix, and
// a row's own slots cost more there than in the per-row form. The rule bounds
// these by the prefix and grows no stricter with fewer of them. us per call, per
// row / joint, 40 slots behind the prefix:
//   16 / 8 heads: 4 rows 8192 slots 26.7 / 27.3, 8 rows 4096 23.8 / 24.4, 8192 34.6 /
//     28.3, 16 rows 2048 23.0 / 21.5, 4096 32.0 / 25.1; 17 rows 2048 22.9 / 25.0, 2560
//     27.3 / 25.6, 4096 40.0 / 27.8, 8192 56.7 / 31.6; 32 rows 2048 24.0 / 26.7, 2560
//     28.4 / 27.5, 4096 40.5 / 28.7; 33 rows 2048 36.4 / 27.9; 64 rows 1024 23.4 / 28.1,
//     1280 27.9 / 28.5, 1536 30.9 / 28.9, 2048 37.8 / 29.8, 8192 144 / 44; 100 rows 1024
//     41.7 / 34.6
//   17 rows 2048, 2560 and 4096: 8 / 8 heads 21.6 / 21.7, 25.8 / 22.5, 38.2 / 25.2; 32 / 8
//     26.2 / 26.3, 30.8 / 29.0, 48.3 / 30.1; 8 / 1 35.6 / 28.7, 37.7 / 30.9, 48.6 / 33.1; 4 /
//     2 16.4 / 25.5, 16.6 / 25.9, 22.1 / 26.6 (so few heads: by the slots saved alone)
//   more slots behind the prefix, 16 / 8 heads: 17 rows 1000 behind 4096 48.4 / 42.1,
//     2000 56.8 / 61.9; 16 rows 1000 behind 1024 22.8 / 34.9, 64 rows 38.0 / 62.7
bool shared_joint(int B, int S, int P, int n_q) {
  const i64 saved = (i64)(B - 1) * P;
  if (B <= 16) return saved >= 24576 && S - P <= imin(P / 16, 512);
  const bool pays = saved >= 81920 || (n_q >= 8 && (P >= 2560 || (P >= 1536 && saved >= 65536)));
  return pays && S - P <= P / 4;
}

struct SharedPlan {
  bool joint;                                          // the prefix read once for the batch
  int ng, qblocks, chunk, nchunks;                     // stat
  int qw, qblocks2, pages2, nchunks2, parts, parts2;   // pv
  int split;                                           // per row: decode_chunk
  i64 bytes;
};
SharedPlan shared_plan(int B, int S, int P, int n_q, int n_kv) {
  SharedPlan p{};
  const int G = n_q / n_kv;
  const i64 M = (i64)B * G;
  p.joint = shared_joint(B, S, P, n_q);
  if (!p.joint) {
    i64 at;
    p.split = B > 0 && S > 0 ? decode_chunk(B, S, n_q, n_kv) : 0;
    p.bytes = p.split ? split_bytes(B, S, n_q, p.split, &at) : 0;
    return p;
  }
  p.ng = p.qw = M <= 16 ? 1 : M <= 32 ? 2 : 4;
  p.qblocks = p.qblocks2 = (int)((M + 16 * p.ng - 1) / (16 * p.ng));
  const i64 per = (i64)p.qblocks * n_kv;  // blocks of one chunk
  // stat: about two blocks per CU, a tile or more for each wave
  i64 want = imax(512 / per, 1);
  i64 tiles = (P / 64 + want - 1) / want;
  p.chunk = (int)((tiles + 3) / 4 * 4 * 64);
  p.nchunks = (P + p.chunk - 1) / p.chunk;
  p.parts = p.nchunks + 1;
  // pv: about one block per CU
  want = imax(256 / per, 1);
  p.pages2 = (int)imin(imax((P / DI_PAGE + want - 1) / want, 1), SH_MAXP);
  p.nchunks2 = (P / DI_PAGE + p.pages2 - 1) / p.pages2;
  p.parts2 = p.nchunks2 * (4 / p.qw);
  p.bytes = n_kv * M * ((i64)p.parts * 12 + (i64)p.parts2 * 512) + 64;
  return p;
}
int shared_args_ok(int B, int S, int n_q, int n_kv, int shared) {
  if (B < 0 || S < 0 || shared < 0 || shared > S || shared % DI_PAGE) return DI_EINVAL;
  if (const int rc = heads_ok(n_q, n_kv)) return rc;
  if (S > DEC_MAX_S) return DI_ERANGE;  // int32 MFMA accumulators of P.V
  return DI_OK;
}

}  // namespace

extern "C" {

int detllm_attn_decode_shared_work(int B, int S, int n_q, int n_kv, int shared, int64_t* bytes,
                                   int* joint) {
  if (!bytes) return DI_EINVAL;
  if (const int rc = shared_args_ok(B, S, n_q, n_kv, shared)) return rc;
  const SharedPlan p = shared_plan(B, S, shared, n_q, n_kv);
  *bytes = p.bytes;
  if (joint) *joint = p.joint;
  return DI_OK;
}

int detllm_attn_decode_shared(const int8_t* q8, const int64_t* tpos, const int8_t* kpool,
                              const int8_t* vpool, const int32_t* table, int width,
                              const uint8_t* valid, int64_t valid_stride, int B, int S, int n_q,
                              int n_kv, const int64_t* s_dev, int shared, void* work,
                              int64_t work_bytes, int64_t* out, int32_t* err, hipStream_t s) {
  if (const int rc = shared_args_ok(B < 0 ? 0 : B, S, n_q, n_kv, shared)) return rc;
  if (B <= 0) return DI_OK;
  if (!kv_ok(kpool, vpool, table, width) || S > (i64)width * DI_PAGE || valid_stride < S || !q8 ||
      !tpos || !valid || !out)
    return DI_EINVAL;
  const SharedPlan p = shared_plan(B, S, shared, n_q, n_kv);
  if (p.bytes > 0 && (!work || work_bytes < p.bytes)) return DI_ERANGE;
  const int G = n_q / n_kv;
  const KVPages kv{(int8_t*)kpool, (int8_t*)vpool, table, width, n_kv};
  if (!p.joint) {
    const DecodeArgs d{q8, tpos, kv, valid, out, nullptr, s_dev, S, n_q, n_kv, valid_stride, err};
    if (p.split) {
      const SplitArgs sa = split_args(d, B, p.split, work);
      const dim3 grid(n_kv, B, sa.ns);
      const size_t dyn = (size_t)G * p.split * 4;
      switch (G) {
#define DI_SHARED_SPLIT(G_)                                                        \
  case G_:                                                                         \
    hipLaunchKernelGGL(k_shared_scores<G_>, grid, dim3(256), 0, s, sa, shared);    \
    hipLaunchKernelGGL(k_shared_split_pv<G_>, grid, dim3(256), dyn, s, sa, shared); \
    break
        DI_SHARED_SPLIT(1);
        DI_SHARED_SPLIT(2);
        DI_SHARED_SPLIT(4);
        DI_SHARED_SPLIT(8);
#undef DI_SHARED_SPLIT
      }
    } else {
      const dim3 grid(n_kv, B);
      const size_t dyn = (size_t)G * (((i64)S + 15) / 16 * 16) * 4;
      switch (G) {
        case 1: hipLaunchKernelGGL(k_shared_one<1>, grid, dim3(512), dyn, s, d, shared); break;
        case 2: hipLaunchKernelGGL(k_shared_one<2>, grid, dim3(512), dyn, s, d, shared); break;
        case 4: hipLaunchKernelGGL(k_shared_one<4>, grid, dim3(512), dyn, s, d, shared); break;
        case 8: hipLaunchKernelGGL(k_shared_one<8>, grid, dim3(512), dyn, s, d, shared); break;
      }
    }
    DI_LAUNCH_CHECK();
    return DI_OK;
  }
  SharedArgs a{};
  a.q8 = q8; a.tpos = tpos; a.kv = kv;
  a.valid = valid; a.valid_stride = valid_stride; a.out = out; a.s_dev = s_dev; a.err = err;
  a.B = B; a.S = S; a.P = shared; a.n_q = n_q; a.n_kv = n_kv;
  a.gs = G == 8 ? 3 : G == 4 ? 2 : G == 2 ? 1 : 0;
  a.M = B * G;
  a.chunk = p.chunk; a.nchunks = p.nchunks; a.qblocks = p.qblocks; a.parts = p.parts;
  a.pages2 = p.pages2; a.nchunks2 = p.nchunks2; a.qblocks2 = p.qblocks2; a.parts2 = p.parts2;
  const i64 rows = (i64)n_kv * a.M;
  a.den = (i64*)work;
  a.cmax = (int32_t*)((char*)work + rows * p.parts * 8);
  a.ctx = (int32_t*)((char*)work + (rows * p.parts * 12 + 63) / 64 * 64);
  const i64 stat = (i64)p.nchunks * p.qblocks * n_kv + (i64)B * n_kv;
  const i64 pv = (i64)p.nchunks2 * p.qblocks2 * n_kv;
  if (stat > 0x7fffffff || pv > 0x7fffffff) return DI_ERANGE;
#define DI_SHARED(N)                                                                           \
  hipLaunchKernelGGL((k_shared_stat<N, false>), dim3((unsigned)stat), dim3(256), 0, s, a);     \
  hipLaunchKernelGGL((k_shared_stat<N, true>), dim3((unsigned)stat), dim3(256), 0, s, a);      \
  hipLaunchKernelGGL(k_shared_pv<N>, dim3((unsigned)pv), dim3(256), 0, s, a)
  if (p.ng == 1) { DI_SHARED(1); }
  else if (p.ng == 2) { DI_SHARED(2); }
  else { DI_SHARED(4); }
#undef DI_SHARED
  hipLaunchKernelGGL(k_shared_out, dim3((unsigned)(B * n_kv)), dim3(256), 0, s, a);
  DI_LAUNCH_CHECK();
  return DI_OK;
}

}  // extern "C"
