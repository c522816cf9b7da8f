// Decode attention of a batch whose rows share their first pages (gfx950). No
// counterpart in the reference; every row's integers are those of
// detllm_attn_decode over its own page table.
//
// Attention of one row reads K and V once for the G query heads of a kv head;
// rows behind one prefix read the same bytes B times. Here the prefix is read
// once for all B * G queries of a kv head, which also fill the 16 columns of
// the MFMA tiles that one row leaves mostly empty.
//
// DI-Exp is not multiplicative, so partial softmaxes cannot be rescaled and
// joined: a row's true maximum comes first, then its denominator, then p. Three
// launches, each over the same tiles: the maxima (PASS 0) and the exponentials'
// sums (PASS 1) of each part of a row, then p and P.V (PASS 2), whose partial
// contexts are added to the output in 64-bit integers. The scores are computed
// again in each launch: a slot's K row is 128 bytes for all queries, its scores
// 4 bytes for each of them.
//
// A prefix block takes one kv head, one chunk of the prefix and QW groups of 16
// queries; its 4 waves are QW groups times 4 / QW interleaved shares of the
// chunk's 64-slot tiles. A suffix block takes one (row, kv head), its G queries
// in one group, and 4 shares of the row's own slots. Lane layout as in
// attn_prefill.h: S^T = K . Q^T, a lane holds one query and 16 slots of a tile.

#include "attn_prefill.h"

namespace {

struct SharedArgs {
  const int8_t* q8;      // [B][n_q][128]
  const int64_t* tpos;   // [B][n_q]
  KVPages kv;
  const uint8_t* valid;  // [B][valid_stride]
  int64_t* out;          // [B][n_q * 128]
  int32_t* cmax;         // [B * n_q][parts] maxima (INT32_MIN: no visible slot)
  i64* den;              // [B * n_q][parts] sums of exponentials
  const int64_t* s_dev;
  int32_t* err;
  i64 valid_stride;
  int B, S, P, n_q, n_kv, G;
  int chunk, nchunks;    // slots per prefix block (a multiple of 64)
  int qblocks;           // prefix blocks along the queries
  int parts;             // nchunks * (4 / QW) + 4
};

template <int QW, int PASS>
__global__ __launch_bounds__(256, 2) void k_shared(SharedArgs a) {
  keep_hidden_args();
  constexpr int SW = 4 / QW;
  const int tid = threadIdx.x, lane = tid & 63, qi = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int npre = a.nchunks * a.qblocks * a.n_kv;
  const bool prefix = (int)blockIdx.x < npre;
  int S = a.S;
  if (a.s_dev) {
    const i64 sd = *a.s_dev;
    S = (int)imax(0, imin((i64)a.S, sd));
    if (PASS == 2 && sd > (i64)a.S && a.err && blockIdx.x == 0 && tid == 0)
      atomicOr(a.err, DI_ERR_SLOTS);
  }
  // the wave's queries m (row m / G, head m % G of the kv head) and tiles
  int kvh, m, mend, trow, tile, step, tend, part;
  if (prefix) {
    const int c = blockIdx.x / (a.qblocks * a.n_kv), r = blockIdx.x % (a.qblocks * a.n_kv);
    kvh = r % a.n_kv;
    m = (r / a.n_kv * QW + wave % QW) * 16 + qi;
    mend = a.B * a.G;
    trow = 0;
    tile = c * (a.chunk / 64) + wave / QW;
    step = SW;
    tend = min((c + 1) * a.chunk, min(a.P, (S + 63) & ~63)) / 64;
    part = c * SW + wave / QW;
  } else {
    const int r = blockIdx.x - npre;
    kvh = r % a.n_kv;
    trow = r / a.n_kv;
    m = trow * a.G + qi;
    mend = (trow + 1) * a.G;
    tile = a.P / 64 + wave;
    step = 4;
    tend = (S + 63) / 64;
    part = a.nchunks * SW + wave;
    if (PASS == 0)
      for (int i = tid; i < a.G * 128; i += 256)
        a.out[((i64)trow * a.n_q + kvh * a.G) * 128 + i] = 0;
  }
  const bool tok = m < mend;
  const int mb = tok ? m / a.G : trow;
  const i64 gq = (i64)mb * a.n_q + kvh * a.G + (tok ? m % a.G : 0);
  const uint8_t* vrow = a.valid + (i64)mb * a.valid_stride;
  v4i qf0 = v4i{0, 0, 0, 0}, qf1 = v4i{0, 0, 0, 0};
  if (tok) {
    qf0 = *(const v4i*)(a.q8 + gq * 128 + g * 16);
    qf1 = *(const v4i*)(a.q8 + gq * 128 + 64 + g * 16);
  }
  const i64 tpos = tok ? a.tpos[gq] : 1;

  // the row's maximum over all parts
  int mx = INT32_MIN;
  if (PASS > 0) {
    for (int k = g; k < a.parts; k += 4) mx = max(mx, a.cmax[gq * a.parts + k]);
    mx = max(mx, __shfl_xor(mx, 16));
    mx = max(mx, __shfl_xor(mx, 32));
    if (mx == INT32_MIN) mx = 0;  // no visible slot: every p = 0
  }
  // the estimated DI-Exp when every query of the wave has tpos < 2^23
  const bool fexp = __ballot(tpos >= (i64)PF_SMALL_T) == 0;
  PfFast F;
  F.E = make_expest(tpos);
  F.kx = dexp_sp_const(F.E);
  F.cx = (int32_t)(F.E.t - (uint32_t)mx);
  const int32_t soff = fexp && PASS > 0 ? F.cx : 0;
  const ExpR Et = make_exp(tpos);
  // exponential of a visible score as the MFMA leaves it (st + soff)
  auto ex = [&](int st) -> i64 {
    return fexp ? (i64)dexp_est_sp(st, F.E, F.kx) : di_exp_neg((u64)(uint32_t)(mx - (st - soff)), Et);
  };
  i64 den = 0;
  if (PASS == 2) {
    for (int k = g; k < a.parts; k += 4) den = wadd(den, a.den[gq * a.parts + k]);
    den = imax(group4_sum(den), 1);
  }
  const bool fdiv = fexp && __ballot(den >= PF_SMALL_DEN) == 0;
  F.D = make_divest(den, 16384.0);
  const Recip Rd = make_recip(imax(den, 1));

  v4i ohi[8], olo[8], ocs[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) ohi[j] = olo[j] = ocs[j] = v4i{0, 0, 0, 0};
  const v4i ones = v4i{0x01010101, 0x01010101, 0x01010101, 0x01010101};
  const v4i z = v4i{soff, soff, soff, soff};
  const int kr = 16 * (qi >> 2) + (qi & 3);
  for (; tile < tend; tile += step) {
    const int s0 = tile * 64;
    const int pg = a.kv.page(trow, s0), pgc = pg < 0 ? 0 : pg;
    const int8_t* kb = a.kv.krow(pgc, kvh, (s0 & (DI_PAGE - 1)) + kr) + g * 16;
    v4i st[4];
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) {
      const v4i k0 = *(const v4i*)(kb + blk * 512), k1 = *(const v4i*)(kb + blk * 512 + 64);
      st[blk] = mfma16(k0, qf0, z);
      st[blk] = mfma16(k1, qf1, st[blk]);
    }
    const uint32_t bits = pg >= 0 && tok ? valid16(vrow, s0 + 16 * g, S) : 0u;
    if (PASS == 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if ((bits >> i) & 1u) mx = max(mx, st[i >> 2][i & 3]);
    } else if (PASS == 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool vis = (bits >> i) & 1u;
        const i64 e = ex(vis ? st[i >> 2][i & 3] : (int32_t)(fexp ? F.E.t : (uint32_t)mx));
        den = wadd(den, vis ? e : 0);
      }
    } else {
      v4i phi, plo;
#pragma unroll
      for (int blk = 0; blk < 4; ++blk) {
        uint32_t p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool vis = (bits >> (4 * blk + r)) & 1u;
          const i64 e = ex(vis ? st[blk][r] : (int32_t)(fexp ? F.E.t : (uint32_t)mx));
          const uint32_t q = fdiv ? rhad_est((double)(uint32_t)e, F.D)
                                  : (uint32_t)to_i32(rhad_r(shl(e, 14), Rd));
          p[r] = vis ? q : 0u;
        }
        int whi, wlo;
        pf_pack(p, whi, wlo);
        phi[blk] = whi;
        plo[blk] = wlo;
      }
      const int8_t* vb = a.kv.vchan(pgc, kvh, qi) + (s0 & (DI_PAGE - 1)) + 16 * g;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const v4i vf = *(const v4i*)(vb + j * 16 * DI_PAGE);
        ohi[j] = mfma16(phi, vf, ohi[j]);
        olo[j] = mfma16(plo, vf, olo[j]);
        ocs[j] = mfma16(ones, vf, ocs[j]);
      }
    }
  }
  if (PASS == 0) {
    mx = max(mx, __shfl_xor(mx, 16));
    mx = max(mx, __shfl_xor(mx, 32));
    if (tok && g == 0) a.cmax[gq * a.parts + part] = mx;
  } else if (PASS == 1) {
    den = group4_sum(den);
    if (tok && g == 0) a.den[gq * a.parts + part] = den;
  } else {
    // lane holds O[query 4 g + r][channel 16 j + qi]
    const int m0 = m - qi + 4 * g;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int mq = m0 + r;
      if (mq < mend) {
        int64_t* o = a.out + ((i64)(mq / a.G) * a.n_q + kvh * a.G + mq % a.G) * 128 + qi;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const i64 v = (i64)ohi[j][r] * 128 + (i64)ocs[j][r] * 8192 + (i64)olo[j][r];
          if (v != 0) atomicAdd((unsigned long long*)(o + 16 * j), (unsigned long long)v);
        }
      }
    }
  }
}

// Groups of 16 queries per prefix block, its slots and the parts of a row.
struct SharedPlan {
  int qw, qblocks, chunk, nchunks, parts;
};
SharedPlan shared_plan(int B, int P, int n_q, int n_kv) {
  const i64 m = (i64)B * (n_q / n_kv);
  SharedPlan p;
  p.qw = m <= 16 ? 1 : m <= 32 ? 2 : 4;
  p.qblocks = (int)((m + 16 * p.qw - 1) / (16 * p.qw));
  // about two blocks per CU
  const i64 want = imax(512 / ((i64)p.qblocks * n_kv), 1);
  const i64 tiles = P / 64, share = 4 / p.qw;
  i64 per = (tiles + want - 1) / want;
  per = (per + share - 1) / share * share;
  p.chunk = (int)imax(per, share) * 64;
  p.nchunks = P > 0 ? (P + p.chunk - 1) / p.chunk : 0;
  p.parts = p.nchunks * (4 / p.qw) + 4;
  return p;
}
int shared_args_ok(int B, int S, int n_q, int n_kv, int shared) {
  if (B < 0 || S < 0 || shared < 0 || shared > S || shared % DI_PAGE) return DI_EINVAL;
  if (n_q <= 0 || n_kv <= 0 || n_q % n_kv) return DI_EINVAL;
  const int G = n_q / n_kv;
  if (G != 1 && G != 2 && G != 4 && G != 8) return DI_ENOSYS;
  if (S > 131071) return DI_ERANGE;  // int32 MFMA accumulators of P.V
  return DI_OK;
}

}  // namespace

extern "C" {

int detllm_attn_decode_shared_work(int B, int S, int n_q, int n_kv, int shared, int64_t* bytes) {
  if (!bytes) return DI_EINVAL;
  if (const int rc = shared_args_ok(B, S, n_q, n_kv, shared)) return rc;
  const SharedPlan p = shared_plan(B, shared, n_q, n_kv);
  *bytes = (i64)B * n_q * p.parts * 12;
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
  const SharedPlan p = shared_plan(B, shared, n_q, n_kv);
  const i64 rows = (i64)B * n_q;
  if (!work || work_bytes < rows * p.parts * 12) return DI_ERANGE;
  SharedArgs a{};
  a.q8 = q8; a.tpos = tpos;
  a.kv = KVPages{(int8_t*)kpool, (int8_t*)vpool, table, width, n_kv};
  a.valid = valid; a.valid_stride = valid_stride; a.out = out; a.s_dev = s_dev; a.err = err;
  a.den = (i64*)work;
  a.cmax = (int32_t*)((char*)work + rows * p.parts * 8);
  a.B = B; a.S = S; a.P = shared; a.n_q = n_q; a.n_kv = n_kv; a.G = n_q / n_kv;
  a.chunk = p.chunk; a.nchunks = p.nchunks; a.qblocks = p.qblocks; a.parts = p.parts;
  const i64 blocks = (i64)p.nchunks * p.qblocks * n_kv + (i64)B * n_kv;
  if (blocks > 0x7fffffff) return DI_ERANGE;
  const dim3 grid((unsigned)blocks);
#define DI_SHARED(QW_)                                                        \
  hipLaunchKernelGGL((k_shared<QW_, 0>), grid, dim3(256), 0, s, a);           \
  hipLaunchKernelGGL((k_shared<QW_, 1>), grid, dim3(256), 0, s, a);           \
  hipLaunchKernelGGL((k_shared<QW_, 2>), grid, dim3(256), 0, s, a)
  if (p.qw == 1) { DI_SHARED(1); }
  else if (p.qw == 2) { DI_SHARED(2); }
  else { DI_SHARED(4); }
#undef DI_SHARED
  DI_LAUNCH_CHECK();
  return DI_OK;
}

}  // extern "C"
