// Decode attention (gfx950): the bodies of attention.hip's one-block and
// split-S kernels and of the windowed and accumulating forms of
// attn_long.hip.
#pragma once

#include "attn_tiles.h"

namespace {

struct DecodeArgs {
  const int8_t* q8;      // [B][n_q][128]
  const int64_t* tpos;   // [B][n_q]
  KVPages kv;
  const uint8_t* valid;  // [B][valid_stride]
  int64_t* out;          // [B][n_q * 128]
  int32_t* scratch;      // [B][n_q][S] when scores do not fit in LDS, else null
  const int64_t* s_dev;  // optional device bound on the scanned slots
  int S, n_q, n_kv;
  i64 valid_stride;
  int32_t* err;          // optional device error word (DI_ERR_SLOTS)
  // optional (both or neither): the attention-output merge's per-column
  // factor om [n_q * 128] and its row statistics ext [B][n_kv][2] — per
  // (row, kv head) block the largest v and the largest ~v over the block's
  // outputs v = out * om (int64, wrapping) and 0
  const int64_t* om;
  int64_t* ext;
};
// Of the accumulating form (ACC): each slot's p, summed over the kv head's query
// heads, is added to acc [B][n_kv][stride]. An argument of its own, so that the
// other kernels' arguments stay where they were: 16 bytes more in DecodeArgs moved
// those of the fused kernel behind it and cost its launch 0.3 of 10.5 us.
struct AccInto {
  int64_t* acc;
  i64 stride;
};

constexpr int DEC_MAX_PAGES = 1024;  // ceil(131071 / DI_PAGE)

constexpr int MAXG = 8;
constexpr i64 DECODE_LDS_BYTES = 48 * 1024;

constexpr int32_t SCORE_MASKED = INT32_MIN;  // |q.k| <= 128*128*128 < 2^31: never a score
constexpr int DEC_MAX_S = 131071;            // int32 MFMA accumulators of P.V
constexpr int VPRE = 4;                      // 64-slot steps of V loaded before the scores
// The same for the fused eight-wave kernel (one 16-channel block per wave):
// six steps (384 slots) measured fastest at c3's ~320 slots (4: 1.595, 6:
// 1.561, 8: 1.569 ms per b8 step): loads past the row's steps are wasted
// traffic through the CU's load path, and the steps past the prefetch cost a
// round trip in the P.V loop.
constexpr int VPRE_FUSED = 6;

// DPP max over each aligned row of 16 lanes (result in every lane of the row)
__device__ __forceinline__ int32_t row16_max(int32_t v) {
  v = ::max(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false));
  v = ::max(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false));
  v = ::max(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, false));
  v = ::max(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, false));
  return v;
}

// The slots a decode block numbers 0, 1, ...: the row's own (WholeRow), or
// the pages a windowed query sees (attn_long.hip's WinView). A view keeps
// pages whole: slot s lies at offset s % DI_PAGE of its page.
struct WholeRow {
  static constexpr bool kWhole = true;
  __device__ __forceinline__ int slot(int s) const { return s; }
  __device__ __forceinline__ int page(const KVPages& kv, int b, int s) const { return kv.page(b, s); }
  __device__ __forceinline__ bool sees(int) const { return true; }
};

// The p of a packed word (pack_p)
__device__ __forceinline__ int unpack_p(int32_t w) {
  return ((int)(int8_t)(w & 0xFF) + 64) * 128 + ((w >> 8) & 0xFF);
}

// Adds the p of slots [0, n), packed at pp[hh * stride + i] for G heads, to
// accrow[i]; zero sums leave their word alone. NT threads.
template <int G, int NT>
__device__ __forceinline__ void acc_add(const int32_t* pp, i64 stride, int n, int64_t* accrow) {
  for (int i = threadIdx.x; i < n; i += NT) {
    int sum = 0;
#pragma unroll
    for (int hh = 0; hh < G; ++hh) sum += unpack_p(pp[hh * stride + i]);
    if (sum != 0) accrow[i] += sum;
  }
}

// Attention of one (batch row b, kv head kvh) over its G query heads, whose
// int8 rows sit at qsrc[hh * 128] and DI-Exp constants at tsrc[hh] (global
// memory or LDS). NW waves (decode_body's template argument, 4 or 8).
//
// Scores and P.V run on v_mfma_i32_16x16x64_i8 with the G query heads as the
// 16 MFMA rows (rows >= G zero):
//   * scores: C[hh][slot] = sum_d q[hh][d] k[slot][d]; a wave takes blocks of
//     16 slots, B-fragment lane l = slot l % 16, bytes 16 (l / 16) (+ 64) of
//     the slot's K row (two MFMAs over the 128 channels);
//   * P.V with the prefill's exact hi/lo split of p in [0, 2^14]:
//     p = 128 hi + lo, sum p v = 128 (sum (hi - 64) v + 64 colsum v) + sum lo v;
//     A rows hh < G hold hi - 64 (resp. lo) of 64 consecutive slots, and row G
//     of the hi product holds ones, so C_hi[G][d] = colsum v over exactly the
//     slots of the B fragments; B-fragment lane l = channel l % 16, slots
//     16 (l / 16) .. + 15 of V^T (slot-contiguous). Wave w owns channels
//     (128 / NW) w .. + 128 / NW - 1 (8 / NW 16-channel blocks).
// Slots past S read zero V fragments (16-slot chunks starting at or past S),
// so their A values do not matter; the p of slots S .. ceil16(S) are 0.
// |accumulators| <= 128 * 128 * S < 2^31 for S <= 131071.
// p in [0, 2^14] packed as (hi - 64) | lo << 8 (p = 128 hi + lo; p = 0 packs
// as hi - 64 = -64, lo = 0)
__device__ __forceinline__ int32_t pack_p(i64 p) {
  const int hi = (int)(p >> 7), lo = (int)(p & 127);
  return (int32_t)((uint32_t)(uint8_t)(int8_t)(hi - 64) | ((uint32_t)lo << 8));
}

// MFMA A fragments of 16 packed p words (16 consecutive slots of one head):
// bytes 0 of the words -> hi - 64 fragment, bytes 1 -> lo
__device__ __forceinline__ void p_frags(const int32_t* pp, v4i& ahi, v4i& alo) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const v4i w = *(const v4i*)(pp + 4 * q);
    const uint32_t h01 = __builtin_amdgcn_perm((uint32_t)w[1], (uint32_t)w[0], 0x0c0c0400u);
    const uint32_t h23 = __builtin_amdgcn_perm((uint32_t)w[3], (uint32_t)w[2], 0x04000c0cu);
    const uint32_t l01 = __builtin_amdgcn_perm((uint32_t)w[1], (uint32_t)w[0], 0x0c0c0501u);
    const uint32_t l23 = __builtin_amdgcn_perm((uint32_t)w[3], (uint32_t)w[2], 0x05010c0cu);
    ahi[q] = (int)(h01 | h23);
    alo[q] = (int)(l01 | l23);
  }
}

// sum_s p_s v_s of the wave's channels from the hi/lo accumulators: lane
// (grp, l16), element r holds head 4 grp + r, channel 16 (NB wave + nb) + l16;
// the colsum of that channel sits in row G (lane 16 (G / 4) + l16, element
// G % 4). out_heads: the block's first head row of [.][128] int64.
// each(nb, r, value) sees every stored value. add: the values are added to
// out_heads (several blocks share it) instead of stored.
template <int G, int NB = 2, class Each>
__device__ __forceinline__ void store_pv(const v4i (&chi)[NB], const v4i (&clo)[NB],
                                         int64_t* out_heads, Each&& each, bool add = false) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, grp = lane >> 4;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int cs_src = (G / 4) * 16 + l16;
    const int32_t cs = __shfl(chi[nb][G % 4], cs_src, 64);
    const int d = wave * 16 * NB + nb * 16 + l16;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int hh = grp * 4 + r;
      if (hh < G) {
        const i64 o = ((i64)chi[nb][r] + 64 * (i64)cs) * 128 + (i64)clo[nb][r];
        if (add) atomicAdd((unsigned long long*)&out_heads[hh * 128 + d], (unsigned long long)o);
        else out_heads[hh * 128 + d] = o;
        each(nb, r, o);
      }
    }
  }
}
template <int G, int NB = 2>
__device__ __forceinline__ void store_pv(const v4i (&chi)[NB], const v4i (&clo)[NB],
                                         int64_t* out_heads, bool add = false) {
  store_pv<G, NB>(chi, clo, out_heads, [](int, int, i64) {}, add);
}

// The slots a decode block scans: a.S, bounded by the device count when one
// is given. Without one the load reads `always` (a pointer every launch
// has) and the value is selected after it: no branch around the load, whose
// merge would make every earlier load complete first. *over: the device
// count exceeds a.S; the reference would scan those slots, so the result
// would differ, and report_slots raises DI_ERR_SLOTS (after the kernel's
// last load: a pending atomic among loads makes every wait a full one).
__device__ __forceinline__ int scanned_slots(const DecodeArgs& a, const int64_t* always,
                                             bool* over) {
  const int64_t* p = a.s_dev ? a.s_dev : always;
  const i64 sd = p[0];
  *over = a.s_dev != nullptr && sd > (i64)a.S;
  return a.s_dev ? (int)imax(0, imin((i64)a.S, sd)) : a.S;
}
__device__ __forceinline__ void report_slots(const DecodeArgs& a, bool over, bool who) {
  if (over && who && a.err && threadIdx.x == 0) atomicOr(a.err, DI_ERR_SLOTS);
}

// K rows and validity flags of the first KPRE_SLOTS slots of the row, loaded
// before the fused kernel's Q/K/V epilogue so that their latency hides behind
// it; the slot the epilogue writes is taken from LDS instead. With NW waves a
// wave holds IT = KPRE_SLOTS / (64 NW) iterations of four 16-slot blocks.
constexpr int KPRE_SLOTS = 512;
template <int IT>
struct KPre {
  v4i kb[IT][4][2];
  int vf[IT][4];                 // 0 for slots of pages that are not mapped
  int pg[KPRE_SLOTS / DI_PAGE];  // the pages of those slots (-1: not mapped or past S)
  const int8_t* k_new;           // LDS, 128 bytes
  i64 new_slot;                  // -1: none
};

// S: the slots to scan (scanned_slots). pg_lds: the row's page ids for
// slots [0, S) (filled by the caller, before a barrier). Slots whose page is
// not mapped are masked and read page 0. VP: 64-slot steps of V loaded ahead.
// SCR: the scores live in the global scratch (a.scratch) instead of LDS (a
// compile-time choice: LDS-only code never issues flat accesses, which would
// wait on every outstanding load). NW: waves of the block (4 or 8): a wave
// takes every NW-th 16-slot block of the scores and 128 / NW channels of P.V.
// The merge factors of a lane's outputs (store_pv's layout: head 4 grp + r,
// channel 16 (NB wave + nb) + l16; heads past G read entry 0), loaded where
// the caller's first loads issue.
template <int G, int NB>
struct OmPre {
  static constexpr int RG = G < 4 ? G : 4;
  i64 v[NB][RG];
  __device__ __forceinline__ void load(const DecodeArgs& a, int kvh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, grp = lane >> 4;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < RG; ++r) {
        const int hh = grp * 4 + r;
        const int d = wave * 16 * NB + nb * 16 + l16;
        v[nb][r] = a.om[hh < G ? (kvh * G + hh) * 128 + d : 0];
      }
  }
};

// OMP: omp holds the merge factors (else decode_body loads them when a.ext
// is set). View: the slots (WholeRow above); ACC: their p are added to `into`.
template <int G, int VP, bool SCR, bool PRE = false, int NW = 4, bool OMP = false,
          class View = WholeRow, bool ACC = false>
__device__ __forceinline__ void decode_body(const DecodeArgs& a, int S, int kvh, int b,
                                            const int8_t* qsrc, const int64_t* tsrc,
                                            int32_t* sh_scores, const int32_t* pg_lds,
                                            const KPre<8 / NW>& pre = KPre<8 / NW>{},
                                            const OmPre<G, 8 / NW>& omp = OmPre<G, 8 / NW>{},
                                            const View& view = View{},
                                            const AccInto& into = AccInto{}) {
  static_assert(G <= 8, "query heads per kv head");
  static_assert(NW == 4 || NW == 8, "waves per block");
  constexpr int NT = NW * 64;  // threads
  constexpr int NB = 8 / NW;   // 16-channel blocks of P.V per wave
  constexpr int IT = 8 / NW;   // prefetched iterations per wave
  __shared__ i64 red_buf[32];
  BlockRedT<NT / 64> red{red_buf, 0, NT};
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int l16 = lane & 15, grp = lane >> 4;
  const int Spad = (a.S + 15) & ~15;
  int32_t* sc = SCR ? a.scratch + ((i64)b * a.n_q + kvh * G) * Spad : sh_scores;
  const uint8_t* vrow = a.valid + (i64)b * a.valid_stride;
  const int nstep = (S + 63) / 64;  // 64-slot steps of P.V
  auto pg_of = [&](int s) -> int {  // page of slot s < S, page 0 when not mapped
    const int pg = pg_lds[s >> 7];
    return pg < 0 ? 0 : pg;
  };

  // V fragments of 64-slot steps (a step lies in one page). Loads are
  // unconditional (no branch whose merge would make them complete early): a
  // 16-slot group at or past S reads slot 0's bytes, and every A row of such
  // a group, the colsum row included, is zero.
  auto vfrag = [&](int st, int nb) -> v4i {
    const int s0 = st * 64 + grp * 16;
    const int sl = s0 < S ? s0 : 0;
    const int8_t* vch = a.kv.vchan(pg_of(sl), kvh, wave * 16 * NB + nb * 16 + l16);
    return *(const v4i*)(vch + (sl & (DI_PAGE - 1)));
  };
  // the same for a step below KPRE_SLOTS with the pages in registers (no LDS
  // read before the load): slot st * 64 + 16 grp lies in page st / 2 (a group
  // at or past S reads offset 0 of that page, or of page 0 when it is not
  // mapped; its A rows are zero)
  auto vfrag_pre = [&](int st, int nb) -> v4i {
    const int s0 = st * 64 + grp * 16;
    const int sl = s0 < S ? s0 : 0;
    const int pg = pre.pg[st >> 1];
    const int8_t* vch = a.kv.vchan(pg < 0 ? 0 : pg, kvh, wave * 16 * NB + nb * 16 + l16);
    return *(const v4i*)(vch + (sl & (DI_PAGE - 1)));
  };

  // the merge factors of this lane's outputs, used after P.V
  constexpr int RG = OmPre<G, NB>::RG;
  OmPre<G, NB> oml;
  if (!OMP && a.ext != nullptr) oml.load(a, kvh);
  const OmPre<G, NB>& omv = OMP ? omp : oml;

  // query fragments (row l16 = head) and the heads' DI-Exp constants
  v4i qa0 = v4i{0, 0, 0, 0}, qa1 = v4i{0, 0, 0, 0};
  if (l16 < G) {
    qa0 = *(const v4i*)(qsrc + l16 * 128 + grp * 16);
    qa1 = *(const v4i*)(qsrc + l16 * 128 + 64 + grp * 16);
  }
  // per head: the fp64-estimate DI-Exp (intops.h dexp_est) when tpos < 2^23
  // (every score difference is below 2^22: |q8 . k8| <= 2^21), else the
  // integer form
  // (the fused kernel's constants are written during the score pass and
  // read after the maxima's barrier)
  i64 tph[G];
  if (!PRE) {
#pragma unroll
    for (int hh = 0; hh < G; ++hh) tph[hh] = tsrc[hh];
  }

  // ---- pass 1: scores on MFMA; masked slots marked; per-head row max.
  // Lane (grp, l16) holds C[4 grp + r][slot l16] in element r.
  int32_t mx[4] = {SCORE_MASKED, SCORE_MASKED, SCORE_MASKED, SCORE_MASKED};
  const int nblk = (S + 15) / 16;
  // blocks blk0 + NW u (u < 4) from K fragments kb and validity flags vf
  auto score4 = [&](int blk0, const v4i (&kb)[4][2], const int (&vf)[4]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int blk = blk0 + u * NW;
      if (blk < nblk) {  // wave-uniform
        v4i c = mfma16(qa0, kb[u][0], v4i{0, 0, 0, 0});
        c = mfma16(qa1, kb[u][1], c);
        const int s = blk * 16 + l16;
        const bool vis = s < S && vf[u] != 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int hh = grp * 4 + r;
          if (hh < G) {
            if (s < S) sc[hh * Spad + s] = vis ? c[r] : SCORE_MASKED;
            if (vis) mx[r] = ::max(mx[r], c[r]);
          }
        }
      }
    }
  };
  int blk0 = wave;
  if (PRE) {
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int bb = wave + 4 * NW * it;
      if (bb >= nblk) continue;  // wave-uniform
      v4i kb[4][2];
      int vf[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        kb[u][0] = pre.kb[it][u][0];
        kb[u][1] = pre.kb[it][u][1];
        if ((bb + u * NW) * 16 + l16 == pre.new_slot) {
          kb[u][0] = *(const v4i*)(pre.k_new + grp * 16);
          kb[u][1] = *(const v4i*)(pre.k_new + 64 + grp * 16);
        }
        vf[u] = pre.vf[it][u];
      }
      score4(bb, kb, vf);
    }
    blk0 = wave + 4 * NW * IT;
  }
  for (; blk0 < nblk; blk0 += 4 * NW) {
    v4i kb[4][2];
    int vraw[4], vf[4];
    bool ok[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = (blk0 + u * NW) * 16 + l16;
      const int sc_ = s < S ? s : 0;
      const int8_t* kr = a.kv.krow(pg_of(sc_), kvh, sc_ & (DI_PAGE - 1));
      kb[u][0] = *(const v4i*)(kr + grp * 16);
      kb[u][1] = *(const v4i*)(kr + 64 + grp * 16);
      // (the flag is loaded unconditionally and masked at use: no wait per block)
      vraw[u] = vrow[view.slot(sc_)];
      ok[u] = pg_lds[sc_ >> 7] >= 0 && view.sees(view.slot(sc_));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) vf[u] = ok[u] ? vraw[u] : 0;
    score4(blk0, kb, vf);
  }
  // the first VP steps of V, loaded now (the K fragments' registers are
  // free) to overlap the maxima, denominators and probabilities
  v4i vpre[VP][NB];
#pragma unroll
  for (int i = 0; i < VP; ++i)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      vpre[i][nb] = (PRE && i * 64 < KPRE_SLOTS) ? vfrag_pre(i, nb) : vfrag(i, nb);
  // per-head row maxima, two heads per block reduction (int32 scores biased
  // to order-preserving unsigned values)
  i64 hmax[G];
#pragma unroll
  for (int r = 0; r < 4; ++r) mx[r] = row16_max(mx[r]);
#pragma unroll
  for (int hh = 0; hh < G; hh += 2) {
    // head hh lives in lanes 16 (hh / 4) .. + 15, element hh % 4
    const int32_t m0 = grp == hh / 4 ? mx[hh % 4] : SCORE_MASKED;
    const int32_t m1 = hh + 1 < G && grp == (hh + 1) / 4 ? mx[(hh + 1) % 4] : SCORE_MASKED;
    uint32_t u0 = (uint32_t)m0 ^ 0x80000000u, u1 = (uint32_t)m1 ^ 0x80000000u;
    red.max2_u32(u0, u1);
    const int32_t r0 = (int32_t)(u0 ^ 0x80000000u), r1 = (int32_t)(u1 ^ 0x80000000u);
    hmax[hh] = r0 == SCORE_MASKED ? 0 : r0;  // no visible slot: max := 0, every p = 0
    if (hh + 1 < G) hmax[hh + 1] = r1 == SCORE_MASKED ? 0 : r1;
  }
  __syncthreads();
  if (PRE) {
#pragma unroll
    for (int hh = 0; hh < G; ++hh) tph[hh] = tsrc[hh];
  }
  // ---- pass 2: denominators (two heads per block reduction). When every
  // head takes the estimate path (the usual case), one loop serves all heads
  // and two slots per thread, the LDS reads of an iteration issued together.
  i64 den[G];
  bool allfast = true;
#pragma unroll
  for (int hh = 0; hh < G; ++hh) allfast = allfast && tph[hh] < ((i64)1 << 23);
  ExpEst Ef[G];
  if (DI_LIKELY(allfast)) {
#pragma unroll
    for (int hh = 0; hh < G; ++hh) {
      Ef[hh] = make_expest(tph[hh]);
      den[hh] = 0;
    }
    for (int s0 = tid; s0 < S; s0 += 2 * NT) {
      const int s1 = s0 + NT;
      const int s1c = s1 < S ? s1 : s0;
      int32_t x0[G], x1[G];
#pragma unroll
      for (int hh = 0; hh < G; ++hh) {
        x0[hh] = sc[hh * Spad + s0];
        x1[hh] = sc[hh * Spad + s1c];
      }
#pragma unroll
      for (int hh = 0; hh < G; ++hh) {
        if (x0[hh] != SCORE_MASKED) den[hh] += dexp_est((uint32_t)(hmax[hh] - x0[hh]), Ef[hh]);
        if (s1 < S && x1[hh] != SCORE_MASKED)
          den[hh] += dexp_est((uint32_t)(hmax[hh] - x1[hh]), Ef[hh]);
      }
    }
  } else {
#pragma unroll
  for (int hh = 0; hh < G; ++hh) {
    i64 acc = 0;
    if (tph[hh] < ((i64)1 << 23)) {
      const ExpEst Ee = make_expest(tph[hh]);
      for (int s = tid; s < S; s += NT) {
        const int32_t x = sc[hh * Spad + s];
        if (x != SCORE_MASKED) acc += dexp_est((uint32_t)(hmax[hh] - x), Ee);
      }
    } else {
      const ExpR E = make_exp(tph[hh]);
      for (int s = tid; s < S; s += NT) {
        const int32_t x = sc[hh * Spad + s];
        if (x != SCORE_MASKED) acc = wadd(acc, di_exp_neg((u64)wsub(hmax[hh], (i64)x), E));
      }
    }
    den[hh] = acc;
  }
  }
#pragma unroll
  for (int hh = 0; hh < G; hh += 2) {
    i64 d1 = hh + 1 < G ? den[hh + 1] : 0;
    red.sum2(den[hh], d1);
    den[hh] = imax(den[hh], 1);
    if (hh + 1 < G) den[hh + 1] = imax(d1, 1);
  }
  // ---- pass 3: p in [0, 2^14] as (hi - 64) | lo << 8 in place of the score
  // (0 for masked slots and the padding up to the next multiple of 16, i.e.
  // hi - 64 = -64, lo = 0)
  const int nchunk = (S + 15) / 16;
  bool pfast = allfast;
#pragma unroll
  for (int hh = 0; hh < G; ++hh) pfast = pfast && den[hh] < ((i64)1 << 34);
  if (DI_LIKELY(pfast)) {
    // as pass 2: every head, two slots per thread, reads first
    DivEst Df[G];
#pragma unroll
    for (int hh = 0; hh < G; ++hh) Df[hh] = make_divest(den[hh], 16384.0);
    const int lim = nchunk * 16;
    for (int s0 = tid; s0 < lim; s0 += 2 * NT) {
      const int s1 = s0 + NT;
      const int s1c = s1 < lim ? s1 : s0;
      int32_t x0[G], x1[G];
#pragma unroll
      for (int hh = 0; hh < G; ++hh) {
        x0[hh] = sc[hh * Spad + s0];
        x1[hh] = sc[hh * Spad + s1c];
      }
#pragma unroll
      for (int hh = 0; hh < G; ++hh) {
        i64 p0 = 0, p1 = 0;
        if (s0 < S && x0[hh] != SCORE_MASKED)
          p0 = rhad_est((double)dexp_est((uint32_t)(hmax[hh] - x0[hh]), Ef[hh]), Df[hh]);
        if (s1 < S && x1[hh] != SCORE_MASKED)
          p1 = rhad_est((double)dexp_est((uint32_t)(hmax[hh] - x1[hh]), Ef[hh]), Df[hh]);
        sc[hh * Spad + s0] = pack_p(p0);
        if (s1 < lim) sc[hh * Spad + s1] = pack_p(p1);
      }
    }
  } else {
#pragma unroll
  for (int hh = 0; hh < G; ++hh) {
    auto put = [&](int s, i64 p) { sc[hh * Spad + s] = pack_p(p); };
    if (tph[hh] < ((i64)1 << 23) && den[hh] < ((i64)1 << 34)) {
      // exps below 2^23, den < 2^34: p = rhad(ex 2^14, den) from rhad_est
      const ExpEst Ee = make_expest(tph[hh]);
      const DivEst D = make_divest(den[hh], 16384.0);
      for (int s = tid; s < nchunk * 16; s += NT) {
        i64 p = 0;
        if (s < S) {
          const int32_t x = sc[hh * Spad + s];
          if (x != SCORE_MASKED) p = rhad_est((double)dexp_est((uint32_t)(hmax[hh] - x), Ee), D);
        }
        put(s, p);
      }
    } else {
      const ExpR E = make_exp(tph[hh]);
      const Recip Rd = make_recip(den[hh]);
      for (int s = tid; s < nchunk * 16; s += NT) {
        i64 p = 0;
        if (s < S) {
          const int32_t x = sc[hh * Spad + s];
          if (x != SCORE_MASKED) {
            const i64 ex = di_exp_neg((u64)wsub(hmax[hh], (i64)x), E);
            p = to_i32(rhad_r(shl(ex, 14), Rd));
          }
        }
        put(s, p);
      }
    }
  }
  }
  __syncthreads();
  if constexpr (ACC) {
    // (a query at a slot that is not valid adds nothing)
    if (S > 0 && vrow[S - 1] != 0)
      acc_add<G, NT>(sc, Spad, S, into.acc + ((i64)b * a.n_kv + kvh) * into.stride);
  }
  // ---- P.V on MFMA
  v4i chi[NB], clo[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) chi[nb] = clo[nb] = v4i{0, 0, 0, 0};
  auto pv_step = [&](int st, const v4i (&vb)[NB]) {
    v4i ahi = v4i{0, 0, 0, 0}, alo = v4i{0, 0, 0, 0};
    const int s0 = st * 64 + grp * 16;
    if (l16 < G && s0 < S) {
      p_frags(sc + l16 * Spad + s0, ahi, alo);  // 16 packed p of head l16
    } else if (l16 == G && s0 < S) {
      ahi = v4i{0x01010101, 0x01010101, 0x01010101, 0x01010101};  // colsum row
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      chi[nb] = mfma16(ahi, vb[nb], chi[nb]);
      clo[nb] = mfma16(alo, vb[nb], clo[nb]);
    }
  };
#pragma unroll
  for (int i = 0; i < VP; ++i)
    if (i < nstep) pv_step(i, vpre[i]);
  for (int st0 = VP; st0 < nstep; st0 += 4) {
    v4i vb[4][NB];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) vb[i][nb] = vfrag(st0 + i, nb);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (st0 + i < nstep) pv_step(st0 + i, vb[i]);
  }
  if (a.ext == nullptr) {
    store_pv<G, NB>(chi, clo, a.out + (i64)b * a.n_q * 128 + kvh * G * 128);
    return;
  }
  // with the merge's row statistics of the block's outputs (0 included, as
  // merge_rowcol_row starts its extremes from 0)
  i64 vmx = 0, nmn = -1;
  store_pv<G, NB>(chi, clo, a.out + (i64)b * a.n_q * 128 + kvh * G * 128,
                  [&](int nb, int r, i64 o) {
                    const i64 v = wmul(o, omv.v[nb][r < RG ? r : 0]);
                    vmx = imax(vmx, v);
                    nmn = imax(nmn, ~v);
                  });
  red.max2(vmx, nmn);
  if (tid == 0) {
    a.ext[((i64)b * a.n_kv + kvh) * 2] = vmx;
    a.ext[((i64)b * a.n_kv + kvh) * 2 + 1] = nmn;
  }
}

// ---------------------------------------------------------------------------
// Split-S decode attention: the slots of a (row, kv head) are cut into chunks
// of `chunk` slots (a multiple of the page), one block per chunk, in two
// launches:
//   k_attn_split_scores: the chunk's scores (int32, to a global scratch) and
//     its per-head maximum over visible slots;
//   k_attn_split_pv: the row maximum (the maximum of the chunk maxima — the
//     TRUE row max, DI-Exp being not multiplicative), the denominator over
//     ALL the row's slots (every block sums the same integers, so every block
//     holds the same den), then p of the chunk's slots and their P.V into the
//     chunk's own int64 partial context.
// The context is the sum of the partials (exact integer addition, in any
// order); the attention-output merge sums them. Same integers as
// k_attn_decode for every chunking.

constexpr int SPLIT_MAX_CHUNK = 4096;                  // slots per chunk
constexpr int SPLIT_MAX_PAGES = SPLIT_MAX_CHUNK / DI_PAGE;
constexpr int SPLIT_DL = 4;  // 16-byte loads of scores in flight per thread and head

struct SplitArgs {
  DecodeArgs d;     // scratch: scores [B][n_q][spad]; out: partials [ns][B][n_q * 128]
  int32_t* cmax;    // [B][n_q][ns] chunk maxima (SCORE_MASKED: no visible slot)
  int chunk, ns;
  i64 spad;         // row stride of the scores (>= S)
  i64 out_stride;   // elements between partials (B * n_q * 128)
  // out is one [B][n_q * 128] context: zeroed by the scores launch, every
  // chunk's partial added to it (integer adds: any order gives the same sum)
  int add;
};

// Chunk c of (row b, kv head kvh). View as in decode_body: a view that is not
// the whole row knows its own slot count (view.n) and calls this for each of
// its chunks.
template <int G, class View = WholeRow>
__device__ __forceinline__ void split_scores_chunk(const SplitArgs& sa, int kvh, int b, int c,
                                                   const View& view = View{}) {
  const DecodeArgs& a = sa.d;
  __shared__ i64 red_buf[32];
  __shared__ int32_t pg_lds[SPLIT_MAX_PAGES];
  BlockRedT<4> red{red_buf, 0, 256};
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l16 = lane & 15, grp = lane >> 4;
  const int lo = c * sa.chunk;
  const i64 q0 = (i64)b * a.n_q + kvh * G;
  // the chunk's pages (below the launch's bound a.S) and the queries load
  // beside the device's slot count, not after it
  int bound = a.S;
  if constexpr (!View::kWhole) bound = view.n;
  const int npg = (::min(sa.chunk, bound - lo) + DI_PAGE - 1) / DI_PAGE;
  const int pgv = tid < npg ? view.page(a.kv, b, lo + tid * DI_PAGE) : -1;
  v4i qa0 = v4i{0, 0, 0, 0}, qa1 = v4i{0, 0, 0, 0};
  if (l16 < G) {
    const int8_t* qsrc = a.q8 + q0 * 128;
    qa0 = *(const v4i*)(qsrc + l16 * 128 + grp * 16);
    qa1 = *(const v4i*)(qsrc + l16 * 128 + 64 + grp * 16);
  }
  if (sa.add && c == 0)
    for (int i = tid; i < G * 128; i += 256) a.out[q0 * 128 + i] = 0;
  bool over = false;
  int S = bound;
  if constexpr (View::kWhole) S = scanned_slots(a, a.tpos, &over);
  const int hi = ::min(lo + sa.chunk, S);
  int32_t* cm = sa.cmax + q0 * sa.ns + c;  // head hh at cm[hh * ns]
  report_slots(a, over, kvh == 0 && c == 0);
  if (lo >= hi) {  // block-uniform: a chunk past the scanned slots
    if (tid < G) cm[tid * sa.ns] = SCORE_MASKED;
    return;
  }
  if (tid < npg) pg_lds[tid] = pgv;
  __syncthreads();
  int32_t* sc = a.scratch + q0 * sa.spad;
  const uint8_t* vrow = a.valid + (i64)b * a.valid_stride;
  int32_t mx[4] = {SCORE_MASKED, SCORE_MASKED, SCORE_MASKED, SCORE_MASKED};
  const int blo = lo / 16, bhi = (hi + 15) / 16;
  for (int blk0 = blo + wave; blk0 < bhi; blk0 += 16) {
    v4i kb[4][2];
    int vraw[4], vf[4], ok[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = (blk0 + u * 4) * 16 + l16;
      const int sc_ = s < hi ? s : lo;
      const int pg = pg_lds[(sc_ - lo) / DI_PAGE];
      const int8_t* kr = a.kv.krow(pg < 0 ? 0 : pg, kvh, sc_ & (DI_PAGE - 1));
      kb[u][0] = *(const v4i*)(kr + grp * 16);
      kb[u][1] = *(const v4i*)(kr + 64 + grp * 16);
      vraw[u] = vrow[view.slot(sc_)];  // masked at use (no wait per block)
      ok[u] = pg >= 0 && view.sees(view.slot(sc_)) ? 0xFF : 0;
      asm("" : "+v"(ok[u]));  // (opaque, or the flag's load moves behind a branch on it)
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) vf[u] = vraw[u] & ok[u];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int blk = blk0 + u * 4;
      if (blk < bhi) {  // wave-uniform
        v4i cc = mfma16(qa0, kb[u][0], v4i{0, 0, 0, 0});
        cc = mfma16(qa1, kb[u][1], cc);
        const int s = blk * 16 + l16;
        const bool vis = s < hi && vf[u] != 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int hh = grp * 4 + r;
          if (hh < G) {
            if (s < hi) sc[hh * sa.spad + s] = vis ? cc[r] : SCORE_MASKED;
            if (vis) mx[r] = ::max(mx[r], cc[r]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) mx[r] = row16_max(mx[r]);
#pragma unroll
  for (int hh = 0; hh < G; ++hh) {
    const int32_t mine = grp == hh / 4 ? mx[hh % 4] : SCORE_MASKED;
    const i64 m = red.max((i64)mine);
    if (tid == 0) cm[hh * sa.ns] = (int32_t)m;
  }
}

// ACC: the chunk's p are added to `into`.
template <int G, class View = WholeRow, bool ACC = false>
__device__ __forceinline__ void split_pv_chunk(const SplitArgs& sa, int kvh, int b, int c,
                                               const View& view = View{},
                                               const AccInto& into = AccInto{}) {
  const DecodeArgs& a = sa.d;
  extern __shared__ __attribute__((aligned(16))) int32_t p_lds[];  // [G][chunk] packed p
  __shared__ i64 red_buf[32];
  __shared__ int32_t pg_lds[SPLIT_MAX_PAGES];
  BlockRedT<4> red{red_buf, 0, 256};
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l16 = lane & 15, grp = lane >> 4;
  const int lo = c * sa.chunk;
  const i64 q0 = (i64)b * a.n_q + kvh * G;
  int64_t* outp = a.out + (sa.add ? 0 : c * sa.out_stride) + q0 * 128;
  // (none of these depends on the device's slot count, which loads last: the
  // page id, then per head the constant and its chunk maxima, each waited for)
  int bound = a.S;
  if constexpr (!View::kWhole) bound = view.n;
  const int npg = (::min(sa.chunk, bound - lo) + DI_PAGE - 1) / DI_PAGE;
  const int pgv = tid < npg ? view.page(a.kv, b, lo + tid * DI_PAGE) : -1;
  i64 tph[G], hmax[G];
#pragma unroll
  for (int hh = 0; hh < G; ++hh) {
    tph[hh] = a.tpos[q0 + hh];
    i64 m = SCORE_MASKED;
    const int32_t* cmh = sa.cmax + (q0 + hh) * sa.ns;
    int ns = sa.ns;
    if constexpr (!View::kWhole) ns = (view.n + sa.chunk - 1) / sa.chunk;
    for (int k = 0; k < ns; ++k) m = imax(m, (i64)cmh[k]);
    hmax[hh] = m == (i64)SCORE_MASKED ? 0 : m;  // no visible slot: max := 0, every p = 0
  }
  bool over;
  int S = bound;
  if constexpr (View::kWhole) S = scanned_slots(a, a.tpos, &over);
  const int hi = ::min(lo + sa.chunk, S);
  if (lo >= hi) {  // block-uniform: this chunk contributes nothing
    if (!sa.add)
      for (int i = tid; i < G * 128; i += 256) outp[i] = 0;
    return;
  }
  if (tid < npg) pg_lds[tid] = pgv;
  __syncthreads();
  // V fragments of the chunk's first VPRE 64-slot steps (a step lies in one
  // page), loaded before the denominator pass
  auto vfrag = [&](int st, int nb) -> v4i {  // unconditional, as in decode_body
    const int s0 = st * 64 + grp * 16;
    const int sl = s0 < hi ? s0 : lo;
    const int pg = pg_lds[(sl - lo) / DI_PAGE];
    const int8_t* vch = a.kv.vchan(pg < 0 ? 0 : pg, kvh, wave * 32 + nb * 16 + l16);
    return *(const v4i*)(vch + (sl & (DI_PAGE - 1)));
  };
  const int st_lo = lo / 64, st_hi = (hi + 63) / 64;
  v4i vpre[VPRE][2];
#pragma unroll
  for (int i = 0; i < VPRE; ++i)
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) vpre[i][nb] = vfrag(st_lo + i, nb);
  const int32_t* sc = a.scratch + q0 * sa.spad;
  // denominators over every scanned slot of the row: 16 bytes of scores per
  // load and SPLIT_DL loads in flight (rows of scores start at multiples of
  // 128 slots; a vector that reaches past S is cut there). One score per load,
  // each waited for in turn, made this pass a chain of S / 256 round trips.
  i64 den[G];
#pragma unroll
  for (int hh = 0; hh < G; ++hh) {
    i64 acc = 0;
    if (tph[hh] < ((i64)1 << 23)) {
      const ExpEst Ee = make_expest(tph[hh]);
      const int32_t* row = sc + hh * sa.spad;
      const int hm = (int)hmax[hh];
      for (int s0 = 4 * tid; s0 < S; s0 += 1024 * SPLIT_DL) {
        v4i x[SPLIT_DL];
#pragma unroll
        for (int u = 0; u < SPLIT_DL; ++u) {
          const int s = s0 + 1024 * u;
          x[u] = *(const v4i*)(row + (s < S ? s : s0));
        }
#pragma unroll
        for (int u = 0; u < SPLIT_DL; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (s0 + 1024 * u + r < S && x[u][r] != SCORE_MASKED)
              acc += dexp_est((uint32_t)(hm - x[u][r]), Ee);
      }
    } else {
      const ExpR E = make_exp(tph[hh]);
      for (int s = tid; s < S; s += 256) {
        const int32_t x = sc[hh * sa.spad + s];
        if (x != SCORE_MASKED) acc = wadd(acc, di_exp_neg((u64)wsub(hmax[hh], (i64)x), E));
      }
    }
    den[hh] = imax(red.sum(acc), 1);
  }
  // p of the chunk's slots, packed into LDS (0 for masked slots and the
  // padding to the next multiple of 16)
  const int n16 = (hi - lo + 15) / 16 * 16;
#pragma unroll
  for (int hh = 0; hh < G; ++hh) {
    int32_t* ph = p_lds + hh * sa.chunk;
    if (tph[hh] < ((i64)1 << 23) && den[hh] < ((i64)1 << 34)) {
      const ExpEst Ee = make_expest(tph[hh]);
      const DivEst D = make_divest(den[hh], 16384.0);
      for (int i = 4 * tid; i < n16; i += 1024) {  // (n16 is a multiple of 16, within the chunk)
        const v4i x = *(const v4i*)(sc + hh * sa.spad + lo + i);
        v4i w;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          i64 p = 0;
          if (lo + i + r < hi && x[r] != SCORE_MASKED)
            p = rhad_est((double)dexp_est((uint32_t)((int)hmax[hh] - x[r]), Ee), D);
          w[r] = pack_p(p);
        }
        *(v4i*)(ph + i) = w;
      }
    } else {
      const ExpR E = make_exp(tph[hh]);
      const Recip Rd = make_recip(den[hh]);
      for (int i = tid; i < n16; i += 256) {
        i64 p = 0;
        if (lo + i < hi) {
          const int32_t x = sc[hh * sa.spad + lo + i];
          if (x != SCORE_MASKED) {
            const i64 ex = di_exp_neg((u64)wsub(hmax[hh], (i64)x), E);
            p = to_i32(rhad_r(shl(ex, 14), Rd));
          }
        }
        ph[i] = pack_p(p);
      }
    }
  }
  __syncthreads();
  if constexpr (ACC) {
    if (a.valid[(i64)b * a.valid_stride + S - 1] != 0)
      acc_add<G, 256>(p_lds, sa.chunk, hi - lo,
                      into.acc + ((i64)b * a.n_kv + kvh) * into.stride + lo);
  }
  // P.V of the chunk
  v4i chi[2] = {v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}}, clo[2] = {v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}};
  auto pv_step = [&](int st, const v4i (&vb)[2]) {
    v4i ahi = v4i{0, 0, 0, 0}, alo = v4i{0, 0, 0, 0};
    const int s0 = st * 64 + grp * 16;
    if (l16 < G && s0 < hi) {
      p_frags(p_lds + l16 * sa.chunk + (s0 - lo), ahi, alo);
    } else if (l16 == G && s0 < hi) {
      ahi = v4i{0x01010101, 0x01010101, 0x01010101, 0x01010101};  // colsum row
    }
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      chi[nb] = mfma16(ahi, vb[nb], chi[nb]);
      clo[nb] = mfma16(alo, vb[nb], clo[nb]);
    }
  };
#pragma unroll
  for (int i = 0; i < VPRE; ++i)
    if (st_lo + i < st_hi) pv_step(st_lo + i, vpre[i]);
  for (int st0 = st_lo + VPRE; st0 < st_hi; st0 += 4) {
    v4i vb[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) vb[i][nb] = vfrag(st0 + i, nb);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (st0 + i < st_hi) pv_step(st0 + i, vb[i]);
  }
  store_pv<G>(chi, clo, outp, sa.add != 0);
}

}  // namespace
