// Integer GQA attention over the int8 KV cache (gfx950).
//
// Semantics (bit-exact): scores = q8 . k8 (int32); DI-Softmax with the TRUE
// row max over visible slots (ops/di_softmax.py:33-61 — DI-Exp is not
// multiplicative, so no online rescaling); probabilities
// p = round_half_away_div(exp << 14, max(sum exp, 1)) in [0, 2^14]; context
// = sum_s p_s * v_s exactly in int64 (model.py:363-402 and the hi/lo GEMM of
// backends.py:152-164 produce the same integer). Slot s is visible to the
// query at absolute slot S_past + t iff s <= S_past + t and valid[b][s]
// (model.py:259-266).
//
// Cache layout in HBM: paged (common.h KVPages). A row's slots map through
// its page table to pages of DI_PAGE = 128 slots; a page holds K rows
// [n_kv][128 slots][128] and V transposed [n_kv][128 channels][128 slots], so
// both the MFMA B-fragments of P.V (16 consecutive slots per lane) and the
// decode reduction over slots read slot-contiguous bytes. A prefill key tile
// is exactly one page.
//
// Prefill (k_attn_prefill): block = 64 queries of one head, 4 waves of 16.
// Scores are computed transposed, S^T = K . Q^T, with v_mfma_i32_16x16x64_i8:
// lane l then holds ONE query (l % 16) and 16 slots of each 64-slot tile, so
// the row max, the denominator and the DI-Exp / normalisation divisors are
// per-lane scalars. Three passes over the key tiles (max, denominator,
// normalise + P.V) recompute S^T on MFMA. P.V uses the same fragments: the
// 15-bit p is split as p = 128*hi + lo, and sum p.v =
// 128*(sum (hi-64).v + 64*colsum(v)) + sum lo.v, both products on i8 MFMA
// (hi-64 in [-64, 64], lo in [0, 127]).
//
// Decode (k_attn_decode): block = one (batch row, kv head), all q heads of
// its group; scores live in LDS (or a global scratch when they do not fit);
// every reduction is an exact integer max/sum.

#include "attn_decode.h"
#include "attn_prefill.h"
#include "qkv_epilogue.h"

namespace {

__global__ __launch_bounds__(256, 2) void k_attn_prefill(PrefillArgs a) {
  keep_hidden_args();
  prefill_body<false, false>(a);
}

template <int G, bool SCR>
__global__ __launch_bounds__(256) void k_attn_decode(DecodeArgs a) {
  keep_hidden_args();
  extern __shared__ __attribute__((aligned(16))) int32_t sh_scores[];
  __shared__ int32_t pg_lds[DEC_MAX_PAGES];
  const int kvh = blockIdx.x, b = blockIdx.y;
  const i64 q0 = (i64)b * a.n_q + kvh * G;
  bool over;
  const int S = scanned_slots(a, a.tpos, &over);
  const int npages = (a.S + DI_PAGE - 1) / DI_PAGE;
  for (int i = threadIdx.x; i < npages; i += 256) pg_lds[i] = a.kv.page(b, (i64)i * DI_PAGE);
  if (npages == 0 && threadIdx.x == 0) pg_lds[0] = -1;  // S = 0: loads read page 0
  __syncthreads();
  decode_body<G, VPRE, SCR>(a, S, kvh, b, a.q8 + q0 * 128, a.tpos + q0, sh_scores, pg_lds);
  report_slots(a, over, kvh == 0);
}

// Decode step with the Q/K/V epilogue fused in (G <= 2): waves 0..G-1 finish
// the block's query heads into LDS, wave G writes the key head and wave G + 1
// the value head of this step's slot into the cache (the other waves only
// prefetch); after one barrier the block's QAD_WAVES waves attend over every
// slot, the new one included (two waves per SIMD, each with half the slots
// and channels of a four-wave block). NS1: the Q/K/V product has no K split
// (qa.nsplit == 1). SCR as in decode_body.
constexpr int QAD_WAVES = 8;
template <int G, bool NS1, bool SCR>
__global__ __launch_bounds__(QAD_WAVES * 64) void k_qkv_attn_decode(DecodeArgs a, QKVArgs qa) {
  keep_hidden_args();
  constexpr int NW = QAD_WAVES, NT = NW * 64, IT = 8 / NW;
  static_assert(G + 2 <= NW, "one wave per head slot");
  extern __shared__ __attribute__((aligned(16))) int32_t sh_scores[];
  __shared__ __attribute__((aligned(16))) int8_t q_lds[G][128];
  __shared__ int64_t t_lds[G];
  __shared__ int64_t am_lds[G];
  const int kvh = blockIdx.x, b = blockIdx.y;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));  // wave-uniform
  // (kernel arguments pass through opaque_* below: the optimizer would
  // otherwise fold selects between them into loads from selected argument
  // addresses, each behind its own wait)
  const int n_q = opaque_i32(qa.n_q), n_kv = opaque_i32(qa.n_kv);
  const int slotw = w < G ? kvh * G + w : w == G ? n_q + kvh : w == G + 1 ? n_q + n_kv + kvh : -1;
  __shared__ __attribute__((aligned(16))) int8_t k_new[128];
  __shared__ int32_t pg_lds[DEC_MAX_PAGES];
  const int lane = threadIdx.x & 63, l16 = lane & 15, grp = lane >> 4;
  constexpr int NPK = KPRE_SLOTS / DI_PAGE;
  // 1. loads whose addresses follow from the kernel arguments alone. The
  // block's scalars come from one vector load (lane i reads word i) and the
  // pages of the prefetched slots from another, instead of a chain of scalar
  // loads (a scalar-load wait covers every scalar load in flight).
  //   word 0 position, 1 xk, 2 xm, 3 the step's slot (device scalar), 4 the
  //   scanned-slot bound (device scalar), 5-8 vq_m, vq_k, ks_m, ks_k of the
  //   kv head; other lanes (and absent device scalars) read the position
  const int64_t* const pos_p = opaque_ptr(qa.positions) + b;
  const int64_t* const sb_p = opaque_ptr(qa.slot_base_dev);
  const int64_t* const sd_p = opaque_ptr(a.s_dev);
  const int64_t* const xk_p = opaque_ptr(qa.xk) + b;
  const int64_t* const xm_p = opaque_ptr(qa.xm) + b;
  const int64_t* const vqm_p = opaque_ptr(qa.vq_m) + kvh;
  const int64_t* const vqk_p = opaque_ptr(qa.vq_k) + kvh;
  const int64_t* const ksm_p = opaque_ptr(qa.ks_m) + kvh;
  const int64_t* const ksk_p = opaque_ptr(qa.ks_k) + kvh;
  const int64_t* wq = pos_p;
  wq = lane == 1 ? xk_p : wq;
  wq = lane == 2 ? xm_p : wq;
  wq = lane == 3 && sb_p ? sb_p : wq;
  wq = lane == 4 && sd_p ? sd_p : wq;
  wq = lane == 5 ? vqm_p : wq;
  wq = lane == 6 ? vqk_p : wq;
  wq = lane == 7 ? ksm_p : wq;
  wq = lane == 8 ? ksk_p : wq;
  const i64 word = ld_global(wq);
  // page j of the row for lanes j < NPK with slots below a.S (<= width * 128,
  // so j < width), else page 0's entry (masked below)
  const bool pk_ok = lane < NPK && lane * DI_PAGE < a.S;
  const int32_t pword = a.kv.table[(i64)b * a.kv.width + (pk_ok ? lane : 0)];
  // the row's page ids (stored to LDS after the epilogue)
  // (npages <= width: each load is in bounds, the ones past npages masked)
  const int npages = (a.S + DI_PAGE - 1) / DI_PAGE;
  int pgv[DEC_MAX_PAGES / NT];
#pragma unroll
  for (int q = 0; q < DEC_MAX_PAGES / NT; ++q) {
    const int i = (int)threadIdx.x + NT * q;
    pgv[q] = a.kv.table[(i64)b * a.kv.width + (i < npages ? i : 0)];
  }
  // the head slot's per-channel loads (unconditional: a wave without a head
  // slot loads slot 0's and ignores them, so no branch merge forces the loads
  // to complete early)
  const int slotl = slotw >= 0 ? slotw : 0;
  QKVHeadIn in = qkv_head_load<NS1>(qa, b, slotl, QKVScalars{});
  // the merge factors of this wave's outputs (for the row statistics)
  OmPre<G, 8 / NW> omp;
  if (a.ext != nullptr) omp.load(a, kvh);
  // (every load above is issued before the wait for the gathered scalars)
  __builtin_amdgcn_sched_barrier(0);
  in.pos_raw = readlane64(word, 0);
  in.xk = readlane64(word, 1);
  in.xm = readlane64(word, 2);
  in.base = sb_p ? readlane64(word, 3) : qa.slot_base;
  in.vqm = readlane64(word, 5);
  in.vqk = readlane64(word, 6);
  in.ksm = readlane64(word, 7);
  in.ksk = readlane64(word, 8);
  const i64 sdev = readlane64(word, 4);
  const bool over = sd_p != nullptr && sdev > (i64)a.S;
  const int S = sd_p ? (int)imax(0, imin((i64)a.S, sdev)) : a.S;
  const i64 base = in.base;
  qkv_head_rope_load(qa, slotl, in);  // waits for the position only
  // 2. the loads that depend on those: this wave's K rows of the scores
  // pass's first iterations (the pass masks slots at or past the scanned
  // count and slots of pages that are not mapped)
  int pgk[NPK];
#pragma unroll
  for (int j = 0; j < NPK; ++j)
    pgk[j] = j * DI_PAGE < a.S ? __builtin_amdgcn_readlane(pword, j) : -1;
  KPre<IT> pre;
  int vraw[IT][4];
  bool vok[IT][4];
  {
    const uint8_t* vrow = a.valid + (i64)b * a.valid_stride;
#pragma unroll
    for (int it = 0; it < IT; ++it)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = (w + 4 * NW * it + u * NW) * 16 + l16;  // < KPRE_SLOTS
        // slots at or past the scanned count read slot 0 (one cached line
        // instead of rows nobody scores; the pass masks them)
        const int sc_ = s < S ? s : 0;
        const int j = sc_ >> 7;
        int pg = pgk[0];
#pragma unroll
        for (int jj = 1; jj < NPK; ++jj) pg = j == jj ? pgk[jj] : pg;
        const int8_t* kr = a.kv.krow(pg < 0 ? 0 : pg, kvh, sc_ & (DI_PAGE - 1));
        pre.kb[it][u][0] = *(const v4i*)(kr + grp * 16);
        pre.kb[it][u][1] = *(const v4i*)(kr + 64 + grp * 16);
        vraw[it][u] = vrow[sc_];  // masked after the epilogue: no wait here
        vok[it][u] = pg >= 0;
      }
    pre.k_new = k_new;
#pragma unroll
    for (int j = 0; j < NPK; ++j) pre.pg[j] = pgk[j];
  }
  // 3. the epilogue
  if (slotw >= 0)
    qkv_head_compute(qa, b, slotw, in, w < G ? q_lds[w] : nullptr, nullptr,
                     w == G ? k_new : nullptr, w < G ? &am_lds[w] : nullptr);
  if (slotw >= 0) qkv_head_report(qa, slotw, in);
#pragma unroll
  for (int it = 0; it < IT; ++it)
#pragma unroll
    for (int u = 0; u < 4; ++u) pre.vf[it][u] = vok[it][u] ? vraw[it][u] : 0;
  // T = 1: the step's slot is base (when its page is not mapped nothing was
  // written, and the slot is masked: the substituted row is never a score)
  pre.new_slot = base;
#pragma unroll
  for (int q = 0; q < DEC_MAX_PAGES / NT; ++q) {
    const int i = (int)threadIdx.x + NT * q;
    if (i < npages) pg_lds[i] = pgv[q];  // (loaded unconditionally above)
  }
  __syncthreads();
  // the query heads' DI-Exp constants (one lane's serial chain per head) on
  // the last wave, while the others start the scores; decode_body reads
  // them after its maxima's barrier
  if (w == NW - 1 && lane < G)
    t_lds[lane] = q_head_tpos(qa, am_lds[lane], in.ksm, in.ksk, nullptr);
  decode_body<G, VPRE_FUSED, SCR, true, NW, true>(a, S, kvh, b, &q_lds[0][0], t_lds, sh_scores,
                                                  pg_lds, pre, omp);
  report_slots(a, over, kvh == 0);
}

template <int G>
__global__ __launch_bounds__(256) void k_attn_split_scores(SplitArgs sa) {
  keep_hidden_args();
  split_scores_chunk<G>(sa, blockIdx.x, blockIdx.y, blockIdx.z);
}
template <int G>
__global__ __launch_bounds__(256) void k_attn_split_pv(SplitArgs sa) {
  keep_hidden_args();
  split_pv_chunk<G>(sa, blockIdx.x, blockIdx.y, blockIdx.z);
}

}  // namespace

extern "C" {

int detllm_attn_prefill(const int8_t* q8, const int64_t* tpos, const int8_t* kpool,
                        const int8_t* vpool, const int32_t* table, int width,
                        const uint8_t* valid, int64_t valid_stride, int B, int T, int S_past,
                        int n_q, int n_kv, int64_t* out, hipStream_t s) {
  if (B <= 0 || T <= 0) return DI_OK;
  const i64 S = (i64)S_past + T;
  if (n_q <= 0 || n_kv <= 0 || n_q % n_kv || S_past < 0 || !kv_ok(kpool, vpool, table, width) ||
      S > (i64)width * DI_PAGE || valid_stride < S || !q8 || !tpos || !valid || !out)
    return DI_EINVAL;
  if (S > 131071) return DI_ERANGE;  // int32 MFMA accumulators of P.V
  PrefillArgs a{q8, tpos, KVPages{(int8_t*)kpool, (int8_t*)vpool, table, width, n_kv}, valid, out,
                T, (int)S, S_past, n_q, n_kv, B, valid_stride};
  const i64 pairs = (i64)(((T + 63) / 64 + 1) / 2) * n_q * B;
  if (2 * pairs > 0x7fffffff) return DI_ERANGE;
  hipLaunchKernelGGL(k_attn_prefill, dim3((unsigned)(2 * pairs)), dim3(256), prefill_lds(S), s, a);
  DI_LAUNCH_CHECK();
  return DI_OK;
}

// Decode (one query per batch row). S: slots to scan (<= width * 128);
// s_dev: optional device scalar that further bounds it (graph replay).
// scratch may be null when n_q/n_kv * ceil16(S) * 4 bytes fit in 48 KiB of LDS.
int detllm_attn_decode(const int8_t* q8, const int64_t* tpos, const int8_t* kpool,
                       const int8_t* vpool, const int32_t* table, int width,
                       const uint8_t* valid, int64_t valid_stride, int B, int S, int n_q, int n_kv,
                       const int64_t* s_dev, int32_t* scratch, int64_t* out, int32_t* err,
                       hipStream_t s) {
  if (B <= 0) return DI_OK;
  if (n_q <= 0 || n_kv <= 0 || n_q % n_kv || S < 0 || !kv_ok(kpool, vpool, table, width) ||
      S > (i64)width * DI_PAGE || valid_stride < S || !q8 || !tpos || !valid || !out)
    return DI_EINVAL;
  const int G = n_q / n_kv;
  if (G > MAXG) return DI_ENOSYS;
  if (S > DEC_MAX_S) return DI_ERANGE;  // int32 MFMA accumulators of P.V
  const i64 Spad = ((i64)S + 15) & ~15;
  const i64 lds = (i64)G * Spad * 4;
  size_t dyn = 0;
  if (lds <= DECODE_LDS_BYTES) {
    dyn = (size_t)lds;
    scratch = nullptr;
  } else if (!scratch) {
    return DI_ERANGE;
  }
  DecodeArgs a{q8, tpos, KVPages{(int8_t*)kpool, (int8_t*)vpool, table, width, n_kv}, valid, out,
               scratch, s_dev, S, n_q, n_kv, valid_stride, err};
  const dim3 grid(n_kv, B);
  switch (G) {
#define DI_DEC_LAUNCH(G_)                                                                      \
  if (scratch) hipLaunchKernelGGL((k_attn_decode<G_, true>), grid, dim3(256), dyn, s, a);    \
  else hipLaunchKernelGGL((k_attn_decode<G_, false>), grid, dim3(256), dyn, s, a)
    case 1: DI_DEC_LAUNCH(1); break;
    case 2: DI_DEC_LAUNCH(2); break;
    case 4: DI_DEC_LAUNCH(4); break;
    case 8: DI_DEC_LAUNCH(8); break;
#undef DI_DEC_LAUNCH
    default: return DI_ENOSYS;
  }
  DI_LAUNCH_CHECK();
  return DI_OK;
}

// Fused decode step for one query token per row: the Q/K/V epilogue of
// detllm_qkv_epilogue (T = 1) followed by detllm_attn_decode, one launch.
static int qkv_attn_decode_launch(const int32_t* P, int nsplit, int64_t split_stride, int B, int n_q,
                           int n_kv, const int64_t* xm, const int64_t* xk,
                           const int64_t* positions, const int64_t* q_m, int64_t q_k,
                           const int64_t* k_m, int64_t k_k, const int64_t* v_m, int64_t v_k,
                           const int64_t* q_norm_m, int64_t q_norm_k, const int64_t* k_norm_m,
                           int64_t k_norm_k, const int64_t* qs_m, int64_t qs_k,
                           const int64_t* kq_m, const int64_t* kq_k, const int64_t* ks_m,
                           const int64_t* ks_k, const int64_t* vq_m, const int64_t* vq_k,
                           const int16_t* cos_t, const int16_t* sin_t, int64_t max_pos,
                           int8_t* kpool, int8_t* vpool, const int32_t* table, int width,
                           const int64_t* slot_base_dev, int64_t slot_base,
                           const uint8_t* valid, int64_t valid_stride, int S,
                           const int64_t* s_dev, int32_t* scratch, int64_t* out, int32_t* err,
                           const int64_t* om, int64_t* ext, hipStream_t s) {
  if (B <= 0) return DI_OK;
  if (n_q <= 0 || n_kv <= 0 || n_q % n_kv || nsplit < 1 || S < 1 ||
      !kv_ok(kpool, vpool, table, width) || S > (i64)width * DI_PAGE || valid_stride < S ||
      max_pos <= 0 || !P || !positions || !out || !valid)
    return DI_EINVAL;
  if (S > DEC_MAX_S) return DI_ERANGE;  // int32 MFMA accumulators of P.V
  if (!slot_base_dev && (slot_base < 0 || slot_base + 1 > (i64)width * DI_PAGE)) return DI_ERANGE;
  const int G = n_q / n_kv;
  if (G > 2) return DI_ENOSYS;  // one wave per head slot of the block
  const i64 Spad = ((i64)S + 15) & ~15;
  const i64 lds = (i64)G * Spad * 4;
  size_t dyn = 0;
  if (lds <= DECODE_LDS_BYTES) {
    dyn = (size_t)lds;
    scratch = nullptr;
  } else if (!scratch) {
    return DI_ERANGE;
  }
  const KVPages kv{kpool, vpool, table, width, n_kv};
  QKVArgs qa{};
  qa.T = 1; qa.n_q = n_q; qa.n_kv = n_kv; qa.P = P; qa.nsplit = nsplit;
  qa.split_stride = split_stride; qa.xm = xm; qa.xk = xk; qa.positions = positions;
  qa.q_m = q_m; qa.k_m = k_m; qa.v_m = v_m; qa.q_k = q_k; qa.k_k = k_k; qa.v_k = v_k;
  qa.q_norm_m = q_norm_m; qa.k_norm_m = k_norm_m; qa.q_norm_k = q_norm_k;
  qa.k_norm_k = k_norm_k; qa.qs_m = qs_m; qa.qs_k = qs_k; qa.kq_m = kq_m; qa.kq_k = kq_k;
  qa.ks_m = ks_m; qa.ks_k = ks_k; qa.vq_m = vq_m; qa.vq_k = vq_k; qa.cos_t = cos_t;
  qa.sin_t = sin_t; qa.max_pos = max_pos; qa.q8 = nullptr; qa.tpos = nullptr; qa.dbg = nullptr;
  qa.kv = kv; qa.slot_base_dev = slot_base_dev; qa.slot_base = slot_base; qa.err = err;
  if ((om == nullptr) != (ext == nullptr)) return DI_EINVAL;
  DecodeArgs a{nullptr, nullptr, kv, valid, out, scratch, s_dev, S, n_q, n_kv, valid_stride, err,
               om, ext};
  const dim3 grid(n_kv, B);
#define DI_QAD_LAUNCH(G_, NS1_)                                                                 \
  if (scratch) hipLaunchKernelGGL((k_qkv_attn_decode<G_, NS1_, true>), grid, dim3(QAD_WAVES * 64), dyn, s, a, qa); \
  else hipLaunchKernelGGL((k_qkv_attn_decode<G_, NS1_, false>), grid, dim3(QAD_WAVES * 64), dyn, s, a, qa)
  if (G == 1) {
    if (nsplit == 1) { DI_QAD_LAUNCH(1, true); }
    else { DI_QAD_LAUNCH(1, false); }
  } else {
    if (nsplit == 1) { DI_QAD_LAUNCH(2, true); }
    else { DI_QAD_LAUNCH(2, false); }
  }
#undef DI_QAD_LAUNCH
  DI_LAUNCH_CHECK();
  return DI_OK;
}

int detllm_qkv_attn_decode(const int32_t* P, int nsplit, int64_t split_stride, int B, int n_q,
                           int n_kv, const int64_t* xm, const int64_t* xk,
                           const int64_t* positions, const int64_t* q_m, int64_t q_k,
                           const int64_t* k_m, int64_t k_k, const int64_t* v_m, int64_t v_k,
                           const int64_t* q_norm_m, int64_t q_norm_k, const int64_t* k_norm_m,
                           int64_t k_norm_k, const int64_t* qs_m, int64_t qs_k,
                           const int64_t* kq_m, const int64_t* kq_k, const int64_t* ks_m,
                           const int64_t* ks_k, const int64_t* vq_m, const int64_t* vq_k,
                           const int16_t* cos_t, const int16_t* sin_t, int64_t max_pos,
                           int8_t* kpool, int8_t* vpool, const int32_t* table, int width,
                           const int64_t* slot_base_dev, int64_t slot_base,
                           const uint8_t* valid, int64_t valid_stride, int S,
                           const int64_t* s_dev, int32_t* scratch, int64_t* out, int32_t* err,
                           hipStream_t s) {
  return qkv_attn_decode_launch(
      P, nsplit, split_stride, B, n_q, n_kv, xm, xk, positions, q_m, q_k, k_m, k_k, v_m, v_k,
      q_norm_m, q_norm_k, k_norm_m, k_norm_k, qs_m, qs_k, kq_m, kq_k, ks_m, ks_k, vq_m, vq_k,
      cos_t, sin_t, max_pos, kpool, vpool, table, width, slot_base_dev, slot_base, valid,
      valid_stride, S, s_dev, scratch, out, err, nullptr, nullptr, s);
}

int detllm_qkv_attn_decode_ext(const int32_t* P, int nsplit, int64_t split_stride, int B, int n_q,
                           int n_kv, const int64_t* xm, const int64_t* xk,
                           const int64_t* positions, const int64_t* q_m, int64_t q_k,
                           const int64_t* k_m, int64_t k_k, const int64_t* v_m, int64_t v_k,
                           const int64_t* q_norm_m, int64_t q_norm_k, const int64_t* k_norm_m,
                           int64_t k_norm_k, const int64_t* qs_m, int64_t qs_k,
                           const int64_t* kq_m, const int64_t* kq_k, const int64_t* ks_m,
                           const int64_t* ks_k, const int64_t* vq_m, const int64_t* vq_k,
                           const int16_t* cos_t, const int16_t* sin_t, int64_t max_pos,
                           int8_t* kpool, int8_t* vpool, const int32_t* table, int width,
                           const int64_t* slot_base_dev, int64_t slot_base,
                           const uint8_t* valid, int64_t valid_stride, int S,
                           const int64_t* s_dev, int32_t* scratch, int64_t* out, int32_t* err,
                               const int64_t* om, int64_t* ext, hipStream_t s) {
  if (!om || !ext) return DI_EINVAL;
  return qkv_attn_decode_launch(
      P, nsplit, split_stride, B, n_q, n_kv, xm, xk, positions, q_m, q_k, k_m, k_k, v_m, v_k,
      q_norm_m, q_norm_k, k_norm_m, k_norm_k, qs_m, qs_k, kq_m, kq_k, ks_m, ks_k, vq_m, vq_k,
      cos_t, sin_t, max_pos, kpool, vpool, table, width, slot_base_dev, slot_base, valid,
      valid_stride, S, s_dev, scratch, out, err, om, ext, s);
}

// Chunking of the split-S decode attention, in multiples of the page, within
// the LDS of the packed p (G * chunk * 4 bytes <= 48 KiB) and SPLIT_MAX_CHUNK.
//
// Below 256 (row, kv head) pairs: chunks of 256 to 1024 slots, cut until the
// launch has about 256 blocks (one per CU: a CU draws no more than about 32
// bytes per ns, so fewer leave bandwidth unused, and every chunk block sums
// the whole row's denominator, so more cost more); for that reason no more
// than 16 chunks per row either, where the limits above allow it. us per call,
// 16 / 8 heads, at 256 / 512 / 1024 / 2048 slots per chunk: 1 x 4000 16.1 /
// 17.7 / 22.3 / 32.2, 8 x 4000 29.1 / 25.9 / 25.7 / 35.0, 2 x 16384 48.9 /
// 36.8 / 33.8 / 42.1.
//
// From 256 pairs on the pairs fill the chip by themselves, and scores and
// partials through HBM only cost: where one chunk holds the row (4096 slots at
// 1 or 2 query heads per kv head) the one-block kernel takes it, and longer
// rows are cut evenly, into as few chunks as the limits allow from 512 pairs
// on, below at 2048 slots (two chunks of 4096 leave a chip of 256 to 511 blocks
// half idle when the second is short). us per decode step of 4 layers, 16 / 8
// heads, one block / chunks of 1024 / 2048 / 4096: 32 x 4000 460 / 509 / 518 /
// -, 64 x 4000 672 / 788 / 754 / -, 128 x 4000 1135 / 1305 / 1267 / -; in a
// launch sized for 8192 slots 32 x 4200 569 / 547 / 539 / 572, 32 x 8100 855 /
// 783 / 726 / 741, 48 x 5000 888 / 784 / 750 / 797, 64 x 4200 851 / 840 / 813 /
// 811, 64 x 8100 1376 / 1287 / 1207 / 1176, 128 x 8100 2549 / 2302 / 2188 / 2140
// (24 rows, 192 pairs: 4000 431 / 457 / 493 / -, 8100 819 / 666 / 625 / 692). us
// per call, 32 / 8 heads, one block / 1024 / 2048: 64 x 4096 160 / 148 / 135,
// 128 x 4096 336 / 279 / 263; at 2048 slots one block against two chunks 37 / 39
// (32 rows), 47 / 63 (64), 100 / 135 (128).
int detllm_attn_split_plan(int B, int S, int n_q, int n_kv, int* chunk, int* nsplit) {
  if (!chunk || !nsplit || B <= 0 || S <= 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv) return DI_EINVAL;
  const int G = n_q / n_kv;
  if (G > MAXG) return DI_ENOSYS;
  const i64 cmax = imin(DECODE_LDS_BYTES / (4 * G) / DI_PAGE * DI_PAGE, SPLIT_MAX_CHUNK);
  const i64 blocks = (i64)B * n_kv;
  i64 ch;
  if (blocks >= 256) {
    const i64 longest = S <= cmax || blocks >= 512 ? cmax : imin(cmax, 2048);
    const i64 ns = ((i64)S + longest - 1) / longest;
    ch = ((i64)S + ns - 1) / ns;
  } else {
    const i64 want = (256 + blocks - 1) / blocks;
    ch = imin(((i64)S + want - 1) / want, 1024);
    ch = imax(ch, ((i64)S + 15) / 16);
  }
  ch = (ch + DI_PAGE - 1) / DI_PAGE * DI_PAGE;
  ch = imax(imin(ch, cmax), (i64)2 * DI_PAGE);
  *chunk = (int)ch;
  *nsplit = (int)(((i64)S + ch - 1) / ch);
  return DI_OK;
}

// Split-S decode attention (one query token per row; q8, tpos as written by
// detllm_qkv_epilogue with T = 1). scores: int32 [B][n_q][nsplit * chunk];
// cmax: int32 [B][n_q][nsplit]; out: int64 partial contexts
// [nsplit][B][n_q * 128] whose sum is detllm_attn_decode's out.
static int attn_split_launch(const int8_t* q8, const int64_t* tpos, const int8_t* kpool,
                             const int8_t* vpool, const int32_t* table, int width,
                             const uint8_t* valid, int64_t valid_stride, int B, int S, int n_q,
                             int n_kv, const int64_t* s_dev, int chunk, int32_t* scores,
                             int32_t* cmax, int64_t* out, bool add, int32_t* err, hipStream_t s) {
  if (B <= 0) return DI_OK;
  if (n_q <= 0 || n_kv <= 0 || n_q % n_kv || S < 1 || !kv_ok(kpool, vpool, table, width) ||
      S > (i64)width * DI_PAGE || valid_stride < S || !q8 || !tpos || !valid || !out || !scores ||
      !cmax || chunk < DI_PAGE || chunk % DI_PAGE || chunk > SPLIT_MAX_CHUNK)
    return DI_EINVAL;
  const int G = n_q / n_kv;
  if (G > MAXG) return DI_ENOSYS;
  if (S > DEC_MAX_S) return DI_ERANGE;  // int32 MFMA accumulators of P.V
  const i64 dyn = (i64)G * chunk * 4;
  if (dyn > DECODE_LDS_BYTES) return DI_ERANGE;
  const int ns = (S + chunk - 1) / chunk;
  SplitArgs sa{};
  sa.d = DecodeArgs{q8, tpos, KVPages{(int8_t*)kpool, (int8_t*)vpool, table, width, n_kv}, valid,
                    out, scores, s_dev, S, n_q, n_kv, valid_stride, err};
  sa.cmax = cmax;
  sa.chunk = chunk;
  sa.ns = ns;
  sa.spad = (i64)ns * chunk;
  sa.out_stride = (i64)B * n_q * 128;
  sa.add = add;
  const dim3 grid(n_kv, B, ns);
#define DI_SPLIT_LAUNCH(G_)                                                                   \
  hipLaunchKernelGGL(k_attn_split_scores<G_>, grid, dim3(256), 0, s, sa);                     \
  hipLaunchKernelGGL(k_attn_split_pv<G_>, grid, dim3(256), (size_t)dyn, s, sa)
  switch (G) {
    case 1: DI_SPLIT_LAUNCH(1); break;
    case 2: DI_SPLIT_LAUNCH(2); break;
    case 4: DI_SPLIT_LAUNCH(4); break;
    case 8: DI_SPLIT_LAUNCH(8); break;
    default: return DI_ENOSYS;
  }
#undef DI_SPLIT_LAUNCH
  DI_LAUNCH_CHECK();
  return DI_OK;
}

int detllm_attn_decode_split(const int8_t* q8, const int64_t* tpos, const int8_t* kpool,
                             const int8_t* vpool, const int32_t* table, int width,
                             const uint8_t* valid, int64_t valid_stride, int B, int S, int n_q,
                             int n_kv, const int64_t* s_dev, int chunk, int32_t* scores,
                             int32_t* cmax, int64_t* out, int32_t* err, hipStream_t s) {
  return attn_split_launch(q8, tpos, kpool, vpool, table, width, valid, valid_stride, B, S, n_q,
                           n_kv, s_dev, chunk, scores, cmax, out, false, err, s);
}

// detllm_attn_decode_split with the partials added up: out [B][n_q * 128] as
// detllm_attn_decode writes it.
int detllm_attn_decode_split_sum(const int8_t* q8, const int64_t* tpos, const int8_t* kpool,
                                 const int8_t* vpool, const int32_t* table, int width,
                                 const uint8_t* valid, int64_t valid_stride, int B, int S,
                                 int n_q, int n_kv, const int64_t* s_dev, int chunk,
                                 int32_t* scores, int32_t* cmax, int64_t* out, int32_t* err,
                                 hipStream_t s) {
  return attn_split_launch(q8, tpos, kpool, vpool, table, width, valid, valid_stride, B, S, n_q,
                           n_kv, s_dev, chunk, scores, cmax, out, true, err, s);
}

}  // extern "C"
