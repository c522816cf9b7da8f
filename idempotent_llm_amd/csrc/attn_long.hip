// Attention forms for long caches (gfx950): windowed attention with sinks and
// attention that accumulates each slot's weight. No counterpart in the
// reference; the integers of a query are those of attention.hip's kernels over
// the slots it sees.
//
// Windowed (attn_window.h has the rule): the kernels are attention.hip's over
// a shorter list of pages, those of the sinks and those from the window's
// first slot on that hold a valid slot, so their work follows the window and not
// the cache. The list is made on the device, per query tile in prefill and per
// row in decode, because it depends on the row's validity flags: a launch is
// sized for rows without gaps, and a row whose window spans more pages takes
// more steps in the same blocks (scores past its LDS go to the scratch).
//
// Accumulating: the p of a slot, summed over the query heads of a kv head (and
// over a tile's queries), is added to acc [B][n_kv][slots]. p is an integer, so
// the order of the additions does not change the sum. A decode block owns its
// (row, kv head, slots) and adds without atomics; prefill tiles share slots
// and add with 64-bit atomics.

#include "attn_plan.h"
#include "attn_prefill.h"

namespace {

// Bound by issue, as k_attn_prefill: about 28 VALU instructions per pair of a
// query and a slot it may see (DI-Exp twice, p, packing) beside 42 MFMAs and as
// many LDS operand reads per 16 x 64 tile, in phases that overlap only in part.
// 64 queries, a window of 1024 and 4 sinks walk about 1340 slots, 1.3 times what
// they see (pages and 64-query tiles are whole). 2048 queries behind 6144 slots,
// 32 heads, window 1024: 129 us, 67 M pairs seen, 267 TOP/s; 3 x 333 queries,
// window 100: 24 us, most of it the chain of three passes over three pages.
__global__ __launch_bounds__(256, 2) void k_window_prefill(PrefillArgs a, PrefillForm form) {
  keep_hidden_args();
  prefill_body<true, false>(a, form);
}
// k_attn_prefill, and per 16 x 64 tile the 16 queries' p of each slot summed over
// lanes (45 VALU instructions, row16_scatter_sum) and one 64-bit atomic per slot:
// 2048 queries, 16 heads 74 us against 61.5 without. Sums of a block's four waves
// joined in LDS first, a fourth of the atomics, measured 1.7 us less (2 %) and were
// not kept: they need a barrier per 64-slot half, where the waves now meet once a
// page, and not at all where the pages are resident.
__global__ __launch_bounds__(256, 2) void k_acc_prefill(PrefillArgs a, PrefillForm form) {
  keep_hidden_args();
  prefill_body<false, true>(a, form);
}

__host__ __device__ constexpr int pages_of(int S) { return (S + DI_PAGE - 1) / DI_PAGE; }

// The listed pages of a row's newest query (window_pages), numbered 0, 1, ...
struct WinView {
  static constexpr bool kWhole = false;
  const uint16_t* list;
  int n;  // slots of the list
  int sink_end, lo;
  __device__ __forceinline__ int slot(int s) const {
    return (int)list[s >> 7] * DI_PAGE + (s & (DI_PAGE - 1));
  }
  __device__ __forceinline__ int page(const KVPages& kv, int b, int s) const {
    return kv.page(b, slot(s));
  }
  __device__ __forceinline__ bool sees(int s) const { return s < sink_end || s >= lo; }
};
__device__ __forceinline__ WinView win_view(const WinRange& r, const uint16_t* list, int S) {
  int n = r.pages * DI_PAGE;
  if (r.pages > 0) n -= ::max(((int)list[r.pages - 1] + 1) * DI_PAGE - S, 0);
  return WinView{list, n, r.sink_end, r.lo};
}

constexpr int NW = 8;  // waves of the one-block kernels (4: 32 rows, window 2048 behind
                       // padding 49 us against 40, 32 x 4000 slots 73 against 57)

struct WindowArgs {
  SplitArgs s;
  int window, sinks;
  int zs;          // blocks per (row, kv head)
  int lds_slots;   // one block: slots whose scores its LDS holds
  WinRange* range; // [B], and the lists [B][pages] (split form: made by the
  uint16_t* lists; // scores launch for the second)
  int pages;
};

// One block per (row, kv head). Scores in LDS; a row whose window spans more
// slots than that holds keeps them in the scratch. Bound by HBM with many rows
// (32 x 8000 slots, window 2048: 39 us for 134 MB seen, about 150 MB in whole
// pages), by the chain flags - list - K - maximum - denominator - p - V with few
// (one row of 320: 10 us).
template <int G>
__global__ __launch_bounds__(64 * NW) void k_window_decode(WindowArgs w) {
  keep_hidden_args();
  extern __shared__ __attribute__((aligned(16))) int32_t sh_scores[];
  __shared__ int32_t pg_lds[DEC_MAX_PAGES];
  __shared__ uint16_t list[DEC_MAX_PAGES];
  DecodeArgs a = w.s.d;
  const int kvh = blockIdx.x, b = blockIdx.y;
  const i64 q0 = (i64)b * a.n_q + kvh * G;
  bool over;
  const int S = scanned_slots(a, a.tpos, &over);
  // the row's page ids load beside the flags
  __shared__ int32_t row_pages[DEC_MAX_PAGES];
  for (int i = threadIdx.x; i < pages_of(a.S); i += 64 * NW)
    row_pages[i] = a.kv.page(b, (i64)i * DI_PAGE);
  const WinView v = win_view(
      window_pages<64 * NW>(a.valid + (i64)b * a.valid_stride, S, S, w.window, w.sinks, list), list, S);
  const int npages = pages_of(v.n);
  for (int i = threadIdx.x; i < npages; i += 64 * NW) pg_lds[i] = row_pages[list[i]];
  if (npages == 0 && threadIdx.x == 0) pg_lds[0] = -1;  // S = 0: loads read page 0
  __syncthreads();
  if (v.n <= w.lds_slots) {
    a.S = v.n;  // (the scores' row stride)
    decode_body<G, VPRE, false, false, NW, false, WinView>(
        a, v.n, kvh, b, a.q8 + q0 * 128, a.tpos + q0, sh_scores, pg_lds, KPre<8 / NW>{},
        OmPre<G, 8 / NW>{}, v);
  } else {
    decode_body<G, VPRE, true, false, NW, false, WinView>(
        a, v.n, kvh, b, a.q8 + q0 * 128, a.tpos + q0, sh_scores, pg_lds, KPre<8 / NW>{},
        OmPre<G, 8 / NW>{}, v);
  }
  report_slots(a, over, kvh == 0);
}

template <int G>
__global__ __launch_bounds__(256) void k_window_scores(WindowArgs w) {
  keep_hidden_args();
  const DecodeArgs& a = w.s.d;
  const int kvh = blockIdx.x, b = blockIdx.y, z = blockIdx.z;
  bool over;
  const int S = scanned_slots(a, a.tpos, &over);
  __shared__ uint16_t list[DEC_MAX_PAGES];
  const WinRange r =
      window_pages<256>(a.valid + (i64)b * a.valid_stride, S, S, w.window, w.sinks, list);
  if (kvh == 0 && z == 0) {
    if (threadIdx.x == 0) w.range[b] = r;
    for (int i = threadIdx.x; i < r.pages; i += 256) w.lists[(i64)b * w.pages + i] = list[i];
  }
  const WinView v = win_view(r, list, S);
  int c = z;
  do {
    split_scores_chunk<G, WinView>(w.s, kvh, b, c, v);
    __syncthreads();  // (the chunk's LDS is reused)
    c += w.zs;
  } while (c * w.s.chunk < v.n);
  report_slots(a, over, kvh == 0 && z == 0);
}

template <int G>
__global__ __launch_bounds__(256) void k_window_pv(WindowArgs w) {
  keep_hidden_args();
  const DecodeArgs& a = w.s.d;
  const int kvh = blockIdx.x, b = blockIdx.y;
  bool over;
  const int S = scanned_slots(a, a.tpos, &over);
  const WinView v = win_view(w.range[b], w.lists + (i64)b * w.pages, S);
  int c = blockIdx.z;
  do {
    split_pv_chunk<G, WinView>(w.s, kvh, b, c, v);
    __syncthreads();
    c += w.zs;
  } while (c * w.s.chunk < v.n);
}

// One block per (row, kv head), as k_window_decode: 32 x 4000 slots 57 us, 4.9 TB/s.
template <int G>
__global__ __launch_bounds__(64 * NW) void k_acc_decode(DecodeArgs a, AccInto into) {
  keep_hidden_args();
  extern __shared__ __attribute__((aligned(16))) int32_t sh_scores[];
  __shared__ int32_t pg_lds[DEC_MAX_PAGES];
  const int kvh = blockIdx.x, b = blockIdx.y;
  const i64 q0 = (i64)b * a.n_q + kvh * G;
  bool over;
  const int S = scanned_slots(a, a.tpos, &over);
  const int npages = (a.S + DI_PAGE - 1) / DI_PAGE;
  for (int i = threadIdx.x; i < npages; i += 64 * NW) pg_lds[i] = a.kv.page(b, (i64)i * DI_PAGE);
  if (npages == 0 && threadIdx.x == 0) pg_lds[0] = -1;
  __syncthreads();
  decode_body<G, VPRE, false, false, NW, false, WholeRow, true>(
      a, S, kvh, b, a.q8 + q0 * 128, a.tpos + q0, sh_scores, pg_lds, KPre<8 / NW>{},
      OmPre<G, 8 / NW>{}, WholeRow{}, into);
  report_slots(a, over, kvh == 0);
}

template <int G>
__global__ __launch_bounds__(256) void k_acc_scores(SplitArgs sa) {
  keep_hidden_args();
  split_scores_chunk<G>(sa, blockIdx.x, blockIdx.y, blockIdx.z);
}
template <int G>
__global__ __launch_bounds__(256) void k_acc_pv(SplitArgs sa, AccInto into) {
  keep_hidden_args();
  split_pv_chunk<G, WholeRow, true>(sa, blockIdx.x, blockIdx.y, blockIdx.z, WholeRow{}, into);
}

// Bytes of the one block's scores where a row may need more than its LDS
i64 one_block_bytes(int B, int S, int n_q, int G) {
  const i64 spad = ((i64)S + 15) / 16 * 16;
  return (i64)G * spad * 4 > DECODE_LDS_BYTES ? (i64)B * n_q * spad * 4 : 0;
}
// Slots that a launch is sized for: what a query sees, and the rest of the
// pages at the ends of the two ranges and around two stretches of padding.
int window_slots(int S, int window, int sinks) {
  return (int)imin(S, (i64)window + sinks + 6 * DI_PAGE);
}
}  // namespace

extern "C" {

int detllm_attn_window_prefill(const int8_t* q8, const int64_t* tpos, const int8_t* kpool,
                               const int8_t* vpool, const int32_t* table, int width,
                               const uint8_t* valid, int64_t valid_stride, int B, int T,
                               int S_past, int n_q, int n_kv, int window, int sinks, int64_t* out,
                               hipStream_t s) {
  if (window < 1 || sinks < 0) return DI_EINVAL;
  if (B <= 0 || T <= 0) return DI_OK;
  const i64 S = (i64)S_past + T;
  if (n_q <= 0 || n_kv <= 0 || n_q % n_kv || S_past < 0 || !kv_ok(kpool, vpool, table, width) ||
      S > (i64)width * DI_PAGE || valid_stride < S || !q8 || !tpos || !valid || !out)
    return DI_EINVAL;
  if (S > DEC_MAX_S) return DI_ERANGE;  // int32 MFMA accumulators of P.V
  PrefillArgs a{q8, tpos, KVPages{(int8_t*)kpool, (int8_t*)vpool, table, width, n_kv}, valid, out,
                T, (int)S, S_past, n_q, n_kv, B, valid_stride};
  const i64 pairs = (i64)(((T + 63) / 64 + 1) / 2) * n_q * B;
  if (2 * pairs > 0x7fffffff) return DI_ERANGE;
  hipLaunchKernelGGL(k_window_prefill, dim3((unsigned)(2 * pairs)), dim3(256),
                     prefill_lds(S, true), s, a, PrefillForm{window, sinks, nullptr, 0});
  DI_LAUNCH_CHECK();
  return DI_OK;
}

int detllm_attn_prefill_acc(const int8_t* q8, const int64_t* tpos, const int8_t* kpool,
                            const int8_t* vpool, const int32_t* table, int width,
                            const uint8_t* valid, int64_t valid_stride, int B, int T, int S_past,
                            int n_q, int n_kv, int64_t* acc, int64_t acc_stride, int64_t* out,
                            hipStream_t s) {
  if (B <= 0 || T <= 0) return DI_OK;
  const i64 S = (i64)S_past + T;
  if (n_q <= 0 || n_kv <= 0 || n_q % n_kv || S_past < 0 || !kv_ok(kpool, vpool, table, width) ||
      S > (i64)width * DI_PAGE || valid_stride < S || acc_stride < S || !q8 || !tpos || !valid ||
      !acc || !out)
    return DI_EINVAL;
  if (S > DEC_MAX_S) return DI_ERANGE;
  PrefillArgs a{q8, tpos, KVPages{(int8_t*)kpool, (int8_t*)vpool, table, width, n_kv}, valid, out,
                T, (int)S, S_past, n_q, n_kv, B, valid_stride};
  const i64 pairs = (i64)(((T + 63) / 64 + 1) / 2) * n_q * B;
  if (2 * pairs > 0x7fffffff) return DI_ERANGE;
  hipLaunchKernelGGL(k_acc_prefill, dim3((unsigned)(2 * pairs)), dim3(256), prefill_lds(S), s, a,
                     PrefillForm{0, 0, acc, acc_stride});
  DI_LAUNCH_CHECK();
  return DI_OK;
}

int detllm_attn_window_decode_work(int B, int S, int n_q, int n_kv, int window, int sinks,
                                   int64_t* bytes) {
  if (!bytes || B < 0 || S < 0 || window < 1 || sinks < 0) return DI_EINVAL;
  if (const int rc = heads_ok(n_q, n_kv)) return rc;
  if (S > DEC_MAX_S) return DI_ERANGE;
  *bytes = 0;
  if (B == 0 || S == 0) return DI_OK;
  const int chunk = decode_chunk(B, window_slots(S, window, sinks), n_q, n_kv);
  i64 at;
  *bytes = chunk ? split_bytes(B, S, n_q, chunk, &at) + (i64)B * (sizeof(WinRange) + 2 * pages_of(S))
                 : one_block_bytes(B, S, n_q, n_q / n_kv);
  return DI_OK;
}

int detllm_attn_window_decode(const int8_t* q8, const int64_t* tpos, const int8_t* kpool,
                              const int8_t* vpool, const int32_t* table, int width,
                              const uint8_t* valid, int64_t valid_stride, int B, int S, int n_q,
                              int n_kv, const int64_t* s_dev, int window, int sinks, void* work,
                              int64_t work_bytes, int64_t* out, int32_t* err, hipStream_t s) {
  i64 need = 0;
  if (const int rc = detllm_attn_window_decode_work(B < 0 ? 0 : B, S, n_q, n_kv, window, sinks, &need))
    return rc;
  if (B <= 0) return DI_OK;
  if (!kv_ok(kpool, vpool, table, width) || S > (i64)width * DI_PAGE || valid_stride < S || !q8 ||
      !tpos || !valid || !out)
    return DI_EINVAL;
  if (need > 0 && (!work || work_bytes < need)) return DI_ERANGE;
  const int G = n_q / n_kv, slots = window_slots(S, window, sinks);
  const int chunk = S > 0 ? decode_chunk(B, slots, n_q, n_kv) : 0;
  WindowArgs w{};
  const DecodeArgs d{q8, tpos, KVPages{(int8_t*)kpool, (int8_t*)vpool, table, width, n_kv}, valid,
                     out, (int32_t*)work, s_dev, S, n_q, n_kv, valid_stride, err};
  w.window = window;
  w.sinks = sinks;
  if (chunk) {
    w.s = split_args(d, B, chunk, work);
    i64 at;
    w.range = (WinRange*)((char*)work + split_bytes(B, S, n_q, chunk, &at));
    w.lists = (uint16_t*)(w.range + B);
    w.pages = pages_of(S);
    w.zs = (slots + chunk - 1) / chunk;
    const dim3 grid(n_kv, B, w.zs);
    const size_t dyn = (size_t)G * chunk * 4;
    switch (G) {
#define DI_WIN_SPLIT(G_)                                                     \
  case G_:                                                                   \
    hipLaunchKernelGGL(k_window_scores<G_>, grid, dim3(256), 0, s, w);       \
    hipLaunchKernelGGL(k_window_pv<G_>, grid, dim3(256), dyn, s, w);         \
    break
      DI_WIN_SPLIT(1);
      DI_WIN_SPLIT(2);
      DI_WIN_SPLIT(4);
      DI_WIN_SPLIT(8);
#undef DI_WIN_SPLIT
    }
  } else {
    w.s.d = d;
    const i64 fit = DECODE_LDS_BYTES / (4 * G) / 16 * 16;
    w.lds_slots = (int)imin(((i64)slots + 15) / 16 * 16, fit);
    if (one_block_bytes(B, S, n_q, G) == 0) w.lds_slots = (S + 15) / 16 * 16;  // no scratch
    const dim3 grid(n_kv, B);
    const size_t dyn = (size_t)G * w.lds_slots * 4;
    switch (G) {
      case 1: hipLaunchKernelGGL(k_window_decode<1>, grid, dim3(64 * NW), dyn, s, w); break;
      case 2: hipLaunchKernelGGL(k_window_decode<2>, grid, dim3(64 * NW), dyn, s, w); break;
      case 4: hipLaunchKernelGGL(k_window_decode<4>, grid, dim3(64 * NW), dyn, s, w); break;
      case 8: hipLaunchKernelGGL(k_window_decode<8>, grid, dim3(64 * NW), dyn, s, w); break;
    }
  }
  DI_LAUNCH_CHECK();
  return DI_OK;
}

int detllm_attn_decode_acc_work(int B, int S, int n_q, int n_kv, int64_t* bytes) {
  if (!bytes || B < 0 || S < 0) return DI_EINVAL;
  if (const int rc = heads_ok(n_q, n_kv)) return rc;
  if (S > DEC_MAX_S) return DI_ERANGE;
  *bytes = 0;
  if (B == 0 || S == 0) return DI_OK;
  const int chunk = decode_chunk(B, S, n_q, n_kv);
  i64 at;
  if (chunk) *bytes = split_bytes(B, S, n_q, chunk, &at);
  return DI_OK;
}

int detllm_attn_decode_acc(const int8_t* q8, const int64_t* tpos, const int8_t* kpool,
                           const int8_t* vpool, const int32_t* table, int width,
                           const uint8_t* valid, int64_t valid_stride, int B, int S, int n_q,
                           int n_kv, const int64_t* s_dev, int64_t* acc, int64_t acc_stride,
                           void* work, int64_t work_bytes, int64_t* out, int32_t* err,
                           hipStream_t s) {
  i64 need = 0;
  if (const int rc = detllm_attn_decode_acc_work(B < 0 ? 0 : B, S, n_q, n_kv, &need)) return rc;
  if (B <= 0) return DI_OK;
  if (!kv_ok(kpool, vpool, table, width) || S > (i64)width * DI_PAGE || valid_stride < S ||
      acc_stride < S || !q8 || !tpos || !valid || !acc || !out)
    return DI_EINVAL;
  if (need > 0 && (!work || work_bytes < need)) return DI_ERANGE;
  const int G = n_q / n_kv;
  const int chunk = S > 0 ? decode_chunk(B, S, n_q, n_kv) : 0;
  const DecodeArgs d{q8, tpos, KVPages{(int8_t*)kpool, (int8_t*)vpool, table, width, n_kv}, valid,
                     out, nullptr, s_dev, S, n_q, n_kv, valid_stride, err};
  const AccInto into{acc, acc_stride};
  if (chunk) {
    const SplitArgs sa = split_args(d, B, chunk, work);
    const dim3 grid(n_kv, B, sa.ns);
    const size_t dyn = (size_t)G * chunk * 4;
    switch (G) {
#define DI_ACC_SPLIT(G_)                                                  \
  case G_:                                                                \
    hipLaunchKernelGGL(k_acc_scores<G_>, grid, dim3(256), 0, s, sa);      \
    hipLaunchKernelGGL(k_acc_pv<G_>, grid, dim3(256), dyn, s, sa, into);  \
    break
      DI_ACC_SPLIT(1);
      DI_ACC_SPLIT(2);
      DI_ACC_SPLIT(4);
      DI_ACC_SPLIT(8);
#undef DI_ACC_SPLIT
    }
  } else {
    const dim3 grid(n_kv, B);
    const size_t dyn = (size_t)G * (((i64)S + 15) / 16 * 16) * 4;
    switch (G) {
      case 1: hipLaunchKernelGGL(k_acc_decode<1>, grid, dim3(64 * NW), dyn, s, d, into); break;
      case 2: hipLaunchKernelGGL(k_acc_decode<2>, grid, dim3(64 * NW), dyn, s, d, into); break;
      case 4: hipLaunchKernelGGL(k_acc_decode<4>, grid, dim3(64 * NW), dyn, s, d, into); break;
      case 8: hipLaunchKernelGGL(k_acc_decode<8>, grid, dim3(64 * NW), dyn, s, d, into); break;
    }
  }
  DI_LAUNCH_CHECK();
  return DI_OK;
}

}  // extern "C"
