// Attention of packed rows over the paged cache (gfx950): each row has its own
// number of new tokens (none, one, a draft, a prompt's chunk), their token rows
// follow each other, and token t of a row at `past` slots sees the row's slots up
// to past + t. The integers of a query are those of the prefill attention.
//
// The rows' lengths are on the device, so a block finds its work itself: the
// launch is sized by bounds (token rows, rows, slots), a block's unit is a row of
// at most 16 query rows (tokens x query heads of a kv head) or 64 query rows of a
// longer one, and every wave finds it by a scan of the rows' lengths, one round
// trip, with no launch before it and nothing read on the host.
//
// DI-Exp is not multiplicative: the row maximum comes before the first
// exponential, the whole denominator before the first probability. One launch
// makes all three passes (k_packed_few, k_packed_one: short rows, or enough units to
// fill the chip); else each pass is a launch over chunks of the slots (k_packed_phase),
// whose maxima, denominators and int32 contexts meet in scratch.
#include "attn_packed.h"

#include "../../include/detllm_hip.h"

namespace {

// Rows of at most 16 query rows alone, all slots in registers: NW waves, NT
// 64-slot tiles each.
template <int NT, bool R8>
__global__ __launch_bounds__(512, 2) void k_packed_few(PackedArgs a) {
  keep_hidden_args();
  __shared__ FewLds<8> lds;
  Rows rows;
  const Finder f(a, rows);
  const int kvh = blockIdx.x % a.n_kv, j = blockIdx.x / a.n_kv;
  if (j < f.total) {
    const Work w = f.find(a, rows, kvh, j);
    report_row(a, w);
    few_one<8, NT, R8>(a, w, lds);
  }
  if (threadIdx.x < 256) zero_tail(a, f.ntok, kvh, j);
}

// All three passes of any rows
__global__ __launch_bounds__(256, 3) void k_packed_one(PackedArgs a) {
  keep_hidden_args();
  __shared__ TileLds lds;
  Rows rows;
  const Finder f(a, rows);
  const int kvh = blockIdx.x % a.n_kv, j = blockIdx.x / a.n_kv;
  if (j < f.total) {
    const Work w = f.find(a, rows, kvh, j);
    report_row(a, w);
    if (w.few && w.len <= FEW_ONE_SLOTS) few_one<4, FEW_ONE_SLOTS / 256, false>(a, w, lds.few);
    else tile_body<PH_ALL>(a, w, lds);
  }
  if (threadIdx.x < 256) zero_tail(a, f.ntok, kvh, j);
}

// One pass over chunks. FEW: the launch's rows have at most FEW (8 or 16) query rows
template <int PH, int FEW>
__global__ __launch_bounds__(256, FEW == 0 || PH == PH_PV ? 3 : 4) void k_packed_phase(PackedArgs a) {
  keep_hidden_args();
  Rows rows;
  const Finder f(a, rows);
  const int kvh = blockIdx.x % a.n_kv, j0 = blockIdx.x / a.n_kv;
  for (int j = j0; j < f.total; j += a.step) {
    if (j != j0) {
      rows.load(a, 0);  // (again, or its registers are held all along)
      __syncthreads();  // the item before is done with LDS
    }
    const Work w = f.find(a, rows, kvh, j);
    if (outside(a, w)) continue;
    if (PH == PH_MAX) report_row(a, w);
    if constexpr (FEW != 0) {
      __shared__ FewLds<4> lds;
      few_phase<PH, 4, FEW == 8>(a, w, lds);
    } else {
      __shared__ TileLds lds;
      if (w.few && (w.T << a.lg) <= 8) few_phase<PH, 4, true>(a, w, lds.few);
      else if (w.few) few_phase<PH, 4, false>(a, w, lds.few);
      else tile_body<PH>(a, w, lds);
    }
  }
  if (PH == PH_PV && !a.part) zero_tail(a, f.ntok, kvh, j0);
}

// The chunks' contexts of a token added up (one block per token row)
__global__ __launch_bounds__(256) void k_packed_join(PackedArgs a) {
  keep_hidden_args();
  const int tok = blockIdx.x, cols = a.n_q * 128, lane = threadIdx.x & 63;
  int b = 0;  // rows that end at or before this token
  int last = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int i = b0 + lane;
    const int e = a.cu[i < a.B ? i + 1 : a.B];
    b += __popcll(__ballot(i < a.B && e <= tok));
  }
  int nc = 0;
  if (b < a.B) {
    last = ::max(0, a.cu[b]);
    nc = (row_limit(a, a.past[b], tok - last) + a.chunk) / a.chunk;  // ceil((limit + 1) / chunk)
    if (tok < last || tok - last >= a.max_new) nc = 0;
  }
  for (int i = 4 * threadIdx.x; i < cols; i += 1024) {
    v4i sum = v4i{0, 0, 0, 0};
    const int32_t* p = a.part + (i64)tok * cols + i;
    for (int c = 0; c < nc; c += 4) {
      v4i x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = *(const v4i*)(p + (i64)::min(c + u, nc - 1) * a.N * cols);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c + u < nc) sum += x[u];
    }
    int64_t* o = a.out + (i64)tok * cols + i;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = sum[r];
  }
}

// How a call is cut, from bounds on its sizes
struct Plan {
  bool few;    // every row has at most 16 query rows
  bool one;    // one launch
  int units;   // units that the rows can make
  int step;    // blocks per kv head
  int rows;    // query rows of a few-row unit
  i64 score_rows;  // rows of scores per kv head: B times that, or the token rows'
  int chunk, nch;
  i64 scores_at, max_at, den_at, part_at, bytes;
};

// The figures beside the rules: us a call, one launch / chunks, 16 query heads over 8
// kv heads unless they say otherwise.
inline Plan packed_plan(int N, int B, int S, int max_new, int n_q, int n_kv) {
  Plan p{};
  const int G = n_q / n_kv;
  const i64 most = imin(max_new, N);
  p.few = most * G <= 16;
  const i64 rows = ::min(B, N);
  const i64 units = p.few ? rows : imin((i64)N * G / 64 + rows, N);
  p.units = (int)imax(1, units);
  p.rows = (int)imin(16, most * G);
  p.score_rows = imin((i64)B * p.rows, (i64)N * G);
  const i64 pairs = imax(1, units) * n_kv;
  const i64 tiles = ((i64)N * G + 63) / 64 * n_kv;  // of 64 query rows, were all in one row
  if (p.few) {
    // one-token rows x slots: 1 x 1024 13 / 16, 1 x 1500 18 / 14, 8 x 1500 19 / 19, 16 x
    // 2048 23 / 25, 48 x 1024 25 / 34, 48 x 2048 53 / 61
    p.one = S <= (pairs >= 128 ? FEW_SLOTS : FEW_SLOTS / 2);
  } else {
    // a tile's chain over its slots, against three launches that fill the chip and
    // parts that are written and added up: tokens behind filled slots 700 + 0 24 / 34,
    // 1500 + 0 44 / 55, 64 + 500 20 / 25, 64 + 1000 31 / 26, 512 + 2000 64 / 50, 1024 +
    // 2000 78 / 68, 1200 + 8000 243 / 186, 1600 + 8000 256 / 253, 2048 + 8000 271 / 302, 4 x
    // 512 + 1000 53 / 67. From 420 tiles on whatever S is: 2048 + 16000 496 /
    // 494, + 64000 1862 / 1713, 4 x 512 + 16000 479 / 511, + 64000 1852 / 1878, 32 heads over 8
    // 4 x 256 + 32000 927 / 955. The bounds do not tell whose S it is: one long row beside
    // tiles that are prompts of 100 tokens lasts as long as its own chain (42 of them + a row
    // of 4000 100 / 71, 16000 368 / 208, 131000 2943 / 1968; 16 rows up to 16000 371 / 274). Chunks
    // would take scratch there, 16 words for each row, kv head and slot (64 rows over
    // 131000 slots 4.3 GB): a call that now needs none could run out of memory.
    p.one = S <= FEW_ONE_SLOTS || S * (420 - tiles) <= 300000;
  }
  p.chunk = S;
  if (!p.one) {
    // few-row units: 256, 512 or 1024 slots (whole steps of a block's waves), the most
    // that make 512 blocks (256 / 512 / 768 / 1024: 1 x 4000 14 / 16 / - / 21, 8 x 4000 30 / 25
    // / - / 27, 48 x 4000 146 / 109 / - / 99, 16 rows of 200 to 3000 29 / 24 / 29 / 29, 16 of
    // 100 to 7500 57 / 46 / - / 46). 64 query rows:
    // three tiles a CU at once, or twice that where their chunks would pass 2048 slots, since
    // a tile takes its chunk's time however few are left (512 tokens behind 8000 slots in
    // 7, 6, 5 chunks: 896, 768, 640 items, 110, 86, 102 us; 256 behind 8000 in 13, 11, 9: 68,
    // 56, 65); a short row beside them counts 5 / 8 of a tile (300 tokens beside 60 rows of 0
    // to 2950 in 1, 2, 3, 6 chunks 75, 70, 72, 78). At least 384 slots (128 tokens behind 2000:
    // 384, 512, 1024 28, 31, 42), 512 beside short rows (whole steps of their waves).
    if (p.few) {
      p.chunk = 256;
      while (p.chunk < 1024 && pairs * ((S + 2 * p.chunk - 1) / (2 * p.chunk)) >= 512) p.chunk *= 2;
    } else {
      const i64 load = (imax(1, N - rows) * G + 63) / 64 * n_kv + imax(0, rows - 2) * n_kv * 5 / 8;
      const i64 rounds = S * load > 2048 * 768 ? 2 : 1, least = rows > 2 ? 512 : 384;
      const i64 top = imin((S + least - 1) / least, imax(32, S / 2048));
      const i64 want = imax(1, imin(top, 768 * rounds / load));
      p.chunk = (int)(((S + want - 1) / want + DI_PAGE - 1) / DI_PAGE * DI_PAGE);
    }
  }
  p.chunk = ::max(p.chunk, 1);
  p.nch = ::max(1, (S + p.chunk - 1) / p.chunk);
  p.step = p.units * p.nch;
  // blocks that share the items out (48 rows of 8000 slots: 1024, 2048, 4096 blocks
  // 207, 187, 184 us)
  if (!p.one) p.step = (int)imin(p.step, imax(1, 2048 / n_kv));
  if (p.one) return p;
  auto room = [&](i64 n) {
    const i64 at = p.bytes;
    p.bytes += (n + 15) / 16 * 16;
    return at;
  };
  p.scores_at = room(p.score_rows * n_kv * p.nch * p.chunk * 4);
  const i64 cells = (i64)p.units * n_kv * p.nch * 64;
  p.max_at = room(cells * 4);
  p.den_at = room(cells * 8);
  p.part_at = room(p.nch > 1 && !p.few ? (i64)p.nch * N * n_q * 128 * 4 : 0);
  return p;
}

inline int packed_check(int N, int B, int S, int max_new, int n_q, int n_kv) {
  if (N < 0 || B < 1 || S < 1 || max_new < 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv) return DI_EINVAL;
  const int G = n_q / n_kv;
  if (G != 1 && G != 2 && G != 4 && G != 8) return DI_ENOSYS;
  if (S > PACKED_MAX_S || B > PACKED_MAX_ROWS || (i64)N * n_q > (1 << 24)) return DI_ERANGE;
  return DI_OK;
}

}  // namespace

extern "C" {

int detllm_attn_packed_work(int N, int B, int S, int max_new, int n_q, int n_kv, int64_t* bytes) {
  if (!bytes) return DI_EINVAL;
  const int rc = packed_check(N, B, S, max_new, n_q, n_kv);
  if (rc != DI_OK) return rc;
  *bytes = packed_plan(N, B, S, max_new, n_q, n_kv).bytes;
  return DI_OK;
}

int detllm_attn_packed(const int8_t* q8, const int64_t* tpos, const int8_t* kpool,
                       const int8_t* vpool, int n_pages, const int32_t* table, int width,
                       const int32_t* cu, const int32_t* past, int N, int B, int S, int max_new,
                       int n_q, int n_kv, void* work, int64_t work_bytes, int64_t* out,
                       int32_t* err, hipStream_t s) {
  const int rc = packed_check(N, B, S, max_new, n_q, n_kv);
  if (rc != DI_OK) return rc;
  if (N == 0) return DI_OK;
  if (!q8 || !tpos || !kv_ok(kpool, vpool, table, width) || n_pages < 1 || !cu || !past || !out ||
      S > (i64)width * DI_PAGE)
    return DI_EINVAL;
  // (16-byte loads)
  if ((((uintptr_t)q8 | (uintptr_t)kpool | (uintptr_t)vpool) & 15) != 0) return DI_EINVAL;
  const Plan p = packed_plan(N, B, S, max_new, n_q, n_kv);
  if (p.bytes > 0 && (!work || ((uintptr_t)work & 15))) return DI_EINVAL;
  if (work_bytes < p.bytes) return DI_ERANGE;
  PackedArgs a{};
  a.q8 = q8; a.tpos = tpos;
  a.kv = KVPages{(int8_t*)kpool, (int8_t*)vpool, table, width, n_kv};
  a.n_pages = n_pages; a.cu = cu; a.past = past; a.N = N; a.B = B; a.S = S;
  a.n_q = n_q; a.n_kv = n_kv; a.lg = __builtin_ctz((unsigned)(n_q / n_kv));
  a.max_new = max_new; a.score_rows = (int)p.score_rows; a.units = p.units; a.step = p.step;
  a.chunk = p.chunk; a.nch = p.nch; a.out = out; a.err = err;
  a.few_rows = p.score_rows < (i64)B * p.rows ? 0 : p.rows;
  char* const w = (char*)work;
  a.scores = (int32_t*)(w + p.scores_at);
  a.smax = (int32_t*)(w + p.max_at);
  a.sden = (int64_t*)(w + p.den_at);
  a.part = p.nch > 1 && !p.few ? (int32_t*)(w + p.part_at) : nullptr;
  const i64 blocks = (i64)p.step * n_kv;
  if (blocks > 0x7fffffff) return DI_ERANGE;
  const dim3 grid((unsigned)blocks);
  if (p.one) {
    if (!p.few) hipLaunchKernelGGL(k_packed_one, grid, dim3(256), 0, s, a);
    else if (p.rows <= 8) {
      if (S <= 512) hipLaunchKernelGGL((k_packed_few<1, true>), grid, dim3(512), 0, s, a);
      else if (S <= 1024) hipLaunchKernelGGL((k_packed_few<2, true>), grid, dim3(512), 0, s, a);
      else hipLaunchKernelGGL((k_packed_few<4, true>), grid, dim3(512), 0, s, a);
    } else {
      if (S <= 512) hipLaunchKernelGGL((k_packed_few<1, false>), grid, dim3(512), 0, s, a);
      else if (S <= 1024) hipLaunchKernelGGL((k_packed_few<2, false>), grid, dim3(512), 0, s, a);
      else hipLaunchKernelGGL((k_packed_few<4, false>), grid, dim3(512), 0, s, a);
    }
    DI_LAUNCH_CHECK();
    return DI_OK;
  }
#define DI_PHASES(FEW_)                                                              \
  hipLaunchKernelGGL((k_packed_phase<PH_MAX, FEW_>), grid, dim3(256), 0, s, a);      \
  DI_LAUNCH_CHECK();                                                                 \
  hipLaunchKernelGGL((k_packed_phase<PH_DEN, FEW_>), grid, dim3(256), 0, s, a);      \
  DI_LAUNCH_CHECK();                                                                 \
  hipLaunchKernelGGL((k_packed_phase<PH_PV, FEW_>), grid, dim3(256), 0, s, a);       \
  DI_LAUNCH_CHECK()
  if (p.few && p.rows <= 8) { DI_PHASES(8); }
  else if (p.few) { DI_PHASES(16); }
  else { DI_PHASES(0); }
#undef DI_PHASES
  if (a.part) {
    hipLaunchKernelGGL(k_packed_join, dim3(N), dim3(256), 0, s, a);
    DI_LAUNCH_CHECK();
  }
  return DI_OK;
}

}  // extern "C"
