// Eviction from the paged KV cache by accumulated attention weight (gfx950).
// No counterpart in the reference: which slots of a row stay
// (detllm_kv_select), and the cache moved together (detllm_kv_compact). The
// weights are integers and ties go to the lower slot, so the choice is the same
// on every run and for every batch a row is in.

#include "attn_tiles.h"
#include "attn_window.h"

namespace {

// ---- the weights of a row's valid slots, over all kv heads: w [B][S]
__global__ __launch_bounds__(256) void k_kv_weight(const int64_t* acc, i64 acc_stride,
                                                   const uint8_t* valid, i64 valid_stride, int S,
                                                   int n_kv, int64_t* w) {
  keep_hidden_args();
  const int s = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
  if (s >= S) return;
  const int64_t* row = acc + (i64)b * n_kv * acc_stride + s;
  i64 sum = 0;
  for (int h = 0; h < n_kv; ++h) sum = wadd(sum, row[h * acc_stride]);
  w[(i64)b * S + s] = sum;
}

// ---- the slots that stay, a block per row. Of the valid slots the first
// `sinks` and the last `recent` stay; between them, the `need` heaviest: their
// least weight comes from a radix selection over the weights' 8 bytes (as
// unsigned keys, the largest first), then one pass in slot order takes every
// slot above it and the first ones that equal it.
constexpr int SEL_NT = 1024;

__device__ __forceinline__ u64 weight_key(i64 w) { return (u64)w ^ (1ull << 63); }

__global__ __launch_bounds__(SEL_NT) void k_kv_select(const int64_t* acc, i64 acc_stride,
                                                      const uint8_t* valid, i64 valid_stride,
                                                      const int64_t* w, int S, int n_kv, int budget,
                                                      int recent, int sinks, int32_t* keep,
                                                      int64_t* kept) {
  keep_hidden_args();
  __shared__ int hist[256], red[SEL_NT / 64], pick[2];
  const int b = blockIdx.x, tid = threadIdx.x;
  const uint8_t* vrow = valid + (i64)b * valid_stride;
  const int64_t* wrow = w + (i64)b * S;
  int32_t* krow = keep + (i64)b * budget;
  int count = 0;
  for (int s0 = 16 * tid; s0 < S; s0 += 16 * SEL_NT) count += __popc(valid16(vrow, s0, S));
  int n;
  block_count_before<SEL_NT>(count, red, &n);
  // valid slots in [lo, hi) compete for `need` places
  int lo = S, hi = S, need = 0;
  if (n > budget) {
    lo = nth_valid_end<SEL_NT>(vrow, S, sinks);
    hi = recent > 0 ? nth_valid_back<SEL_NT>(vrow, S, recent) : S;
    need = budget - sinks - recent;
  }
  u64 least = 0;  // the need-th largest key
  int ties = 0;   // places left for slots of that key
  if (need > 0) {
    u64 known = 0;
    int left = need;
    for (int sh = 56; sh >= 0; sh -= 8) {
      const u64 mask = sh == 56 ? 0ull : ~0ull << (sh + 8);
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int s = lo + tid; s < hi; s += SEL_NT)
        if (vrow[s] != 0) {
          const u64 k = weight_key(wrow[s]);
          if ((k & mask) == known) atomicAdd(&hist[(k >> sh) & 255], 1);
        }
      __syncthreads();
      // the digit that holds the left-th largest: keys above digit d number
      // fewer than left, with d's at least left
      const int d = 255 - tid;
      const int c = tid < 256 ? hist[d] : 0;
      int total;
      const int above = block_count_before<SEL_NT>(c, red, &total);
      if (tid < 256 && above < left && above + c >= left) {
        pick[0] = d;
        pick[1] = left - above;
      }
      __syncthreads();
      known |= (u64)pick[0] << sh;
      left = pick[1];
    }
    least = known;
    ties = left;
  }
  // the kept slots in order
  int at = 0, tied = 0;
  for (int base = 0; base < S; base += SEL_NT) {
    const int s = base + tid;
    const bool v = s < S && vrow[s < S ? s : 0] != 0;
    bool in = v && (n <= budget || s < lo || s >= hi);
    bool tie = false;
    if (v && !in && need > 0) {
      const u64 k = weight_key(wrow[s]);
      in = k > least;
      tie = k == least;
    }
    int total;
    const int before = block_count_before<SEL_NT>(tie ? 1 : 0, red, &total);
    in = in || (tie && tied + before < ties);
    tied += total;
    const int place = at + block_count_before<SEL_NT>(in ? 1 : 0, red, &total);
    if (in) krow[place] = s;
    at += total;
  }
  for (int i = at + tid; i < budget; i += SEL_NT) krow[i] = -1;
  __syncthreads();
  for (i64 i = tid; i < (i64)n_kv * budget; i += SEL_NT) {
    const int h = (int)(i / budget), p = (int)(i % budget);
    kept[((i64)b * n_kv + h) * budget + p] =
        p < at ? acc[((i64)b * n_kv + h) * acc_stride + krow[p]] : 0;
  }
}

// ---- the kept slots' K and V moved to the pages of dst, in slot order
constexpr int KVC_LAYERS = 32;  // layers per launch (pool pointers by value)
constexpr int KVC_PAGES = 4;    // source pages of V in LDS at once

struct CompactArgs {
  int8_t* k[KVC_LAYERS];
  int8_t* v[KVC_LAYERS];
  const int32_t* table;  // [B][width]
  const int32_t* dst;    // [B][dst_width]
  const int32_t* keep;   // [B][budget] ascending, -1 behind
  int width, dst_width, budget, n_kv;
};

// Block = (kv head and K or V, row, layer), page after page of dst: slot i
// comes from slot keep[i] >= i, so a page of dst may be the table's page of the
// same place or an earlier one (everything it held has been read by then), and
// the reads of a page end before its writes begin.
__global__ __launch_bounds__(256) void k_kv_compact(CompactArgs a) {
  keep_hidden_args();
  __shared__ __attribute__((aligned(16))) int8_t src[KVC_PAGES][128 * DI_PAGE];
  __shared__ int32_t slot[DI_PAGE];  // the page's source slots
  const int h = blockIdx.x >> 1, b = blockIdx.y, tid = threadIdx.x;
  const bool is_v = blockIdx.x & 1;
  const KVPages kv{a.k[blockIdx.z], a.v[blockIdx.z], a.table, a.width, a.n_kv};
  const int32_t* krow = a.keep + (i64)b * a.budget;
  const int npages = min(a.dst_width, (a.budget + DI_PAGE - 1) / DI_PAGE);
  for (int j = 0; j < npages; ++j) {
    const int to = a.dst[(i64)b * a.dst_width + j];
    __syncthreads();  // (the last page's reads of slot)
    if (tid < DI_PAGE) {
      const int i = j * DI_PAGE + tid;
      slot[tid] = i < a.budget ? krow[i] : -1;
    }
    __syncthreads();
    if (to < 0) continue;  // block-uniform
    if (!is_v) {
      v4i x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = slot[u * 32 + (tid >> 3)];
        const int pg = kv.page(b, s);
        x[u] = v4i{0, 0, 0, 0};
        if (pg >= 0) x[u] = *(const v4i*)(kv.krow(pg, h, s & (DI_PAGE - 1)) + (tid & 7) * 16);
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *(v4i*)(kv.krow(to, h, u * 32 + (tid >> 3)) + (tid & 7) * 16) = x[u];
      continue;
    }
    // V^T: thread (tid / 32, tid % 32) makes slots 4 (tid % 32) .. + 3 of
    // channels tid / 32 + 8 u
    uint32_t x[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) x[u] = 0;
    int s4[4], first = -1, last = -1;
#pragma unroll
    for (int r = 0; r < 4; ++r) s4[r] = slot[4 * (tid & 31) + r];
    for (int i = 0; i < DI_PAGE; ++i) {
      const int s = slot[i];
      if (s >= 0) {
        first = first < 0 ? s / DI_PAGE : first;
        last = s / DI_PAGE;
      }
    }
    for (int p0 = first; first >= 0 && p0 <= last; p0 += KVC_PAGES) {
      __syncthreads();  // (the last pages' reads)
      for (int q = 0; q < KVC_PAGES; ++q) {
        const int pg = p0 + q <= last ? kv.page(b, (i64)(p0 + q) * DI_PAGE) : -1;
        const int8_t* from = kv.vchan(pg < 0 ? 0 : pg, h, 0);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          v4i y = v4i{0, 0, 0, 0};
          if (pg >= 0) y = *(const v4i*)(from + (u * 256 + tid) * 16);
          *(v4i*)(src[q] + (u * 256 + tid) * 16) = y;
        }
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int q = s4[r] / DI_PAGE - p0;
        if (s4[r] >= 0 && q >= 0 && q < KVC_PAGES) {
          const int8_t* from = src[q] + (tid >> 5) * DI_PAGE + (s4[r] & (DI_PAGE - 1));
#pragma unroll
          for (int u = 0; u < 16; ++u)
            x[u] |= (uint32_t)(uint8_t)from[u * 8 * DI_PAGE] << (8 * r);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 16; ++u)
      *(uint32_t*)(kv.vchan(to, h, (tid >> 5) + 8 * u) + 4 * (tid & 31)) = x[u];
  }
}

}  // namespace

extern "C" {

int detllm_kv_select_work(int B, int S, int64_t* bytes) {
  if (!bytes || B < 0 || S < 0) return DI_EINVAL;
  *bytes = (i64)B * S * 8;
  return DI_OK;
}

int detllm_kv_select(const int64_t* acc, int64_t acc_stride, const uint8_t* valid,
                     int64_t valid_stride, int B, int S, int n_kv, int budget, int recent,
                     int sinks, int32_t* keep, int64_t* kept, void* work, int64_t work_bytes,
                     hipStream_t s) {
  if (S < 0 || n_kv < 1 || budget < 1 || recent < 0 || sinks < 0 ||
      (i64)recent + sinks > budget || acc_stride < S || valid_stride < S)
    return DI_EINVAL;
  if (B <= 0) return DI_OK;
  if (!keep || !kept || (S > 0 && (!acc || !valid))) return DI_EINVAL;
  if (B > 65535) return DI_ERANGE;
  if (S > 0 && (!work || work_bytes < (i64)B * S * 8)) return DI_ERANGE;
  if (S > 0)
    hipLaunchKernelGGL(k_kv_weight, dim3((S + 255) / 256, B), dim3(256), 0, s, acc, acc_stride,
                       valid, valid_stride, S, n_kv, (int64_t*)work);
  hipLaunchKernelGGL(k_kv_select, dim3(B), dim3(SEL_NT), 0, s, acc, acc_stride, valid, valid_stride,
                     (const int64_t*)work, S, n_kv, budget, recent, sinks, keep, kept);
  DI_LAUNCH_CHECK();
  return DI_OK;
}

int detllm_kv_compact(int8_t* const* kpools, int8_t* const* vpools, int n_layers,
                      const int32_t* table, int width, const int32_t* dst, int dst_width,
                      const int32_t* keep, int B, int budget, int n_kv, hipStream_t s) {
  if (n_layers < 0 || width < 1 || dst_width < 0 || budget < 0 || n_kv < 1) return DI_EINVAL;
  if (B <= 0 || n_layers == 0 || dst_width == 0 || budget == 0) return DI_OK;
  if (!kpools || !vpools || !table || !dst || !keep) return DI_EINVAL;
  if (B > 65535 || n_kv > (1 << 20)) return DI_ERANGE;
  for (int l = 0; l < n_layers; ++l)
    if (!kpools[l] || !vpools[l]) return DI_EINVAL;
  for (int l0 = 0; l0 < n_layers; l0 += KVC_LAYERS) {
    CompactArgs a{};
    const int n = n_layers - l0 < KVC_LAYERS ? n_layers - l0 : KVC_LAYERS;
    for (int l = 0; l < n; ++l) {
      a.k[l] = kpools[l0 + l];
      a.v[l] = vpools[l0 + l];
    }
    a.table = table; a.dst = dst; a.keep = keep;
    a.width = width; a.dst_width = dst_width; a.budget = budget; a.n_kv = n_kv;
    hipLaunchKernelGGL(k_kv_compact, dim3(2 * n_kv, B, n), dim3(256), 0, s, a);
  }
  DI_LAUNCH_CHECK();
  return DI_OK;
}

}  // extern "C"
