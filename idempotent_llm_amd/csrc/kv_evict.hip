// Eviction from the paged KV cache by accumulated attention weight (gfx950).
// No counterpart in the reference: which slots of a row stay
// (detllm_kv_select), and the cache moved together (detllm_kv_compact). The
// weights are integers and ties go to the lower slot, so the choice is the same
// on every run and for every batch a row is in.

#include "attn_tiles.h"
#include "attn_window.h"

namespace {

// ---- the weights of a row's slots over all kv heads: w [B][S]
__global__ __launch_bounds__(256) void k_kv_weight(const int64_t* acc, i64 acc_stride, int S,
                                                   int n_kv, int64_t* w) {
  keep_hidden_args();
  const int s = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
  if (s >= S) return;
  const int64_t* row = acc + (i64)b * n_kv * acc_stride + s;
  i64 sum = 0;
  for (int h = 0; h < n_kv; ++h) sum = wadd(sum, row[h * acc_stride]);
  w[(i64)b * S + s] = sum;
}

// ---- the slots that stay, a block per row. A thread owns `per` consecutive
// slots, so one scan of the valid counts gives every slot its rank among the
// valid ones (the first `sinks` and the last `recent` stay by rank) and one scan
// of the kept counts its place. Between them the `need` heaviest stay. Their
// least weight is found by digits of 8 bits from the highest bit in which the
// weights differ (keys: the weight as unsigned, larger first), until the digit
// that holds the need-th largest has few slots left; these are ranked one
// against the other, by key and then by slot.
// Bound by the chain of these steps on one CU per row and by that CU's loads (a
// row of 4000 slots and 8 heads is 256 KB, 5 us; the kept accumulators 3.5): 20 us
// at 8 rows of 4000 slots, 7 at one of 400.
// E > 0: a thread's keys stay in registers, summed here over the kv heads (rows
// of at most 1024 E slots); E = 0: k_kv_weight has summed them to w.
constexpr int SEL_NT = 1024;
constexpr int SEL_RANK = SEL_NT / 8;  // slots ranked one against the other, 8 threads each

struct SelectArgs {
  const int64_t* acc;
  i64 acc_stride;
  const uint8_t* valid;
  i64 valid_stride;
  const int64_t* w;
  int S, n_kv, budget, recent, sinks;
  int32_t* keep;
  int64_t* kept;
};

// The wave's OR of v, in lane 63
__device__ __forceinline__ u64 wave_or(u64 v) {
  v |= (u64)dpp64<0xB1, 0xF>((i64)v, 0);
  v |= (u64)dpp64<0x4E, 0xF>((i64)v, 0);
  v |= (u64)dpp64<0x141, 0xF>((i64)v, 0);
  v |= (u64)dpp64<0x140, 0xF>((i64)v, 0);
  v |= (u64)dpp64<0x142, 0xA>((i64)v, 0);
  v |= (u64)dpp64<0x143, 0xC>((i64)v, 0);
  return v;
}

template <int E>
__global__ __launch_bounds__(SEL_NT) void k_kv_select(SelectArgs a) {
  keep_hidden_args();
  __shared__ int hist[256], red[SEL_NT / 64], pick[3], nlist;
  __shared__ u64 least_key, keys[SEL_RANK];
  __shared__ int slots[SEL_RANK];
  const int b = blockIdx.x, tid = threadIdx.x;
  const uint8_t* vrow = a.valid + (i64)b * a.valid_stride;
  int32_t* krow = a.keep + (i64)b * a.budget;
  const int per = E > 0 ? E : (a.S + SEL_NT - 1) / SEL_NT;
  const int s0 = tid * per;
  auto key_of = [](i64 w) { return (u64)w ^ (1ull << 63); };
  u64 reg[E > 0 ? E : 1];
  if constexpr (E > 0) {
    // slots tid, tid + 1024, ... load together; LDS turns them into runs
    i64 sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0;
    constexpr int HU = E > 4 ? 2 : 8;  // heads in flight
    for (int h = 0; h < (a.S > 0 ? a.n_kv : 0); h += HU) {
      i64 x[HU][E];
#pragma unroll
      for (int q = 0; q < HU; ++q) {
        const int64_t* row = a.acc + ((i64)b * a.n_kv + ::min(h + q, a.n_kv - 1)) * a.acc_stride;
#pragma unroll
        for (int e = 0; e < E; ++e) x[q][e] = row[::min(tid + e * SEL_NT, a.S - 1)];
      }
#pragma unroll
      for (int q = 0; q < HU; ++q)
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] = wadd(sum[e], h + q < a.n_kv ? x[q][e] : 0);
    }
    if constexpr (E == 1) {
      reg[0] = key_of(sum[0]);
    } else {
      extern __shared__ __attribute__((aligned(16))) u64 turn[];  // [1024 E]
#pragma unroll
      for (int e = 0; e < E; ++e) turn[tid + e * SEL_NT] = key_of(sum[e]);
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) reg[e] = turn[s0 + e];
    }
  }
  // each(f): f(slot, key, valid) of the thread's slots below S, in order
  uint32_t vbits = 0;
  if constexpr (E > 0) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      vbits |= (s0 + e < a.S && vrow[s0 + e < a.S ? s0 + e : 0] != 0 ? 1u : 0u) << e;
  }
  auto each = [&](auto&& f) {
    if constexpr (E > 0) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if ((vbits >> e) & 1u) f(s0 + e, reg[e]);
    } else {
      for (int e = 0; e < per; ++e)
        if (s0 + e < a.S && vrow[s0 + e] != 0) f(s0 + e, key_of(a.w[(i64)b * a.S + s0 + e]));
    }
  };
  int mine = 0, n;
  each([&](int, u64) { ++mine; });
  const int rank0 = block_count_before<SEL_NT>(mine, red, &n);
  // the valid slots of rank [lo, hi) compete for `need` places
  const bool all = n <= a.budget;
  const int lo = a.sinks, hi = n - a.recent, need = all ? 0 : a.budget - a.sinks - a.recent;
  // each competing slot of this thread
  auto compete = [&](auto&& f) {
    int r = rank0;
    each([&](int s, u64 k) {
      if (r >= lo && r < hi) f(s, k);
      ++r;
    });
  };
  u64 least = 0;     // the digits found so far of the need-th largest key
  u64 known = 0;     // their mask
  int left = need;   // places for keys whose known digits are `least`
  bool ranked = false;
  if (need > 0) {
    // the bits in which the competing keys differ: set in one, clear in another
    u64 ones = 0, zeros = 0;
    compete([&](int, u64 k) {
      ones |= k;
      zeros |= ~k;
    });
    ones = wave_or(ones);
    zeros = wave_or(zeros);
    if ((tid & 63) == 63) {
      keys[tid >> 6] = ones;
      keys[SEL_NT / 64 + (tid >> 6)] = zeros;
    }
    __syncthreads();
    ones = zeros = 0;
#pragma unroll
    for (int w = 0; w < SEL_NT / 64; ++w) {
      ones |= keys[w];
      zeros |= keys[SEL_NT / 64 + w];
    }
    const u64 first = ones & ~zeros;  // (what all agree on)
    int top = 64 - clz64(ones & zeros);  // bits [0, top) may differ (0: all keys are equal)
    known = top == 64 ? 0 : ~0ull << top;
    least = first & known;
    int count = hi - lo;  // keys whose known digits are `least`
    while (top > 0 && left < count) {
      if (count <= SEL_RANK) {  // block-uniform
        ranked = true;
        break;
      }
      const int sh = top > 8 ? top - 8 : 0;
      const u64 digits = (1ull << (top - sh)) - 1;
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      compete([&](int, u64 k) {
        if ((k & known) == least) atomicAdd(&hist[(k >> sh) & digits], 1);
      });
      __syncthreads();
      // the digit that holds the left-th largest: keys of the digits above
      // number fewer than left, with its own at least left
      const int dg = 255 - tid, c = tid < 256 ? hist[dg] : 0;
      int total;
      const int above = block_count_before<SEL_NT>(c, red, &total);
      if (tid < 256 && above < left && above + c >= left) {
        pick[0] = dg;
        pick[1] = left - above;
        pick[2] = c;
      }
      __syncthreads();
      least |= (u64)pick[0] << sh;
      known |= digits << sh;
      left = pick[1];
      count = pick[2];
      top = sh;
    }
    if (ranked) {
      // the key of the left-th largest, and the slots at or before which equal
      // keys stay: every listed slot counts those ahead of it
      __syncthreads();
      if (tid == 0) nlist = 0;
      __syncthreads();
      compete([&](int s, u64 k) {
        if ((k & known) == least) {
          const int i = atomicAdd(&nlist, 1);
          keys[i] = k;
          slots[i] = s;
        }
      });
      __syncthreads();
      const int c = nlist, at = tid >> 3;
      const u64 k = keys[at < c ? at : 0];
      const int s = slots[at < c ? at : 0];
      int ahead = 0;
#pragma unroll 4
      for (int i = tid & 7; i < c; i += 8)
        ahead += keys[i] > k || (keys[i] == k && slots[i] < s) ? 1 : 0;
      ahead = sum8_i32(ahead);
      if (at < c && (tid & 7) == 0 && ahead == left - 1) {
        least_key = k;
        pick[0] = s;
      }
      __syncthreads();
      least = least_key;
      known = ~0ull;
    }
  }
  // A competing slot stays if its known digits are above `least`, or equal it
  // and: all of those stay (left covers them), or it lies at or before the last
  // one that does (ranked), or its place among them is below left.
  const int upto = ranked ? pick[0] : 0;
  int tied = 0;
  if (need > 0 && !ranked) {
    int c = 0, total;
    compete([&](int, u64 k) { c += (k & known) == least ? 1 : 0; });
    tied = block_count_before<SEL_NT>(c, red, &total);
  }
  auto kept_each = [&](auto&& f) {
    int r = rank0, t = tied;
    each([&](int s, u64 k) {
      bool in = all || r < lo || r >= hi;
      if (!in && need > 0) {
        const u64 kk = k & known;
        in = kk > least;
        if (kk == least) {
          in = ranked ? s <= upto : t < left;
          ++t;
        }
      }
      ++r;
      if (in) f(s);
    });
  };
  int c = 0, total;
  kept_each([&](int) { ++c; });
  int place = block_count_before<SEL_NT>(c, red, &total);
  kept_each([&](int s) { krow[place++] = s; });
  // (unsigned: a budget near 2^31 plus a step of SEL_NT passes an int)
  for (uint32_t i = total + tid; i < (uint32_t)a.budget; i += SEL_NT) krow[i] = -1;
  __syncthreads();
  for (uint32_t p = tid; p < (uint32_t)a.budget; p += SEL_NT) {
    const int s = p < (uint32_t)total ? krow[p] : 0;
    const int64_t* from = a.acc + (i64)b * a.n_kv * a.acc_stride + s;
    int64_t* to = a.kept + (i64)b * a.n_kv * a.budget + p;
#pragma unroll 8
    for (int h = 0; h < a.n_kv; ++h)
      to[(i64)h * a.budget] = p < (uint32_t)total ? from[(i64)h * a.acc_stride] : 0;
  }
}

// ---- the kept slots' K and V moved to the pages of dst, in slot order. Bound by
// HBM: a kept slot's K row is one line, but its V is a byte of 128 lines, so V is
// read whole. 8 rows, 8 layers and 8 kv heads, 1024 of 4000 slots: 114 us for 460
// MB, 270 of them V's pages.
constexpr int KVC_LAYERS = 32;  // layers per launch (pool pointers by value)
constexpr int KVC_PAGES = 2;    // source pages of V in LDS at once
constexpr int KVC_MAXP = 1024;  // pages of V listed at once
constexpr int KVC_MAXDST = 1 << 23;  // pages of dst (their slots are numbered in 32 bits)

struct CompactArgs {
  int8_t* k[KVC_LAYERS];
  int8_t* v[KVC_LAYERS];
  const int32_t* table;  // [B][width]
  const int32_t* dst;    // [B][dst_width]
  const int32_t* keep;   // [B][budget] ascending, -1 behind (budget 0: any address)
  int width, dst_width, budget, n_kv, n_pages;
  int nseg, per;         // parts of dst's pages (one block each), pages of a part

  // page of row b's slot s, and the page for j of dst (-1: none, or not of the
  // pools)
  __device__ __forceinline__ int from(const KVPages& kv, int b, i64 s) const {
    const int pg = kv.page(b, s);
    return pg < n_pages ? pg : -1;
  }
  __device__ __forceinline__ int to(int b, int j) const {
    const int pg = j < dst_width ? dst[(i64)b * dst_width + j] : -1;
    return pg < n_pages ? pg : -1;
  }
};

// K: page after page of dst, 8 lanes a row of 128 bytes. Slot i comes from slot
// keep[i] >= i, so a page of dst may be the table's page of the same place or an
// earlier one: everything it held for later pages has been read, because the
// reads of a page end before its writes begin (the barrier) and those of the
// page after it come from places behind it.
__device__ __forceinline__ void compact_k(const CompactArgs& a, const KVPages& kv, int h, int b,
                                          int j0, int j1) {
  const int tid = threadIdx.x;
  const int32_t* krow = a.keep + (i64)b * a.budget;
  int s[4];  // the next page's source slots of this thread's rows
  auto load_slots = [&](int j) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = j * DI_PAGE + u * 32 + (tid >> 3);
      s[u] = i < a.budget ? krow[i] : -1;
    }
  };
  v4i x[4], y[4];
  auto load_rows = [&](v4i (&r)[4]) {
    int pg[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) pg[u] = a.from(kv, b, s[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      r[u] = v4i{0, 0, 0, 0};
      if (pg[u] >= 0) r[u] = *(const v4i*)(kv.krow(pg[u], h, s[u] & (DI_PAGE - 1)) + (tid & 7) * 16);
    }
  };
  load_slots(j0);
  load_rows(x);
  if (j0 + 1 < j1) load_slots(j0 + 1);
  for (int j = j0; j < j1; ++j) {
    const int to = a.to(b, j);
    if (j + 1 < j1) load_rows(y);
    if (j + 2 < j1) load_slots(j + 2);
#pragma unroll
    for (int u = 0; u < 4; ++u) asm volatile("" ::"v"(x[u]));  // (this page's reads have ended)
    __syncthreads();
    if (to >= 0) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *(v4i*)(kv.krow(to, h, u * 32 + (tid >> 3)) + (tid & 7) * 16) = x[u];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = y[u];
  }
}

// V^T: a kept slot is a byte of each of 128 channel rows, so whole source pages
// are read, each once, KVC_PAGES at a time: the two next lots load to registers
// while bytes are taken from the one in LDS. Thread (tid / 32, tid % 32) makes
// slots 4 (tid % 32) .. + 3 of channels tid / 32 + 8 u of a page of dst in
// registers and writes them when every source page of that page has passed. The
// same order as in compact_k: a page is written when its last source page, and
// all before it, are in LDS or behind.
__device__ __forceinline__ void compact_v(const CompactArgs& a, const KVPages& kv, int h, int b,
                                          int j0, int j1) {
  __shared__ __attribute__((aligned(16))) int8_t src[KVC_PAGES][128 * DI_PAGE];
  __shared__ uint16_t list[KVC_MAXP];    // source pages with kept slots, ascending
  __shared__ int32_t start[KVC_MAXP + 1];  // the first kept slot from each
  __shared__ int red[4];
  const int tid = threadIdx.x;
  const int32_t* krow = a.keep + (i64)b * a.budget;
  int np = 0, n = 0;  // listed pages, kept slots
  const int ifirst = j0 * DI_PAGE, iend = ::min(j1 * DI_PAGE, a.budget);
  for (int i0 = ifirst; i0 < iend; i0 += 256) {
    const int i = i0 + tid;
    const int s = i < iend ? krow[i] : -1;
    const int before_s = i > ifirst && i < iend ? krow[i - 1] : -1;
    const bool lead = s >= 0 && (i == ifirst || s / DI_PAGE != before_s / DI_PAGE);
    int total;
    const int before = block_count_before<256>((lead ? 1 : 0) | (s >= 0 ? 0x10000 : 0), red, &total);
    const int at = np + (before & 0xFFFF);
    if (lead && at < KVC_MAXP) {  // (an ascending keep within the table has no more)
      list[at] = (uint16_t)(s / DI_PAGE);
      start[at] = i;
    }
    np = ::min(np + (total & 0xFFFF), KVC_MAXP);
    n += total >> 16;
  }
  if (tid == 0) start[np] = ifirst + n;
  __syncthreads();
  v4i pa[KVC_PAGES][4], pb[KVC_PAGES][4];
  auto load = [&](int p0, v4i (&x)[KVC_PAGES][4]) {
#pragma unroll
    for (int q = 0; q < KVC_PAGES; ++q) {
      const int pg = p0 + q < np ? a.from(kv, b, (i64)list[p0 + q] * DI_PAGE) : -1;
      const int8_t* from = kv.vchan(pg < 0 ? 0 : pg, h, 0);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        x[q][u] = v4i{0, 0, 0, 0};
        if (pg >= 0) x[q][u] = *(const v4i*)(from + (u * 256 + tid) * 16);
      }
    }
  };
  const int ch = tid >> 5, i4 = 4 * (tid & 31);
  uint32_t x[16];
#pragma unroll
  for (int u = 0; u < 16; ++u) x[u] = 0;
  int j = j0;  // the page of dst being made, and this thread's source slots of it
  int s4[4];
  auto load_slots = [&] {
#pragma unroll
    for (int r = 0; r < 4; ++r) s4[r] = krow[::max(::min(j * DI_PAGE + i4 + r, a.budget - 1), 0)];
  };
  load_slots();
  auto flush = [&] {
    const int to = a.to(b, j);
    if (to >= 0) {
#pragma unroll
      for (int u = 0; u < 16; ++u) *(uint32_t*)(kv.vchan(to, h, ch + 8 * u) + i4) = x[u];
    }
#pragma unroll
    for (int u = 0; u < 16; ++u) x[u] = 0;
    ++j;
    load_slots();
  };
  auto step = [&](int p0, v4i (&in)[KVC_PAGES][4]) {
    __syncthreads();  // the last pages have been read
#pragma unroll
    for (int q = 0; q < KVC_PAGES; ++q)
#pragma unroll
      for (int u = 0; u < 4; ++u) *(v4i*)(src[q] + (u * 256 + tid) * 16) = in[q][u];
    __syncthreads();
    if (p0 + 2 * KVC_PAGES < np) load(p0 + 2 * KVC_PAGES, in);
    const int begin = start[p0], end = start[::min(p0 + KVC_PAGES, np)];
    for (;;) {
      // bytes of page j from these source pages
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = j * DI_PAGE + i4 + r;
        if (i >= begin && i < end) {
          const int s = s4[r], pg = s / DI_PAGE;
          int q = 0;
#pragma unroll
          for (int t = 1; t < KVC_PAGES; ++t) q = p0 + t < np && (int)list[p0 + t] <= pg ? t : q;
          const int8_t* from = src[q] + ch * DI_PAGE + (s & (DI_PAGE - 1));
#pragma unroll
          for (int u = 0; u < 16; ++u)
            x[u] |= (uint32_t)(uint8_t)from[u * 8 * DI_PAGE] << (8 * r);
        }
      }
      if (end < (j + 1) * DI_PAGE) break;  // block-uniform
      flush();
    }
  };
  if (np > 0) load(0, pa);
  if (np > KVC_PAGES) load(KVC_PAGES, pb);
  for (int p0 = 0; p0 < np; p0 += 2 * KVC_PAGES) {
    step(p0, pa);
    if (p0 + KVC_PAGES < np) step(p0 + KVC_PAGES, pb);
  }
  while (j < j1) flush();
}

// Where the (kv head, K or V, row, layer) blocks alone leave the card idle, dst's
// pages are cut into parts, about four blocks per CU. That holds for rows whose
// dst pages are none of their table's; where one is, the order above has to be
// kept and the row's first block takes all parts. Kept of a row's slots, new pages
// against its own: 150 of 400 (8 layers, 8 heads) 7.5 and 8.7 us, 2000 of 4000 (2
// layers, 2 heads) 8.6 and 54, 20000 of 131000 (1 layer, 8 heads) 179 and 1332.
__global__ __launch_bounds__(256) void k_kv_compact(CompactArgs a) {
  keep_hidden_args();
  const int seg = blockIdx.x / (2 * a.n_kv), hk = blockIdx.x % (2 * a.n_kv);
  const int h = hk >> 1, b = blockIdx.y, npages = a.dst_width;  // (zeros past the budget)
  const KVPages kv{a.k[blockIdx.z], a.v[blockIdx.z], a.table, a.width, a.n_kv};
  int j0 = seg * a.per, j1 = ::min(j0 + a.per, npages);
  if (a.nseg > 1) {  // block-uniform
    bool hit = false;
    for (int t = threadIdx.x; t < a.width; t += 256) {
      const int x = a.table[(i64)b * a.width + t];
      for (int j = 0; j < npages; ++j) hit |= x >= 0 && a.dst[(i64)b * a.dst_width + j] == x;
    }
    if (__syncthreads_or(hit)) {
      if (seg > 0) return;
      j1 = npages;
    }
  }
  if (hk & 1) compact_v(a, kv, h, b, j0, j1);
  else compact_k(a, kv, h, b, j0, j1);
}

constexpr int SEL_FUSED = 16 * SEL_NT;  // slots per row whose keys fit registers

}  // namespace

extern "C" {

int detllm_kv_select_work(int B, int S, int64_t* bytes) {
  if (!bytes || B < 0 || S < 0) return DI_EINVAL;
  *bytes = S > SEL_FUSED ? (i64)B * S * 8 : 0;
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
  if (B > 65535 || S > 131071) return DI_ERANGE;
  const SelectArgs a{acc, acc_stride, valid, valid_stride, (const int64_t*)work, S, n_kv, budget,
                     recent, sinks, keep, kept};
  const dim3 grid(B), block(SEL_NT);
  if (S <= SEL_NT) {
    hipLaunchKernelGGL(k_kv_select<1>, grid, block, 0, s, a);
  } else if (S <= 4 * SEL_NT) {
    hipLaunchKernelGGL(k_kv_select<4>, grid, block, 4 * SEL_NT * 8, s, a);
  } else if (S <= SEL_FUSED) {
    hipLaunchKernelGGL(k_kv_select<16>, grid, block, 16 * SEL_NT * 8, s, a);
  } else {
    if (!work || work_bytes < (i64)B * S * 8) return DI_ERANGE;
    hipLaunchKernelGGL(k_kv_weight, dim3((S + 255) / 256, B), dim3(256), 0, s, acc, acc_stride, S,
                       n_kv, (int64_t*)work);
    hipLaunchKernelGGL(k_kv_select<0>, grid, block, 0, s, a);
  }
  DI_LAUNCH_CHECK();
  return DI_OK;
}

int detllm_kv_compact(int8_t* const* kpools, int8_t* const* vpools, int n_layers, int n_pages,
                      const int32_t* table, int width, const int32_t* dst, int dst_width,
                      const int32_t* keep, int B, int budget, int n_kv, hipStream_t s) {
  if (n_layers < 0 || n_pages < 1 || width < 1 || dst_width < 0 || budget < 0 || n_kv < 1)
    return DI_EINVAL;
  if (B <= 0 || n_layers == 0 || dst_width == 0) return DI_OK;
  if (!kpools || !vpools || !table || !dst || (!keep && budget > 0)) return DI_EINVAL;
  if (B > 65535 || n_kv > (1 << 20) || width > KVC_MAXP || budget > KVC_MAXP * DI_PAGE ||
      dst_width > KVC_MAXDST)
    return DI_ERANGE;
  for (int l = 0; l < n_layers; ++l)
    if (!kpools[l] || !vpools[l]) return DI_EINVAL;
  for (int l0 = 0; l0 < n_layers; l0 += KVC_LAYERS) {
    CompactArgs a{};
    const int n = n_layers - l0 < KVC_LAYERS ? n_layers - l0 : KVC_LAYERS;
    for (int l = 0; l < n; ++l) {
      a.k[l] = kpools[l0 + l];
      a.v[l] = vpools[l0 + l];
    }
    a.table = table; a.dst = dst; a.keep = budget > 0 ? keep : dst;
    a.width = width; a.dst_width = dst_width; a.budget = budget; a.n_kv = n_kv;
    a.n_pages = n_pages;
    const i64 blocks = 2 * (i64)n_kv * B * n, npages = dst_width;
    a.per = (int)imin(imax(npages * blocks / 1024, 1), npages);
    a.nseg = (int)((npages + a.per - 1) / a.per);
    hipLaunchKernelGGL(k_kv_compact, dim3((unsigned)(2 * n_kv * a.nseg), B, n), dim3(256), 0, s, a);
  }
  DI_LAUNCH_CHECK();
  return DI_OK;
}

}  // extern "C"
