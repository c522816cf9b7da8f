// Which slots a windowed query sees (gfx950).
//
// The query at slot t sees the valid slots s <= t with fewer than `window`
// valid slots in (s, t] or fewer than `sinks` valid slots in [0, s): its
// last `window` tokens and the row's first `sinks`. Counting valid slots
// instead of slots keeps what a row sees independent of its padding, so a
// row's result does not depend on the batch it is in. In slot numbers that is
// s >= lo(t) or s < e: lo(t) the window-th valid slot from t backward (0 if
// there are fewer), e one past the sinks-th valid slot. A block finds both by
// counting the row's validity flags, from its query backward and from slot 0
// forward, 16 flags per thread and step: as many as it is going to scan. The
// pages it scans are then those of the two ranges that hold a valid slot: a row
// whose window reaches back over padding does not scan the padding's pages (32
// rows of 8000 slots, a window of 2048 behind prompts padded by up to 3000
// slots: 110 us with them, 49 without, on four waves a block).
#pragma once

#include "common.h"

using namespace di;

namespace {

// The nonzero bytes of 16 flags, as bits.
__device__ __forceinline__ uint32_t flag_bits(const uint32_t (&x)[4]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = ((((x[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x[i]) & 0x80808080u) >> 7;
    m |= ((u | u >> 7 | u >> 14 | u >> 21) & 0xFu) << (4 * i);
  }
  return m;
}

// The nonzero flags of slots s0 .. s0 + 15 below `end`, as bits.
__device__ __forceinline__ uint32_t valid16(const uint8_t* vrow, int s0, int end) {
  if (s0 >= end) return 0;
  if (end >= 16) {  // (16 flags that end at `end` where the group would pass it)
    const int s1 = ::min(s0, end - 16);
    uint32_t x[4];
    __builtin_memcpy(x, vrow + s1, 16);
    return flag_bits(x) >> (s0 - s1);
  }
  uint32_t m = 0;
  for (int i = 0; i < end - s0; ++i) m |= (vrow[s0 + i] != 0 ? 1u : 0u) << i;
  return m;
}

// Position of the k-th (0-based) set bit of m, which has more than k.
__device__ __forceinline__ int nth_bit(u64 m, int k) {
  int pos = 0;
#pragma unroll
  for (int w = 32; w >= 1; w >>= 1) {
    const int c = __popcll(m & ((1ull << w) - 1));
    const bool up = k >= c;
    k -= up ? c : 0;
    m = up ? m >> w : m;
    pos += up ? w : 0;
  }
  return pos;
}

// The block's NT threads hold counts c in thread order: the number before
// this thread's (exclusive) and, in *total, the whole sum. red: NT / 64 words.
template <int NT>
__device__ __forceinline__ int block_count_before(int c, int* red, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = c;  // inclusive over the wave: DPP shifts within rows of 16, then row ends
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x111, 0xF, 0xF, false);
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x112, 0xF, 0xF, false);
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x114, 0xF, 0xF, false);
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x118, 0xF, 0xF, false);
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x142, 0xA, 0xF, false);
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x143, 0xC, 0xF, false);
  __syncthreads();  // (the words may still be read from the last call)
  if (lane == 63) red[wave] = incl;
  __syncthreads();
  int before = incl - c, sum = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    before += w < wave ? red[w] : 0;
    sum += red[w];
  }
  *total = sum;
  return before;
}

// The n-th valid slot is found in steps of 16 NT flags; the first step of both
// directions is loaded and counted together (one round trip and one count where
// the window and the sinks lie in it).
template <int NT>
struct ValidScan {
  int* red;    // shared: NT / 64 words
  int* found;  // shared: 2 words

  // one past the n-th valid slot of [0, end) after `seen` in [0, base): `end` if
  // there are fewer. All of these are block-uniform.
  __device__ __forceinline__ int forward(const uint8_t* vrow, int end, int n, int base, int seen) {
    for (; base < end; base += 16 * NT) {
      const int s0 = base + 16 * (int)threadIdx.x;
      const uint32_t m = valid16(vrow, s0, end);
      int total;
      const int before = seen + block_count_before<NT>(__popc(m), red, &total);
      if (seen + total >= n) {
        if (before < n && before + __popc(m) >= n) found[0] = s0 + nth_bit(m, n - 1 - before) + 1;
        __syncthreads();
        return found[0];
      }
      seen += total;
    }
    return end;
  }
  // the n-th valid slot from end - 1 backward after `seen` in [top, end): 0 if
  // there are fewer
  __device__ __forceinline__ int backward(const uint8_t* vrow, int end, int n, int top, int seen) {
    for (; top > 0; top -= 16 * NT) {
      const int s0 = top - 16 * NT + 16 * (int)threadIdx.x;
      const uint32_t m = s0 >= 0 ? valid16(vrow, s0, end) : 0u;
      const int c = __popc(m);
      int total;
      const int before = block_count_before<NT>(c, red, &total);
      const int after = seen + total - before - c;
      if (seen + total >= n) {
        if (after < n && after + c >= n) found[1] = s0 + nth_bit(m, c - (n - after));
        __syncthreads();
        return found[1];
      }
      seen += total;
    }
    return 0;
  }
};

// What queries see from the one at slot end1 - 1 on (its window begins lowest),
// below slot `end`.
struct WinRange {
  int sink_end;  // e
  int lo;        // lo(end1 - 1)
  int pre;       // listed pages before the window's first page
  int pages;     // listed pages
};

// The pages that hold a valid slot of either range, ascending, to list (shared
// memory, room for all pages below `end`), ready for the whole block. Sinks and
// window that lie in the first step (NT / 8 pages from either end) are listed
// from that step's flags; else the ranges' flags are read again.
template <int NT>
__device__ __forceinline__ WinRange window_pages(const uint8_t* vrow, int end1, int end, int window,
                                                 int sinks, uint16_t* list) {
  __shared__ int red[NT / 64], found[2];
  ValidScan<NT> scan{red, found};
  WinRange r;
  // forward from slot 0, and backward from the end of the last query's page
  const int top = (end + DI_PAGE - 1) / DI_PAGE * DI_PAGE;
  const int f0 = 16 * (int)threadIdx.x, b0 = top - 16 * NT + f0;
  const uint32_t mf = sinks > 0 ? valid16(vrow, f0, end) : 0u;
  const uint32_t mb = b0 >= 0 ? valid16(vrow, b0, end) : 0u;
  // (the window counts from the first query on)
  const int cut = end1 - b0;
  const uint32_t m1 = cut >= 16 ? mb : cut <= 0 ? 0u : mb & ((1u << cut) - 1);
  const int cf = __popc(mf), cb = __popc(m1);
  int total;  // (a step's count is at most 16 NT < 2^16)
  int before = block_count_before<NT>(cf | cb << 16, red, &total);
  const int tf = total & 0xFFFF, tb = total >> 16;
  const int bf = before & 0xFFFF, after = tb - (before >> 16) - cb;
  if (sinks > 0 && bf < sinks && bf + cf >= sinks) found[0] = f0 + nth_bit(mf, sinks - 1 - bf) + 1;
  if (after < window && after + cb >= window) found[1] = b0 + nth_bit(m1, cb - (window - after));
  __syncthreads();
  const int fe = found[0], fl = found[1];
  const bool once = (sinks <= 0 || tf >= sinks || end <= 16 * NT) && (tb >= window || top <= 16 * NT);
  r.sink_end = sinks <= 0 ? 0 : tf >= sinks ? fe : scan.forward(vrow, end, sinks, 16 * NT, tf);
  r.lo = tb >= window ? fl : scan.backward(vrow, end1, window, top - 16 * NT, tb);
  // the sinks' pages below the window's first page, then those from there on
  const int pw = r.lo / DI_PAGE, np = ::min((r.sink_end + DI_PAGE - 1) / DI_PAGE, pw);
  const int sh = threadIdx.x & 56;  // 8 threads a page
  const bool lead = (threadIdx.x & 7) == 0;
  if (once) {
    const int pf = f0 / DI_PAGE, pb = b0 / DI_PAGE;
    const bool inf = ((__ballot(mf != 0) >> sh) & 0xFF) != 0 && lead && pf < np;
    const bool inb = ((__ballot(mb != 0) >> sh) & 0xFF) != 0 && lead && b0 >= 0 && pb >= pw;
    before = block_count_before<NT>((inf ? 1 : 0) | (inb ? 0x10000 : 0), red, &total);
    r.pre = total & 0xFFFF;
    r.pages = r.pre + (total >> 16);
    if (inf) list[before & 0xFFFF] = (uint16_t)pf;
    if (inb) list[r.pre + (before >> 16)] = (uint16_t)pb;
  } else {
    const int cand = np + top / DI_PAGE - pw;
    int n = 0;
    r.pre = 0;
    for (int i0 = 0; i0 < cand; i0 += NT / 8) {
      const int i = i0 + (int)threadIdx.x / 8;
      const int page = i < np ? i : i - np + pw;
      const uint32_t m = i < cand ? valid16(vrow, page * DI_PAGE + 16 * ((int)threadIdx.x & 7), end) : 0u;
      const bool in = ((__ballot(m != 0) >> sh) & 0xFF) != 0 && lead;
      before = block_count_before<NT>(in ? (i < np ? 0x10001 : 1) : 0, red, &total);
      if (in) list[n + (before & 0xFFFF)] = (uint16_t)page;
      n += total & 0xFFFF;
      r.pre += total >> 16;
    }
    r.pages = n;
  }
  __syncthreads();
  r.sink_end = __builtin_amdgcn_readfirstlane(r.sink_end);  // (the same in every lane)
  r.lo = __builtin_amdgcn_readfirstlane(r.lo);
  r.pre = __builtin_amdgcn_readfirstlane(r.pre);
  r.pages = __builtin_amdgcn_readfirstlane(r.pages);
  return r;
}

// First slot of the listed 64-slot tile `it`
__device__ __forceinline__ int listed_slot64(const uint16_t* list, int it) {
  return (int)list[it >> 1] * DI_PAGE + (it & 1) * 64;
}

// lo(t) from the validity masks of the listed tiles: the window-th valid slot
// from t backward.
__device__ __forceinline__ int window_begin(const u64* vmask, const uint16_t* list,
                                            const WinRange& r, int ntiles, int t, int window) {
  const int first = 2 * r.pre;
  int c = 0;  // valid slots from the window's first page to t
  for (int it = first; it < ntiles; ++it) {
    const int d = t - listed_slot64(list, it);
    if (d < 0) break;
    c += __popcll(d >= 63 ? vmask[it] : vmask[it] & (~0ull >> (63 - d)));
  }
  int k = c - window;  // those before the window
  if (k < 0) return 0;
  int it = first;
  u64 m = vmask[it];
  for (int n = __popcll(m); k >= n; n = __popcll(m)) {
    k -= n;
    m = vmask[++it];
  }
  return listed_slot64(list, it) + nth_bit(m, k);
}

}  // namespace
