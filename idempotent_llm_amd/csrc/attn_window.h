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
// forward, 16 flags per thread and step: as many as it is going to scan.
#pragma once

#include "common.h"

using namespace di;

namespace {

// The nonzero flags of slots s0 .. s0 + 15 below `end`, as bits.
__device__ __forceinline__ uint32_t valid16(const uint8_t* vrow, int s0, int end) {
  if (s0 >= end) return 0;
  uint32_t m = 0;
  if (s0 + 16 <= end) {
    uint32_t x[4];
    __builtin_memcpy(x, vrow + s0, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = ((((x[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x[i]) & 0x80808080u) >> 7;
      m |= ((u | u >> 7 | u >> 14 | u >> 21) & 0xFu) << (4 * i);
    }
  } else {
    for (int i = 0; i < end - s0; ++i) m |= (vrow[s0 + i] != 0 ? 1u : 0u) << i;
  }
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
  int incl = c;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(incl, d, 64);
    if (lane >= d) incl += o;
  }
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

// One past the n-th valid slot of [0, end) (`end` if there are fewer; 0 for
// n <= 0). Every thread of the block calls it and gets the result.
template <int NT>
__device__ __forceinline__ int nth_valid_end(const uint8_t* vrow, int end, int n) {
  __shared__ int red[NT / 64], found;
  if (n <= 0) return 0;
  int seen = 0;
  for (int base = 0; base < end; base += 16 * NT) {
    const int s0 = base + 16 * (int)threadIdx.x;
    const uint32_t m = valid16(vrow, s0, end);
    int total;
    const int before = seen + block_count_before<NT>(__popc(m), red, &total);
    if (seen + total >= n) {  // block-uniform
      if (before < n && before + __popc(m) >= n) found = s0 + nth_bit(m, n - 1 - before) + 1;
      __syncthreads();
      return found;
    }
    seen += total;
  }
  return end;
}

// The n-th valid slot from end - 1 backward (0 if there are fewer; n >= 1).
template <int NT>
__device__ __forceinline__ int nth_valid_back(const uint8_t* vrow, int end, int n) {
  __shared__ int red[NT / 64], found;
  int seen = 0;
  for (int top = (end + 15) & ~15; top > 0; top -= 16 * NT) {
    // the step's slots [top - 16 NT, top), none below 0
    const int s0 = top - 16 * NT + 16 * (int)threadIdx.x;
    const uint32_t m = s0 >= 0 ? valid16(vrow, s0, end) : 0u;
    const int c = __popc(m);
    int total;
    const int before = block_count_before<NT>(c, red, &total);
    const int after = seen + total - before - c;
    if (seen + total >= n) {  // block-uniform
      if (after < n && after + c >= n) found = s0 + nth_bit(m, c - (n - after));
      __syncthreads();
      return found;
    }
    seen += total;
  }
  return 0;
}

// The pages that queries see from the one at slot end1 - 1 on (its window
// begins lowest), below slot `end`: pages [0, pre) and those from pre + skip.
struct WinRange {
  int sink_end;  // e
  int lo;        // lo(end1 - 1)
  int pre;       // pages before the gap (0 when there is none)
  int skip;      // pages left out
};
template <int NT>
__device__ __forceinline__ WinRange window_range(const uint8_t* vrow, int end1, int end, int window,
                                                 int sinks) {
  WinRange r;
  r.sink_end = nth_valid_end<NT>(vrow, end, sinks);
  r.lo = nth_valid_back<NT>(vrow, end1, window);
  const int np = (r.sink_end + DI_PAGE - 1) / DI_PAGE, pw = r.lo / DI_PAGE;
  r.pre = pw > np ? np : 0;
  r.skip = pw > np ? pw - np : 0;
  return r;
}

// lo(t) from the validity masks of the listed 64-slot tiles (window_range's
// pages in order): the window-th valid slot from t backward.
__device__ __forceinline__ int window_begin(const u64* vmask, const WinRange& r, int t, int window) {
  const int first = 2 * r.pre, last = (t >> 6) - 2 * r.skip;
  int c = __popcll(vmask[last] & (~0ull >> (63 - (t & 63))));
  for (int it = first; it < last; ++it) c += __popcll(vmask[it]);
  int k = c - window;  // valid slots of the tiles before the window
  if (k < 0) return 0;
  int it = first;
  u64 m = vmask[it];
  for (int n = __popcll(m); k >= n; n = __popcll(m)) {
    k -= n;
    m = vmask[++it];
  }
  return (it + 2 * r.skip) * 64 + nth_bit(m, k);
}

}  // namespace
