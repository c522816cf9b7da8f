// Prefill attention (gfx950): the block of attention.hip's k_attn_prefill and
// of the windowed and accumulating forms of attn_long.hip.
#pragma once

#include <type_traits>

#include "attn_tiles.h"
#include "attn_window.h"

namespace {

struct PrefillArgs {
  const int8_t* q8;      // [B][n_q][T][128]
  const int64_t* tpos;   // [B][n_q][T]
  KVPages kv;
  const uint8_t* valid;  // [B][valid_stride]
  int64_t* out;          // [B][T][n_q * 128]
  int T, S, S_past, n_q, n_kv, B;
  i64 valid_stride;
};
// Of the windowed form (WIN): a query sees the last `window` and the first
// `sinks` valid slots up to its own. Of the accumulating form (ACC): each slot's p
// is added to acc [B][n_kv][acc_stride]. (Apart: the plain kernel's arguments stay
// as they are.)
struct PrefillForm {
  int window, sinks;
  int64_t* acc;
  i64 acc_stride;
};

constexpr int PF_KBYTES = 128 * 128;      // K tile: 128 slot rows of 128 B
constexpr int PF_VBYTES = 128 * 128;      // V^T tile: 128 dim rows of 128 B
constexpr int PF_RING = 64 * 1024;        // 4 K stages, or 2 K+V stages
constexpr int PF_RESIDENT = PF_RING / (PF_KBYTES + PF_VBYTES);  // pages whose K and V fit the ring
constexpr int PF_CSUM = 128 * 4;          // column sums of V (int32 per dim)
constexpr uint32_t PF_SMALL_T = 1u << 23;  // estimated DI-Exp below this tpos
constexpr i64 PF_SMALL_DEN = (i64)1 << 34;  // estimated p below this den

// 16-byte chunk swizzles of the LDS tiles (128-byte rows, physical chunk =
// logical ^ swz). An MFMA operand read takes one chunk column of 16 rows per
// 16 lanes: K rows 16(i/4) + 4 blk + i%4 and V^T rows (dims) 16 j + i for
// i = 0..15. With swz = bits 0, 1 and 4 of the K row (i % 4 and i / 4 % 2)
// and the low 3 bits of the V^T row, both reads run at the full LDS rate of
// 16 bytes per lane (measured on gfx950; an unswizzled read takes 4 times as
// long, swizzles on other row bits twice as long).
__device__ __forceinline__ int pf_kswz(int row) { return (row & 3) | ((row >> 2) & 4); }
__device__ __forceinline__ int pf_vswz(int d) { return d & 7; }

// Per-query constants of the estimated DI-Exp and division (intops.h).
struct PfFast {
  ExpEst E;    // tpos < 2^23
  double kx;   // dexp_sp_const(E)
  int32_t cx;  // t - mx: the score MFMAs of passes 2 and 3 start from it
  DivEst D;    // make_divest(den, 2^14): p = rhad(ex << 14, den), den < 2^34
};

// Four probabilities (slot order = byte order) as the two MFMA operands of
// the hi/lo split p = 128 hi + lo: bytes hi - 64 = (p - 8192) >> 7 in
// [-64, 64] (byte 1 of 2p - 16384) and lo = p & 127.
__device__ __forceinline__ void pf_pack(const uint32_t (&p)[4], int& whi, int& wlo) {
  uint32_t y[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = (p[r] << 1) - 16384u;
  const uint32_t h01 = __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0501u);
  const uint32_t h23 = __builtin_amdgcn_perm(y[3], y[2], 0x05010c0cu);
  const uint32_t l01 = __builtin_amdgcn_perm(p[1], p[0], 0x0c0c0400u);
  const uint32_t l23 = __builtin_amdgcn_perm(p[3], p[2], 0x04000c0cu);
  whi = (int)(h01 | h23);
  wlo = (int)((l01 | l23) & 0x7f7f7f7fu);
}

// Dynamic LDS of a launch over S slots: column sums, tile masks, page ids (and
// the windowed form's page numbers)
inline size_t prefill_lds(i64 S, bool win = false) {
  return PF_CSUM + 8 * (size_t)((S + 63) / 64) + (win ? 6 : 4) * (size_t)((S + 127) / 128);
}

// v[i] of each lane summed over its aligned row of 16 lanes: lane i of the row
// returns the sum of v[i]. Four halving steps; the partner of each step (DPP
// mirror, half mirror, two quad permutations) differs in the lane bit that
// picks the half and agrees in those that picked before.
__device__ __forceinline__ uint32_t row16_scatter_sum(uint32_t (&v)[16]) {
  const int l = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t send = l & 8 ? v[i] : v[i + 8], keep = l & 8 ? v[i + 8] : v[i];
    v[i] = keep + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)send, 0x140, 0xF, 0xF, false);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t send = l & 4 ? v[i] : v[i + 4], keep = l & 4 ? v[i + 4] : v[i];
    v[i] = keep + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)send, 0x141, 0xF, 0xF, false);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t send = l & 2 ? v[i] : v[i + 2], keep = l & 2 ? v[i + 2] : v[i];
    v[i] = keep + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)send, 0x4E, 0xF, 0xF, false);
  }
  const uint32_t send = l & 1 ? v[0] : v[1], keep = l & 1 ? v[1] : v[0];
  return keep + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)send, 0xB1, 0xF, 0xF, false);
}

// A 64-slot key tile in work: its number, which half of its page it is, its
// first slot and (windowed form) its validity mask
struct TileOf {
  int it, hf, s0;
  u64 vm;
};

// The block's work: every query of its tile against the key tiles it sees.
// WIN: the windowed form (window_pages below), ACC: the accumulating form.
template <bool WIN, bool ACC>
__device__ __forceinline__ void prefill_body(const PrefillArgs& a,
                                             const PrefillForm& form = PrefillForm{}) {
  __shared__ __attribute__((aligned(1024))) int8_t ring[PF_RING];
  // PF_CSUM + 8 per 64 slots (tile masks) + 4 per page (page ids)
  extern __shared__ __attribute__((aligned(16))) int8_t dyn[];
  int32_t* const csum_lds = (int32_t*)dyn;
  u64* const vmask = (u64*)(dyn + PF_CSUM);  // per 64-slot key tile
  int32_t* const pages = (int32_t*)(dyn + PF_CSUM + 8 * ((a.S + 63) / 64));
  // Causal work per query tile grows with its index. Pair pi = (b, h, k)
  // (k fastest) stands for the heavy tile nqt - 1 - k and its light partner
  // k. Blocks are dispatched round-robin over the 8 XCDs (XCD = blockIdx % 8);
  // when the pairs split evenly, XCD x takes the contiguous pairs
  // [x pairs/8, (x + 1) pairs/8) — whole heads, so each XCD's L2 holds only
  // its own heads' K and V — heavy tiles first, then the light ones, so the
  // two blocks a CU holds together add up to about the same work. Otherwise
  // the first half of the grid takes the heavy tiles and the second half the
  // light ones. The middle tile of an odd count appears once.
  const int nqt = (a.T + 63) / 64, np = (nqt + 1) / 2;
  const int pairs = np * a.n_q * a.B;
  int half, pi;
  if (pairs % 8 == 0) {
    const int per = pairs / 8, j = blockIdx.x >> 3;
    half = j >= per;
    pi = (blockIdx.x & 7) * per + (j - half * per);
  } else {
    half = blockIdx.x >= pairs;
    pi = blockIdx.x - half * pairs;
  }
  const int kk = pi % np, hb = pi / np;
  if (half && kk == nqt - 1 - kk) return;  // middle tile: done by the first half
  const int qt = half ? kk : nqt - 1 - kk;
  const int h = hb % a.n_q, b = hb / a.n_q;
  const int kvh = h / (a.n_q / a.n_kv);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // wave-uniform
  const int qi = lane & 15, g = lane >> 4;
  const int t = qt * 64 + wave * 16 + qi;  // this lane's query
  const bool tok = t < a.T;
  const i64 qrow = ((i64)b * a.n_q + h) * a.T + (tok ? t : 0);
  v4i qf0 = v4i{0, 0, 0, 0}, qf1 = v4i{0, 0, 0, 0};
  if (tok) {
    qf0 = *(const v4i*)(a.q8 + qrow * 128 + g * 16);
    qf1 = *(const v4i*)(a.q8 + qrow * 128 + 64 + g * 16);
  }
  const i64 tpos = tok ? a.tpos[qrow] : 1;
  const int limit = a.S_past + t;              // last visible slot of this query
  const int wlim = a.S_past + qt * 64 + wave * 16;  // the smallest limit in the wave
  const int kend = min(a.S, a.S_past + qt * 64 + 64);
  const uint8_t* vrow = a.valid + (i64)b * a.valid_stride;
  // The windowed form walks the pages that its queries see (window_pages);
  // tile and page numbers below count that list.
  uint16_t* const list = (uint16_t*)(pages + (a.S + 127) / 128);  // WIN: the pages' numbers
  WinRange wr{};
  int ntiles = (kend + 63) / 64;
  if constexpr (WIN) {
    wr = window_pages<256>(vrow, a.S_past + qt * 64 + 1, kend, form.window, form.sinks, list);
    ntiles = 2 * wr.pages;
    if (wr.pages > 0 && listed_slot64(list, ntiles - 1) >= kend) --ntiles;
    ntiles = __builtin_amdgcn_readfirstlane(ntiles);
  }
  const int ntiles2 = (ntiles + 1) / 2;  // 128-slot tiles = pages
  auto slot64 = [&](int it) {
    if constexpr (WIN) return __builtin_amdgcn_readfirstlane(listed_slot64(list, it));
    return it * 64;
  };
  auto page_of = [&](int i) {
    if constexpr (WIN) return a.kv.page(b, (int)list[i] * DI_PAGE);
    return a.kv.page(b, (i64)i * DI_PAGE);
  };

  // Key tiles of 128 slots reach LDS by direct-to-LDS loads; each tile is
  // processed as two 64-slot halves (the 64-slot tiles `it` of the masks). K:
  // instruction j of wave w covers tile rows 8(4w + j) .. +7, lane l row
  // 8(4w + j) + l/8 at physical chunk l % 8; V^T likewise with dims for rows.
  // A tile is one page; the buffer resources span that page's (kv head) part,
  // 16 KB of K and of V^T. A page that is not mapped gets a zero-length
  // resource, so its loads read 0. Slots past the scanned range in a mapped
  // page read whatever the page holds; such slots are never visible (p = 0:
  // their hi byte -64 and the +64 column-sum term cancel).
  int koffl[4], voffl[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = (wave * 4 + j) * 8 + (lane >> 3);
    koffl[j] = row * 128 + ((lane & 7) ^ pf_kswz(row)) * 16;
    voffl[j] = row * DI_PAGE + ((lane & 7) ^ pf_vswz(row)) * 16;
  }
  auto issue = [&](int page, int8_t* st, bool with_v) {
    const int pg = __builtin_amdgcn_readfirstlane(page);
    const int pgc = pg < 0 ? 0 : pg;
    const int nrec = pg < 0 ? 0 : DI_PAGE * 128;
    const __amdgpu_buffer_rsrc_t krs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)a.kv.krow(pgc, kvh, 0), (short)0, nrec, 0x00020000);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(krs, (lds_ptr_t)(st + (wave * 4 + j) * 1024), 16,
                                               koffl[j], 0, 0, 0);
    if (with_v) {
      const __amdgpu_buffer_rsrc_t vrs = __builtin_amdgcn_make_buffer_rsrc(
          (void*)a.kv.vchan(pgc, kvh, 0), (short)0, nrec, 0x00020000);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            vrs, (lds_ptr_t)(st + PF_KBYTES + (wave * 4 + j) * 1024), 16, voffl[j], 0, 0, 0);
    }
  };
  // A block of few pages keeps all of K and V in the ring for its three
  // passes: its loads are made once, before the mask's, with no barrier per
  // tile (a round trip of each pass's loads is most of a short prompt's
  // launch). The second page's id is waited for behind the first page's loads.
  const bool resident = ntiles2 <= PF_RESIDENT;
  if (resident) {
    for (int i = 0; i < ntiles2; ++i)
      issue(page_of(i), ring + i * (PF_KBYTES + PF_VBYTES), true);
  } else {
    for (int i = tid; i < ntiles2; i += 256) pages[i] = page_of(i);
  }

  // validity bitmask of every key tile (bit s - 64 i of tile i: slot s < S
  // and valid), made once and read by all three passes for the tiles that
  // are not valid in full; nfull = the first tile that is not
  int nf = ntiles;
  for (int i0 = wave; i0 < ntiles; i0 += 16) {
    uint32_t f[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = (!WIN || i0 + 4 * u < ntiles ? slot64(i0 + 4 * u) : 0) + lane;
      const uint32_t v = vrow[s < a.S ? s : 0];  // (the guard below still waits for each)
      f[u] = (i0 + 4 * u < ntiles && s < a.S) ? v : 0u;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + 4 * u;
      const u64 m = __ballot(f[u] != 0);
      if (lane == 0 && i < ntiles) vmask[i] = m;
      if (i < ntiles && m != ~0ull) nf = min(nf, i);
    }
  }
  if (lane == 0) csum_lds[wave] = nf;  // the column-sum area is free until the end
  wait_vmcnt<0>();  // query operands in registers before the ring's loads count; resident tiles here
  __syncthreads();
  const int nfull = min(min(csum_lds[0], csum_lds[1]), min(csum_lds[2], csum_lds[3]));

  // More pages stream through the ring, issued STAGES - 1 tiles ahead, one
  // barrier per tile.
  // one pass over the key tiles; body(it2, stage) runs with tile it2 in LDS.
  // Each wave waits for its own loads of the tile (vmcnt: loads complete in
  // order), then one barrier publishes every wave's part and frees the
  // stage that the next issue overwrites.
  auto pass = [&](auto kv, auto&& body) {
    constexpr bool KV = decltype(kv)::value;
    constexpr int STAGE = KV ? PF_KBYTES + PF_VBYTES : PF_KBYTES;
    constexpr int ST = PF_RING / STAGE;
    constexpr int LPT = KV ? 8 : 4;  // loads per tile per wave
    static_assert(ST >= 2 && ST <= 4 && 2 * LPT < 64, "ring stages");
    if (resident) {
      for (int it2 = 0; it2 < ntiles2; ++it2) body(it2, ring + it2 * (PF_KBYTES + PF_VBYTES));
      return;
    }
    __builtin_amdgcn_s_barrier();  // the previous pass is done with the ring
#pragma unroll
    for (int s = 0; s < ST - 1; ++s)
      if (s < ntiles2) issue(pages[s], ring + s * STAGE, KV);
    for (int it2 = 0; it2 < ntiles2; ++it2) {
      const int after = min(ST - 2, ntiles2 - 1 - it2);  // tiles issued after it2
      if (after >= 2) wait_vmcnt<2 * LPT>();
      else if (after == 1) wait_vmcnt<LPT>();
      else wait_vmcnt<0>();
      __builtin_amdgcn_s_barrier();
      if (it2 + ST - 1 < ntiles2) issue(pages[it2 + ST - 1], ring + ((it2 + ST - 1) % ST) * STAGE, KV);
      body(it2, ring + (it2 % ST) * STAGE);
    }
  };

  // S^T = K . Q^T for one 64-slot half: MFMA block blk takes K rows
  // 16(i/4) + 4 blk + i%4 as its rows i, so lane (qi, g) receives the scores
  // of query qi for the 16 consecutive slots 16 g + 4 blk + r (blk, r < 4):
  // st[blk][r]. Those are also the 16 bytes of its P operand for P.V, in
  // the slot order of the V^T rows.
  const int kr = 16 * (qi >> 2) + (qi & 3);
  const int koff0 = kr * 128 + ((g ^ pf_kswz(kr)) << 4);
  const int koff1 = kr * 128 + (((g + 4) ^ pf_kswz(kr)) << 4);
  auto load_k = [&](const int8_t* st_k, v4i (&kf)[8]) {
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) {
      kf[2 * blk] = *(const v4i*)(st_k + koff0 + blk * 512);
      kf[2 * blk + 1] = *(const v4i*)(st_k + koff1 + blk * 512);
    }
  };
  // both halves' K operands read at once (one LDS latency), then their
  // score MFMAs from accumulator z: the first 64 dims of all 8 blocks, then
  // the second 64 — the
  // two MFMAs of a block are 8 issues apart, so none waits on the previous
  // one's result — overlapping the first half's VALU work; then
  // fn(st, it, half) per half that holds key slots
  auto halves = [&](const int8_t* stg, int it2, const v4i z, auto&& fn) {
    v4i ka[8], kb[8], sa[4], sb[4];
    TileOf ta{2 * it2, 0, it2 * 128, 0}, tb{2 * it2 + 1, 1, it2 * 128 + 64, 0};
    if constexpr (WIN) {  // (read beside the K operands, kept as scalars)
      const int s0 = __builtin_amdgcn_readfirstlane((int)list[it2] * DI_PAGE);
      const v4i m = *(const v4i*)(vmask + 2 * it2);
      auto word = [&](int i) { return (u64)(uint32_t)__builtin_amdgcn_readfirstlane(m[i]); };
      ta.s0 = s0;
      tb.s0 = s0 + 64;
      ta.vm = word(0) | word(1) << 32;
      tb.vm = word(2) | word(3) << 32;
    }
    load_k(stg, ka);
    load_k(stg + 64 * 128, kb);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) sa[blk] = mfma16(ka[2 * blk], qf0, z);
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) sb[blk] = mfma16(kb[2 * blk], qf0, z);
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) sa[blk] = mfma16(ka[2 * blk + 1], qf1, sa[blk]);
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) sb[blk] = mfma16(kb[2 * blk + 1], qf1, sb[blk]);
    __builtin_amdgcn_sched_barrier(0);
    fn(sa, ta);
    if (2 * it2 + 1 < ntiles) fn(sb, tb);
  };
  // the windowed form: where this lane's window begins, and the extremes of
  // that over the wave
  int wlo = 0, wlo_min = 0, wlo_max = 0;
  if constexpr (WIN) {
    wlo = window_begin(vmask, list, wr, ntiles, a.S_past + (tok ? t : a.T - 1), form.window);
    wlo_min = __builtin_amdgcn_readfirstlane(wlo);
    wlo_max = __builtin_amdgcn_readlane(wlo, 15);
  }
  // the validity mask of a tile
  auto mask = [&](const TileOf& t) { return WIN ? t.vm : vmask[t.it]; };
  // the tile is visible in full to every query of the wave (wave-uniform)
  auto full_tile = [&](const TileOf& t) {
    if constexpr (WIN)
      return t.vm == ~0ull && t.s0 + 63 <= wlim && (t.s0 >= wlo_max || t.s0 + 63 < wr.sink_end);
    return t.it < nfull && t.it * 64 + 63 <= wlim;
  };
  // no query of the wave sees any of its slots (wave-uniform; the windowed form
  // only: a page's other half, the other waves' window ends)
  auto dead_tile = [&](const TileOf& t) {
    return WIN && (t.s0 > wlim + 15 || (t.s0 + 63 < wlo_min && t.s0 >= wr.sink_end));
  };
  // this lane's visibility bits: bit 4 blk + r for slot 16 g + 4 blk + r
  auto lane_bits = [&](const TileOf& t) -> uint32_t {
    // (the plain form counts from the tile's number: from t.s0 it took 2 % longer at 8
    // prompts of 110 tokens, 0.8 % at 512 behind 3000)
    const int s0 = (WIN ? t.s0 : t.it * 64) + 16 * g;
    // last visible offset in the lane's 16
    const int e = WIN ? limit - s0 : limit - t.it * 64 - 16 * g;
    uint32_t cb = e >= 15 ? 0xFFFFu : (e < 0 ? 0u : (2u << e) - 1u);
    if constexpr (WIN) {
      const int f = wlo - s0, z = wr.sink_end - s0;
      const uint32_t wb = f <= 0 ? 0xFFFFu : (f >= 16 ? 0u : 0xFFFFu << f);
      const uint32_t sb = z >= 16 ? 0xFFFFu : (z <= 0 ? 0u : (1u << z) - 1u);
      cb &= wb | sb;
    }
    return (uint32_t)(mask(t) >> (16 * g)) & cb;
  };

  // ---- pass 1: row max over visible slots (scores are int32)
  int mx = INT32_MIN;
  pass(std::false_type{}, [&](int it2, const int8_t* stg) { halves(stg, it2, v4i{0, 0, 0, 0}, [&](const v4i (&st)[4], const TileOf& t) {
    if (dead_tile(t)) return;
    if (full_tile(t)) {
#pragma unroll
      for (int blk = 0; blk < 4; ++blk)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = max(mx, st[blk][r]);
    } else {
      const uint32_t bits = lane_bits(t);
#pragma unroll
      for (int blk = 0; blk < 4; ++blk)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if ((bits >> (4 * blk + r)) & 1u) mx = max(mx, st[blk][r]);
    }
  }); });
  mx = max(mx, __shfl_xor(mx, 16));
  mx = max(mx, __shfl_xor(mx, 32));
  if (mx == INT32_MIN) mx = 0;  // no visible slot: max := 0, every p = 0

  // ---- pass 2: denominator. The estimated DI-Exp runs when every query of
  // the wave has tpos < 2^23 (then every exp is below 2^23 and 16 of them sum
  // in 32 bits); otherwise the general 64-bit form. Masked slots enter the
  // estimate as st = mx (a defined conversion) and are then dropped.
  const bool fexp = __ballot(tpos >= (i64)PF_SMALL_T) == 0;
  PfFast F;
  F.E = make_expest(tpos);
  F.kx = dexp_sp_const(F.E);
  F.cx = (int32_t)(F.E.t - (uint32_t)mx);
  // fast path: scores arrive as st + t - mx; the general path subtracts it
  const int32_t soff = fexp ? F.cx : 0;
  const v4i cinit = v4i{soff, soff, soff, soff};
  const ExpR Et = make_exp(tpos);
  i64 den = 0;
  pass(std::false_type{}, [&](int it2, const int8_t* stg) { halves(stg, it2, cinit, [&](const v4i (&st)[4], const TileOf& t) {
    if (dead_tile(t)) return;
    if (fexp && full_tile(t)) {
      uint32_t sum = 0;
#pragma unroll
      for (int blk = 0; blk < 4; ++blk)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += dexp_est_sp(st[blk][r], F.E, F.kx);
      den += sum;
      return;
    }
    const uint32_t bits = lane_bits(t);
    if (fexp) {
      uint32_t sum = 0;
#pragma unroll
      for (int blk = 0; blk < 4; ++blk)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool vis = (bits >> (4 * blk + r)) & 1u;
          const uint32_t e = dexp_est_sp(vis ? st[blk][r] : (int32_t)F.E.t, F.E, F.kx);
          sum += vis ? e : 0u;
        }
      den += sum;
    } else {
#pragma unroll
      for (int blk = 0; blk < 4; ++blk)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if ((bits >> (4 * blk + r)) & 1u)
            den = wadd(den, di_exp_neg((u64)(uint32_t)(mx - (st[blk][r] - soff)), Et));
    }
  }); });
  den = imax(group4_sum(den), 1);
  const bool fdiv = fexp && __ballot(den >= PF_SMALL_DEN) == 0;
  F.D = make_divest(den, 16384.0);
  const Recip Rd = make_recip(den);

  // ---- pass 3: p, then P.V on MFMA with the hi/lo split; wave w also sums
  // the V^T rows of dims 32w .. 32w + 31 (an all-ones A operand) for the
  // +64 correction of the hi bytes
  bool counts = false;  // ACC: a query at a slot that is not valid adds nothing
  int64_t* accrow = nullptr;
  if constexpr (ACC) {
    counts = tok && vrow[tok ? a.S_past + t : 0] != 0;
    accrow = form.acc + ((i64)b * a.n_kv + kvh) * form.acc_stride;
  }
  v4i ohi[8], olo[8], ocs[2];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    ohi[j] = v4i{0, 0, 0, 0};
    olo[j] = v4i{0, 0, 0, 0};
  }
  ocs[0] = ocs[1] = v4i{0, 0, 0, 0};
  const v4i ones = v4i{0x01010101, 0x01010101, 0x01010101, 0x01010101};
  // V^T operand of half `hf`: dim 16 j + qi, slots 64 hf + 16 g .. + 15
  // (the swizzle of dim 16 j + qi does not depend on j)
  int voff[2];
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) voff[hf] = PF_KBYTES + qi * 128 + (((4 * hf + g) ^ pf_vswz(qi)) << 4);
  pass(std::true_type{}, [&](int it2, const int8_t* stg) { halves(stg, it2, cinit, [&](const v4i (&st)[4], const TileOf& t) {
    const int hf = t.hf;
    v4i vf[8], vc[2];
#pragma unroll
    for (int j = 0; j < 8; ++j) vf[j] = *(const v4i*)(stg + voff[hf] + j * 2048);
#pragma unroll
    for (int c = 0; c < 2; ++c) vc[c] = *(const v4i*)(stg + voff[hf] + (2 * wave + c) * 2048);
    __builtin_amdgcn_sched_barrier(0);
    v4i phi, plo;
    if (dead_tile(t)) {
      // p = 0: bytes -64 and 0 (the tile's column sums count for the block)
      const int m64 = (int)0xC0C0C0C0u;
      phi = v4i{m64, m64, m64, m64};
#pragma unroll
      for (int j = 0; j < 8; ++j) ohi[j] = mfma16(phi, vf[j], ohi[j]);
#pragma unroll
      for (int c = 0; c < 2; ++c) ocs[c] = mfma16(ones, vc[c], ocs[c]);
      return;
    }
    const bool full = full_tile(t);
    uint32_t bits = 0xFFFFu;
    if (!full) bits = lane_bits(t);
    uint32_t pw[ACC ? 16 : 1];  // (the accumulating form keeps the p)
    auto put = [&](int blk, const uint32_t (&p)[4]) {
      int whi, wlo;
      pf_pack(p, whi, wlo);
      phi[blk] = whi;
      plo[blk] = wlo;
      if constexpr (ACC) {
#pragma unroll
        for (int r = 0; r < 4; ++r) pw[4 * blk + r] = counts ? p[r] : 0u;
      }
    };
    if (fdiv && full) {
#pragma unroll
      for (int blk = 0; blk < 4; ++blk) {
        uint32_t p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = rhad_est((double)dexp_est_sp(st[blk][r], F.E, F.kx), F.D);
        put(blk, p);
      }
    } else if (fdiv) {
#pragma unroll
      for (int blk = 0; blk < 4; ++blk) {
        uint32_t p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool vis = (bits >> (4 * blk + r)) & 1u;
          const uint32_t e = dexp_est_sp(vis ? st[blk][r] : (int32_t)F.E.t, F.E, F.kx);
          p[r] = rhad_est((double)(vis ? e : 0u), F.D);
        }
        put(blk, p);
      }
    } else {
#pragma unroll
      for (int blk = 0; blk < 4; ++blk) {
        uint32_t p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          i64 pv = 0;
          if ((bits >> (4 * blk + r)) & 1u) {
            const i64 ex = di_exp_neg((u64)(uint32_t)(mx - (st[blk][r] - soff)), Et);
            pv = to_i32(rhad_r(shl(ex, 14), Rd));
          }
          p[r] = (uint32_t)pv;
        }
        put(blk, p);
      }
    }
    if constexpr (ACC) {
      // the 16 queries' sums: lane (qi, g) that of slot 16 g + qi
      const uint32_t sum = row16_scatter_sum(pw);
      if (sum != 0)
        atomicAdd((unsigned long long*)&accrow[t.s0 + 16 * g + qi], (unsigned long long)sum);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ohi[j] = mfma16(phi, vf[j], ohi[j]);
      olo[j] = mfma16(plo, vf[j], olo[j]);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) ocs[c] = mfma16(ones, vc[c], ocs[c]);
  }); });
  // column sums: every row of ocs[c] holds sum_s v[s][32 wave + 16 c + qi]
  if (resident) __syncthreads();  // every wave has read its nfull there (no barrier since)
  if (g == 0) {
    csum_lds[32 * wave + qi] = ocs[0][0];
    csum_lds[32 * wave + 16 + qi] = ocs[1][0];
  }
  __syncthreads();
  // write: lane holds O[query 4g + r][d = 16j + qi]
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const i64 cs = csum_lds[16 * j + qi];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int tq = qt * 64 + wave * 16 + g * 4 + r;
      if (tq < a.T) {
        const i64 v = (i64)ohi[j][r] * 128 + cs * 8192 + (i64)olo[j][r];
        a.out[((i64)b * a.T + tq) * (a.n_q * 128) + h * 128 + j * 16 + qi] = v;
      }
    }
  }
}

}  // namespace
