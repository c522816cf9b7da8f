// How a decode launch over a long cache is cut, and its scratch (host).
#pragma once

#include "../../include/detllm_hip.h"
#include "attn_decode.h"

namespace {

// How a decode over about n slots per row runs: chunk slots per block (a
// multiple of the page), or 0: one block of eight waves per (row, kv head).
//
// Few pairs of (row, kv head) leave CUs idle, so long rows are cut; two launches
// and a denominator that every chunk block sums over the whole row cost more the
// more heads a kv head has. Past 12288 / G slots the one block's scores leave its
// 48 KiB of LDS and every row is cut. us per call, one block /
// cut (accumulating form, 8 kv heads):
//   G = 1: 8 pairs 768 slots 11.0 / 10.2, 64 pairs 768 11.1 / 12.1, 1024 14.1 / 11.5,
//     128 pairs 1536 19.0 / 19.3, 2048 23.5 / 22.5, 4096 44 / 33, 256 pairs 8000
//     113 / 123
//   G = 2: 8 pairs 768 12.0 / 12.9, 1024 13.7 / 13.0, 64 pairs 768 12.2 / 13.2,
//     1024 15.1 / 14.1, 128 pairs 2048 24.9 / 26.1, 3000 33.3 / 32.6, 256 pairs
//     8000 175 / 131
//   G = 4: 32 pairs 1024 16.5 / 18.6, 1536 21.6 / 20.2, 64 pairs 1536 23.4 / 23.8,
//     2048 28.5 / 25.6, 128 pairs 3000 38.0 / 40.8, 4096 89 / 48, 512 pairs 4096
//     165 / 141
//   G = 8: 8 pairs 1536 27.9 / 31.4, 2048 51 / 33, 256 pairs 2048 63 / 61, 3000
//     93 / 83
inline int decode_chunk(int B, int n, int n_q, int n_kv) {
  const int G = n_q / n_kv;
  const i64 pairs = (i64)B * n_kv;
  int from = 12288 / G + 1;
  if (G == 1) from = pairs <= 32 ? 768 : pairs <= 64 ? 960 : pairs <= 128 ? 1920 : from;
  if (G == 2) from = pairs <= 64 ? 960 : pairs <= 128 ? 2816 : from;
  if (G == 4) from = pairs <= 32 ? 1280 : pairs <= 64 ? 1664 : from;
  if (n < from) return 0;
  int chunk = 0, ns = 0;
  if (detllm_attn_split_plan(B, n, n_q, n_kv, &chunk, &ns) != 0 || ns <= 1) return 0;
  return chunk;
}

// Bytes of the split form's scores and chunk maxima: [B][n_q][ns * chunk] and
// [B][n_q][ns] int32 with ns = ceil(S / chunk), 16-byte sizes.
inline i64 split_bytes(int B, int S, int n_q, int chunk, i64* cmax_at) {
  const i64 ns = ((i64)S + chunk - 1) / chunk, rows = (i64)B * n_q;
  *cmax_at = rows * ns * chunk * 4;
  return *cmax_at + (rows * ns * 4 + 15) / 16 * 16;
}
inline int heads_ok(int n_q, int n_kv) {
  if (n_q <= 0 || n_kv <= 0 || n_q % n_kv) return DI_EINVAL;
  const int G = n_q / n_kv;
  return G == 1 || G == 2 || G == 4 || G == 8 ? DI_OK : DI_ENOSYS;
}
inline SplitArgs split_args(const DecodeArgs& d, int B, int chunk, void* work) {
  SplitArgs sa{};
  sa.d = d;
  i64 cmax_at = 0;
  split_bytes(B, d.S, d.n_q, chunk, &cmax_at);
  sa.d.scratch = (int32_t*)work;
  sa.cmax = (int32_t*)((char*)work + cmax_at);
  sa.chunk = chunk;
  sa.ns = (d.S + chunk - 1) / chunk;
  sa.spad = (i64)sa.ns * chunk;
  sa.out_stride = (i64)B * d.n_q * 128;
  sa.add = 1;
  return sa;
}

}  // namespace
