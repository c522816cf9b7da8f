// How a decode launch over a long cache is cut, and its scratch (host).
#pragma once

#include "../../include/detllm_hip.h"
#include "attn_decode.h"

namespace {

// How a decode over about n slots per row runs: chunk slots per block (a
// multiple of the page; 0: one block per (row, kv head)).
inline int decode_chunk(int B, int n, int n_q, int n_kv) {
  const int G = n_q / n_kv;
  const i64 pairs = (i64)B * n_kv;
  const int from = pairs > 128 ? INT32_MAX : G > 4 ? 1537 : G > 2 ? (pairs <= 64 ? 896 : 1536) : pairs <= 64 ? 768 : 1152;
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
inline i64 one_block_bytes(int B, int S, int n_q, int G) {
  const i64 spad = ((i64)S + 15) / 16 * 16;
  return (i64)G * spad * 4 > DECODE_LDS_BYTES ? (i64)B * n_q * spad * 4 : 0;
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
