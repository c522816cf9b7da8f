// What the attention kernels share (gfx950).
#pragma once

#include "common.h"

using namespace di;

typedef int v4i __attribute__((ext_vector_type(4)));

namespace {

__device__ __forceinline__ v4i mfma16(v4i a, v4i b, v4i c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// The paged cache arguments of every entry: kpool / vpool the layer's page
// pools (common.h KVPages), table [B][width] int32 page ids (-1: not mapped); a
// row holds width * 128 slots.
inline bool kv_ok(const int8_t* kpool, const int8_t* vpool, const int32_t* table, int width) {
  return kpool && vpool && table && width > 0 && width <= (1 << 24);
}

}  // namespace
