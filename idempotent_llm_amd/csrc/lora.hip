// Low-rank adapters beside a shared projection (gfx950): every token row its own
// adapter or none.
//
// Of a token row with adapter a: u = A_a x (int32, |u| <= 2^14 K), the row shift
// h = max(ilog2(max |u|) - 12, 0), w = rshift_round(u, h), |w| <= 2^13 (the rule of
// requant_i32_common at 13 bits), v = B_a w (int32, |v| <= rank 2^20), and the
// product's column c gets rshift_round(v[c] bm_a[c], bk_a - h) (a left shift by
// h - bk_a where that is positive, 0 from shifts of 64 on; int64, then added as int32).
//
// A block takes up to 16 consecutive token rows and up to four times 256 columns. Its
// adapters are the distinct ones of those rows, one after another: u on i8 MFMA with
// K split over the four waves, the other adapters' rows dropped as the sums meet in
// LDS; then w as two int8 operands (w = 256 H + L - 128, bytes H and L ^ 0x80), rows
// of other adapters zero, so the adapters' products add up in one accumulator. Each
// group of column blocks makes u for itself. What bounds it: at
// few rows one chain of loads (adapters, x and A, B, then the product's own
// columns; 8 rows of K 1024, 4096 columns and rank 16: 6 us), at many the product's
// columns read and written once more (2000 rows of K 1024, 4096 columns and rank 32:
// 27 us, 65 MB in 14 us of them).
#include "attn_tiles.h"

#include "../../include/detllm_hip.h"

namespace {

constexpr int LR_MAX_RANK = 128;
constexpr int LR_COLS = 256;
constexpr int LR_MAX_ROWS = 65535 * 16;  // blocks of a grid's second dimension

struct LoraArgs {
  int32_t* P;         // [N][C]
  const int8_t* x8;   // [N][K]
  const int8_t* a8;   // [n_ad][rank][K]
  const int8_t* b8;   // [n_ad][C][rank]
  const int64_t* bm;  // [n_ad][C]
  const int64_t* bk;  // [n_ad]
  const int32_t* adapter;  // [N]
  int N, K, C, rank, n_ad;
  int tm;      // token rows a block, at most 16
  int groups;  // of 256 columns a block
};

template <int NR>  // 16-wide steps of the rank, at least rank / 16
__global__ __launch_bounds__(256) void k_lora(LoraArgs a) {
  keep_hidden_args();
  constexpr int RK = 16 * NR;
  constexpr int RP = (RK + 63) / 64 * 64;  // the second product's K, in whole steps
  __shared__ int32_t u_lds[16][RK];
  __shared__ __attribute__((aligned(16))) int8_t w_lds[2][16][RP];
  __shared__ int h_lds[16];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r0 = blockIdx.y * a.tm, rows = ::min(a.tm, a.N - r0);
  int ad = l16 < rows ? a.adapter[r0 + l16] : -1;
  ad = ad >= 0 && ad < a.n_ad ? ad : -1;
  if (__ballot(ad >= 0) == 0) return;
  for (int i = tid; i < 16 * RK; i += 256) ((int32_t*)u_lds)[i] = 0;
  for (int i = tid; i < 2 * 16 * RP / 4; i += 256) ((int32_t*)w_lds)[i] = 0;
  __syncthreads();
  const v4i z = v4i{0, 0, 0, 0};
  const int8_t* xrow = a.x8 + (i64)(r0 + (l16 < rows ? l16 : 0)) * a.K;
  const int ksteps = (a.K + 63) / 64;
  // u of each adapter's rows
  for (u64 left = __ballot(ad >= 0 && grp == 0); left != 0;) {
    const int cur = __builtin_amdgcn_readlane(ad, __ffsll((unsigned long long)left) - 1);
    left &= ~__ballot(ad == cur);
    v4i acc[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) acc[n] = z;
    const int8_t* arow = a.a8 + ((i64)cur * a.rank + l16) * a.K;
    for (int k0 = wave; k0 < ksteps; k0 += 16) {
      v4i x[4], w[4][NR];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int k = (k0 + 4 * q) * 64 + 16 * grp;
        const bool in = k < a.K;  // (K is a multiple of 16)
        const int kc = in ? k : 0;
        const v4i xv = *(const v4i*)(xrow + kc);
        x[q] = in ? xv : z;
#pragma unroll
        for (int n = 0; n < NR; ++n) w[q][n] = *(const v4i*)(arow + (i64)n * 16 * a.K + kc);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int n = 0; n < NR; ++n) acc[n] = mfma16(x[q], w[q][n], acc[n]);
    }
    // lane (grp, l16): token rows 4 grp + r, rank 16 n + l16
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool mine = __shfl(ad, 4 * grp + r) == cur;
#pragma unroll
      for (int n = 0; n < NR; ++n)
        if (mine) atomicAdd(&u_lds[4 * grp + r][16 * n + l16], acc[n][r]);
    }
  }
  __syncthreads();
  {  // 16 threads a token row: its shift, its bytes
    const int row = tid >> 4, j = tid & 15;
    int u[NR], m = 0;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      u[n] = u_lds[row][16 * n + j];
      m = ::max(m, u[n] < 0 ? -u[n] : u[n]);
    }
    m = ::max(m, __shfl_xor(m, 1));
    m = ::max(m, __shfl_xor(m, 2));
    m = ::max(m, __shfl_xor(m, 4));
    m = ::max(m, __shfl_xor(m, 8));
    const int h = ::max(31 - __clz(::max(m, 1)) - 12, 0);
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int w = (h > 0 ? (u[n] + (1 << (h - 1))) >> h : u[n]) + 128;
      w_lds[0][row][16 * n + j] = (int8_t)(w >> 8);
      w_lds[1][row][16 * n + j] = (int8_t)((w & 255) ^ 128);
    }
    if (j == 0) h_lds[row] = h;
  }
  __syncthreads();
  // rows 4 grp + r of the lane
  int h[4], ar[4];
  i64 bk[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    ar[r] = __shfl(ad, 4 * grp + r);
    h[r] = h_lds[4 * grp + r];
    bk[r] = a.bk[::max(ar[r], 0)];
  }
  // (most tiles of a prompt have one adapter: its scales are loaded once)
  const u64 with = __ballot(ad >= 0 && grp == 0);
  const int first = __builtin_amdgcn_readlane(ad, __ffsll((unsigned long long)with) - 1);
  const bool single = __ballot(ad >= 0 && ad != first) == 0;
  for (int cg = 0; cg < a.groups; ++cg) {
    // v of the wave's 64 columns
    const int c0 = (blockIdx.x * a.groups + cg) * LR_COLS + wave * 64;
    if (c0 >= a.C) return;
    auto col = [&](int n) { return ::min(c0 + 16 * n + l16, a.C - 1); };
    // the product's own values load first
    int p[4][4];
    i64 m[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 4 * grp + r;
        p[r][n] = a.P[(i64)(r0 + (row < rows ? row : 0)) * a.C + col(n)];
      }
#pragma unroll
    for (int n = 0; n < 4; ++n) m[0][n] = a.bm[(i64)(single ? first : ::max(ar[0], 0)) * a.C + col(n)];
    if (single) {
#pragma unroll
      for (int r = 1; r < 4; ++r)
#pragma unroll
        for (int n = 0; n < 4; ++n) m[r][n] = m[0][n];
    } else {
#pragma unroll
      for (int r = 1; r < 4; ++r)
#pragma unroll
        for (int n = 0; n < 4; ++n) m[r][n] = a.bm[(i64)::max(ar[r], 0) * a.C + col(n)];
    }
    v4i hi[4], lo[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) hi[n] = lo[n] = z;
    for (u64 left = with; left != 0;) {
      const int cur = __builtin_amdgcn_readlane(ad, __ffsll((unsigned long long)left) - 1);
      left &= ~__ballot(ad == cur);
#pragma unroll
      for (int k = 0; k < RP; k += 64) {
        const int at = k + 16 * grp;
        const bool in = at < a.rank;
        v4i wh = z, wl = z;
        if (ad == cur && in) {
          wh = *(const v4i*)&w_lds[0][l16][at];
          wl = *(const v4i*)&w_lds[1][l16][at];
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const v4i b = *(const v4i*)(a.b8 + ((i64)cur * a.C + col(n)) * a.rank + (in ? at : 0));
          hi[n] = mfma16(wh, b, hi[n]);
          lo[n] = mfma16(wl, b, lo[n]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 4 * grp + r;
      const i64 s = wsub(bk[r], h[r]);
      // (shifts from 64 on leave nothing; rshift_round's half would wrap)
      const bool adds = row < rows && ar[r] >= 0 && s < 64;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int c = c0 + 16 * n + l16;
        const i64 t = wmul((i64)hi[n][r] * 256 + lo[n][r], m[r][n]);
        const i64 d = s > 0 ? rshift_round(t, s) : shl(t, wneg(s));
        if (adds && c < a.C)
          a.P[(i64)(r0 + row) * a.C + c] = (int32_t)((uint32_t)p[r][n] + (uint32_t)(u64)d);
      }
    }
  }
}

}  // namespace

extern "C" {

int detllm_lora_add(int32_t* P, const int8_t* x8, const int8_t* a8, const int8_t* b8,
                    const int64_t* bm, const int64_t* bk, const int32_t* adapter, int N, int K,
                    int C, int rank, int n_ad, hipStream_t s) {
  if (N < 0 || K < 16 || K % 16 || C < 1 || rank < 16 || rank % 16 || n_ad < 1) return DI_EINVAL;
  if (K > 65536 || rank > LR_MAX_RANK || C > (1 << 24) || N > LR_MAX_ROWS) return DI_ERANGE;
  if (N == 0) return DI_OK;
  if (!P || !x8 || !a8 || !b8 || !bm || !bk || !adapter) return DI_EINVAL;
  // (16-byte loads)
  if ((((uintptr_t)x8 | (uintptr_t)a8 | (uintptr_t)b8) & 15) != 0) return DI_EINVAL;
  LoraArgs a{P, x8, a8, b8, bm, bk, adapter, N, K, C, rank, n_ad, 16, 1};
  const int cb = (C + LR_COLS - 1) / LR_COLS;
  // fewer rows a block while the blocks are few: a block's adapters run one after another
  // (rows a block 1, 4, 16; K 1024, 4096 columns, rank 16, eight adapters row by row: 8
  // rows 6.0, 9.3, 13.6 us, 64 rows 9.2, 9.6, 15.1, 200 rows 24, 17, 15)
  while (a.tm > 1 && (i64)cb * ((N + a.tm - 1) / a.tm) < 192) a.tm /= 2;
  // and more columns while they are many: u is made again by every block of the same
  // rows (the 2000 rows above: 34 us at 1 group, 15 of them for u, 29.5 at 2, 27 at 4)
  while (a.groups < 4 && (i64)cb * ((N + a.tm - 1) / a.tm) > 512 * a.groups) a.groups *= 2;
  const dim3 grid((cb + a.groups - 1) / a.groups, (N + a.tm - 1) / a.tm);
  switch ((rank + 15) / 16) {
    case 1: hipLaunchKernelGGL(k_lora<1>, grid, dim3(256), 0, s, a); break;
    case 2: hipLaunchKernelGGL(k_lora<2>, grid, dim3(256), 0, s, a); break;
    case 3: hipLaunchKernelGGL(k_lora<3>, grid, dim3(256), 0, s, a); break;
    case 4: hipLaunchKernelGGL(k_lora<4>, grid, dim3(256), 0, s, a); break;
    case 5: hipLaunchKernelGGL(k_lora<5>, grid, dim3(256), 0, s, a); break;
    case 6: hipLaunchKernelGGL(k_lora<6>, grid, dim3(256), 0, s, a); break;
    case 7: hipLaunchKernelGGL(k_lora<7>, grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL(k_lora<8>, grid, dim3(256), 0, s, a); break;
  }
  DI_LAUNCH_CHECK();
  return DI_OK;
}

}  // extern "C"
