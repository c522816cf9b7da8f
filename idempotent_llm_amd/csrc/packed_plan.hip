// The bookkeeping of a packed step on the device (gfx950): from the rows' filled
// and new tokens the token rows' offsets, positions and slots, and the pages that
// the rows need or give back.
//
// What bounds it is latency: a few words a row and 20 bytes a token. One block
// scans the rows (their new tokens, surplus and missing pages, three prefix sums
// at once), moves the pages, element by element over the sums so that the loads
// of different rows run side by side, and, where the tokens are few, writes them
// too: one launch. More tokens are a second launch of many blocks, which read the
// rows' sums from scratch.
#include "common.h"

#include "../../include/detllm_hip.h"

using namespace di;

namespace {

constexpr int PLAN_NT = 1024;
constexpr int PLAN_MAX_ROWS = 2048;   // 16 bytes of LDS each
constexpr int PLAN_MAX_WIDTH = 1024;  // 131072 slots
constexpr int PLAN_MAX_SLOTS = 131071;
// Token rows that the one block writes itself (64 rows; us, one launch / two: 8 tokens
// 3.3 / 4.7, 1024 5.5 / 7.1, 2048 6.4 / 7.1, 4096 8.0 / 7.1, 16384 18 / 7.2)
constexpr int PLAN_ONE = 2048;

struct PlanArgs {
  int32_t* table;  // [B][width]
  int32_t* free;   // [cap]
  int32_t* n_free;
  const int32_t* past;
  const int32_t* fresh;
  int32_t* cu;   // [B + 1]
  int32_t* row;  // [N]
  int64_t* pos;
  int64_t* slot;
  int4* rows;  // scratch [B + 1] (two launches)
  int32_t* err;
  int width, cap, B, N;
};

// A row: .x its first token row, .y pages it has | pages it needs << 16, .z and .w
// missing and surplus pages of the rows before it. Behind the last: the sums, and
// .y the length of the free list with the surplus, -1 - that where the missing
// ones do not fit.
struct PlanRow {
  int cu, have, need, miss, spare;
};
__device__ __forceinline__ PlanRow plan_row(int4 v) {
  return PlanRow{v.x, v.y & 0xFFFF, v.y >> 16, v.z, v.w};
}

// The number of leading mapped pages of a row. A running row has its filled
// slots' pages, no more: two loads, side by side, tell. Another is searched 16
// ways (mapped pages come first).
__device__ __forceinline__ int plan_have(const int32_t* t, int width, int past) {
  const int g = ::min((past + DI_PAGE - 1) / DI_PAGE, width);
  const int a = t[g > 0 ? g - 1 : 0], b = t[g < width ? g : width - 1];
  if ((g == 0 || a >= 0) && (g == width || b < 0)) return g;
  int lo = 0, hi = width;  // pages before lo are there, from hi on not
  while (lo < hi) {
    const int step = (hi - lo + 15) / 16;
    int v[16], n = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = t[::min(lo + k * step, width - 1)];
#pragma unroll
    for (int k = 0; k < 16; ++k) n += lo + k * step < hi && v[k] >= 0 && n == k ? 1 : 0;
    if (n == 0) return lo;
    const int last = lo + (n - 1) * step;
    hi = ::min(hi, last + step);
    lo = last + 1;
  }
  return lo;
}

__device__ __forceinline__ int scan64(int v) {  // inclusive, over the wave
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
}

// The last row b < B whose key(b) is at most x (key ascending, key(0) <= x): the
// row that holds element x
template <class Key>
__device__ __forceinline__ int row_of(int B, int x, Key&& key) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (key(mid) <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Token row i
__device__ __forceinline__ void plan_token(const PlanArgs& a, const int4* rows, int i) {
  int r = -1;
  i64 pos = 0, slot = -1;
  if (i < rows[a.B].x) {
    r = row_of(a.B, i, [&](int b) { return rows[b].x; });
    const PlanRow p = plan_row(rows[r]);
    const int n1 = rows[a.B].y;
    const int s = a.past[r] + i - p.cu, j = s / DI_PAGE;
    // (a page that this step maps comes from the free list: its place in the table
    // may not be written yet)
    int page = -1;
    if (j < p.have) page = a.table[(i64)r * a.width + j];
    else if (n1 >= 0) page = a.free[n1 - 1 - (p.miss + j - p.have)];
    pos = s;
    if (page >= 0) slot = (i64)page * DI_PAGE + s % DI_PAGE;
  }
  a.row[i] = r;
  a.pos[i] = pos;
  a.slot[i] = slot;
}

template <bool ONE>
__global__ __launch_bounds__(PLAN_NT) void k_plan_rows(PlanArgs a) {
  keep_hidden_args();
  extern __shared__ __attribute__((aligned(16))) int4 rows[];  // [B + 1]
  __shared__ int part[3][PLAN_NT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n0 = ::min(::max(a.n_free[0], 0), a.cap);
  int total[3] = {0, 0, 0};  // new tokens, missing and surplus pages so far
  int bad = 0;
  for (int b0 = 0; b0 < a.B; b0 += PLAN_NT) {
    const int b = b0 + tid;
    int v[3] = {0, 0, 0}, have = 0, need = 0;
    if (b < a.B) {
      const int past = a.past[b], fresh = a.fresh[b];
      const i64 end = (i64)past + fresh;
      const bool ok = past >= 0 && fresh >= 0 && end <= imin((i64)a.width * DI_PAGE, PLAN_MAX_SLOTS);
      have = plan_have(a.table + (i64)b * a.width, a.width, ok ? past : 0);
      // a row outside the table keeps its pages and gets no tokens
      need = ok ? (int)((end + DI_PAGE - 1) / DI_PAGE) : have;
      v[0] = ok ? fresh : 0;
      v[1] = ::max(need - have, 0);
      v[2] = ::max(have - need, 0);
      bad |= ok ? 0 : DI_ERR_SLOTS;
    }
    int in[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      in[k] = scan64(v[k]);
      if (lane == 63) part[k][wave] = in[k];
    }
    __syncthreads();
    int before[3] = {total[0], total[1], total[2]};
#pragma unroll
    for (int w = 0; w < PLAN_NT / 64; ++w)
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const int x = part[k][w];
        before[k] += w < wave ? x : 0;
        total[k] += x;
      }
    if (b < a.B)
      rows[b] = int4{before[0] + in[0] - v[0], have | need << 16, before[1] + in[1] - v[1],
                     before[2] + in[2] - v[2]};
    __syncthreads();
  }
  const int n1 = ::min(n0 + total[2], a.cap);
  const bool fits = total[1] <= n1;
  // token rows past the step's end are not made (and a free list with no room
  // for what comes back loses it)
  if (total[0] > a.N) bad |= DI_ERR_SLOTS;
  if (!fits || n0 + total[2] > a.cap) bad |= DI_ERR_PAGES;
  if (tid == 0) {
    rows[a.B] = int4{total[0], fits ? n1 : -1 - n1, total[1], total[2]};
    a.n_free[0] = fits ? n1 - total[1] : n1;
  }
  if (bad && a.err) atomicOr(a.err, bad);
  __syncthreads();
  for (int e = tid; e < total[2]; e += PLAN_NT) {
    const int b = row_of(a.B, e, [&](int i) { return rows[i].w; });
    const PlanRow p = plan_row(rows[b]);
    int32_t* t = a.table + (i64)b * a.width + p.need + (e - p.spare);
    if (n0 + e < a.cap) a.free[n0 + e] = *t;
    *t = -1;
  }
  __syncthreads();
  if (fits)
    for (int e = tid; e < total[1]; e += PLAN_NT) {
      const int b = row_of(a.B, e, [&](int i) { return rows[i].z; });
      const PlanRow p = plan_row(rows[b]);
      a.table[(i64)b * a.width + p.have + (e - p.miss)] = a.free[n1 - 1 - e];
    }
  for (int b = tid; b <= a.B; b += PLAN_NT) {
    a.cu[b] = rows[b].x;
    if (!ONE) a.rows[b] = rows[b];
  }
  if (ONE)
    for (int i = tid; i < a.N; i += PLAN_NT) plan_token(a, rows, i);
}

__global__ __launch_bounds__(256) void k_plan_tokens(PlanArgs a) {
  keep_hidden_args();
  extern __shared__ __attribute__((aligned(16))) int4 rows[];
  for (int b = threadIdx.x; b <= a.B; b += 256) rows[b] = a.rows[b];
  __syncthreads();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < a.N) plan_token(a, rows, i);
}

}  // namespace

extern "C" {

int detllm_packed_plan_work(int B, int N, int64_t* bytes) {
  if (!bytes || B < 1 || N < 0) return DI_EINVAL;
  if (B > PLAN_MAX_ROWS) return DI_ERANGE;
  *bytes = N > PLAN_ONE ? (int64_t)(B + 1) * 16 : 0;
  return DI_OK;
}

int detllm_packed_plan(int32_t* table, int width, int32_t* free_pages, int cap, int32_t* n_free,
                       const int32_t* past, const int32_t* fresh, int B, int N, int32_t* cu,
                       int32_t* row, int64_t* pos, int64_t* slot, void* work, int64_t work_bytes,
                       int32_t* err, hipStream_t s) {
  int64_t bytes = 0;
  const int rc = detllm_packed_plan_work(B, N, &bytes);
  if (rc != DI_OK) return rc;
  if (!table || width < 1 || !free_pages || cap < 0 || !n_free || !past || !fresh || !cu ||
      (N > 0 && (!row || !pos || !slot)) || (bytes > 0 && (!work || ((uintptr_t)work & 15))))
    return DI_EINVAL;
  if (width > PLAN_MAX_WIDTH || work_bytes < bytes) return DI_ERANGE;
  PlanArgs a{table, free_pages, n_free, past, fresh, cu, row, pos, slot, (int4*)work, err,
             width, cap, B, N};
  const size_t lds = (size_t)(B + 1) * 16;
  if (bytes == 0) {
    hipLaunchKernelGGL(k_plan_rows<true>, dim3(1), dim3(PLAN_NT), lds, s, a);
    DI_LAUNCH_CHECK();
    return DI_OK;
  }
  hipLaunchKernelGGL(k_plan_rows<false>, dim3(1), dim3(PLAN_NT), lds, s, a);
  DI_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_plan_tokens, dim3((N + 255) / 256), dim3(256), lds, s, a);
  DI_LAUNCH_CHECK();
  return DI_OK;
}

}  // extern "C"
