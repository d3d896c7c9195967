// The kernels of attention over a paged cache whose requests share prefixes, and their launch.
//
// One grid takes the prefixes, each read once for the rows of all its requests, and every request's own keys:
// the tiles of many rows first, whose MFMAs the loads of the others then run beside.  A second launch merges the
// states that they leave, a row at a time, in the order of the prefix's shares.  (The two parts one after the
// other, a part's shares merged by its last work-group and the prefix's state taken up by the own part: 64
// requests behind 8192 tokens 41 and 29 us, and 24 us of one row's 64 shares behind 65536.)
//
// What bounds it, at 32 heads on 8 of 128 in bf16: behind long prefixes HBM (32 requests behind 65536, 358 MB: 90
// us of 104, 4.0 TB/s), with chunks the tiles' MFMAs (12 of 100 to 600 tokens behind 12000 to 16384: the call
// 0.95 to 0.98 ms, 0.92 to 0.96 PFLOP/s), else what is outside the steps: 64 requests behind 8192 tokens, whose prefix is 176 units of 12
// steps, 43 us, then 7 of the merge, 5 of the plan and the launches' gaps, where its 128 MB take 26.
#pragma once

#include "paged_rows.hpp"
#include "paged_tile.hpp"

namespace pa {
namespace {

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2)))
void shared_rows_kernel(const PagedK a) {
  __shared__ __attribute__((aligned(256))) char smem[RowsShape<T, D>::SMEM];
  __shared__ int32_t flag;
  const int32_t id = (int32_t)blockIdx.x;
  if (id < a.pre_rows.grid)
    rows_body<T, D, kPrefix>(a, id, smem, &flag);
  else
    rows_body<T, D, kOwn>(a, id - a.pre_rows.grid, smem, &flag);
}

template <typename T, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void shared_both_kernel(const PagedK a) {
  constexpr int A = RowsShape<T, D>::SMEM, B = TileShape<T, D>::SMEM;
  __shared__ __attribute__((aligned(2 * TileShape<T, D>::SLOT))) char smem[A > B ? A : B];
  __shared__ int32_t flag;
  int32_t id = (int32_t)blockIdx.x;
  if (id < a.pre_tiles.grid) {
    tile_body<T, D, kPrefix>(a, id, smem, &flag);
    return;
  }
  id -= a.pre_tiles.grid;
  if (id < a.tiles.grid) {
    tile_body<T, D, kOwn>(a, id, smem, &flag);
    return;
  }
  id -= a.tiles.grid;
  // (beside tiles a prefix of few rows is rare: its work-groups, mostly without work, last)
  if (id < a.rows.grid)
    rows_body<T, D, kOwn>(a, id, smem, &flag);
  else
    rows_body<T, D, kPrefix>(a, id - a.rows.grid, smem, &flag);
}

// A row's state: D / 4 lanes with 4 columns each.
struct MergeState {
  float m, rest, l;
  f32x4 x;
  __device__ __forceinline__ void add(const f32x4& ml, const f32x4& y) {
    const float top = nan_max(m, ml[0]);
    const float r = ml[0] > m ? ml[1] : ml[0] == m ? nan_max(rest, ml[1]) : rest;
    const float f0 = __builtin_amdgcn_exp2f((m - base_of(top)) + (rest - r)), f1 = __builtin_amdgcn_exp2f((ml[0] - base_of(top)) + (ml[1] - r));
    m = top;
    rest = r;
    l = f0 * l + f1 * ml[2];
    x = f0 * x + f1 * y;
  }
};

// ONE: a work-group merges one row, its states dealt to 256 / (D / 4) lots of lanes and those in order; else each
// lot a row.
template <typename T, int D, bool ONE>
__global__ __launch_bounds__(256) void shared_merge_kernel(const PagedK a) {
  constexpr int LPR = D / 4, LOTS = 256 / LPR, STATE = state_floats(D) / 4;
  __shared__ f32x4 part[ONE ? LOTS : 1][LPR + 1];
  const int col = (int)threadIdx.x % LPR, lot = (int)threadIdx.x / LPR;
  const int Hq = a.Hkv * a.G;
  const int64_t id = ONE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * LOTS + lot;
  const int32_t i = imin((int32_t)(id / Hq), a.T - 1), head = (int32_t)(id % Hq);
  // (all on their way at once)
  const int32_t last = a.share.start[a.R], end = *a.end, tok = a.share.rows[i];
  StatesAt at = a.at[(int64_t)i * Hq + head];
  // (a sharing of another step: rows past the requests' last stay, and states are read from within their memory)
  if (id >= (int64_t)imin(imax(last, 0), a.T) * Hq || tok < 0 || tok >= end) return;
  if (at.n < 0 || at.n > (1 << 20) || ((int64_t)at.first + (int64_t)at.step * imax(at.n - 1, 0) + STATE) * 4 > a.n_states) at.n = 0;
  const f32x4* state = reinterpret_cast<const f32x4*>(a.states) + at.first;
  const f32x4* own = reinterpret_cast<const f32x4*>(a.own) + ((int64_t)tok * Hq + head) * STATE;
  MergeState s{-INFINITY, 0.f, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}};
  if (!ONE || lot == 0) s.add(own[D / 4], own[col]);
#pragma unroll 4
  for (int j = ONE ? lot : 0; j < at.n; j += ONE ? LOTS : 1) {
    const f32x4* y = state + (int64_t)j * at.step;
    s.add(y[D / 4], y[col]);
  }
  if constexpr (ONE) {
    part[lot][col] = s.x;
    if (col == 0) part[lot][LPR] = f32x4{s.m, s.rest, s.l, 0.f};
    __syncthreads();
    if (lot) return;
    for (int j = 1; j < imin(LOTS, at.n); ++j) s.add(part[j][LPR], part[j][col]);
  }
  const float inv = s.l == 0.f ? 0.f : 1.f / s.l;
  Mma<T>::store4(a.o + (int64_t)tok * a.o_st + (int64_t)head * a.o_sh + 4 * (int)sizeof(T) * col, s.x * inv);
  if (a.lse && col == 0)
    a.lse[(int64_t)tok * a.lse_st + (int64_t)head * a.lse_sh] = s.l == 0.f ? -INFINITY : (s.m + (log2f(s.l) + s.rest)) * kLn2;
}

// Rows (of all heads) up to which each has a work-group of its own to merge it.  The call with one each / with several
// rows to a work-group, tokens of 32 heads on 8 of 128 in bf16: 1024 rows 24.0 / 23.8 us behind 2048 tokens and 36.7 / 41
// behind 16384, 2048 rows 32.9 / 32.8 and 54 / 57, 4096 rows 59.5 / 57.1 and 98.3 / 97.3, 8192 rows 130 / 123 and 184 /
// 178, 32768 of chunks 103 / 77 and 313 / 286; 2192 of 16 heads of 64 in f16 27.7 / 28.0.
constexpr int64_t kMergeRows = 2560;

template <typename T, int D>
int launch_shared_t(const PagedK& a, hipStream_t s) {
  const unsigned grid = (unsigned)((int64_t)a.pre_tiles.grid + a.tiles.grid + a.pre_rows.grid + a.rows.grid);
  bool both = false;
  if constexpr (sizeof(T) == 2) {
    both = a.pre_tiles.grid || a.tiles.grid;
    if (both) hipLaunchKernelGGL((shared_both_kernel<T, D>), dim3(grid), dim3(256), 0, s, a);
  }
  if (!both) hipLaunchKernelGGL((shared_rows_kernel<T, D>), dim3(grid), dim3(64 * kWaves), 0, s, a);
  PA_LAUNCH_CHECK("shared_kernel");
  const int64_t rows = (int64_t)a.T * a.Hkv * a.G;
  if (rows <= kMergeRows)
    hipLaunchKernelGGL((shared_merge_kernel<T, D, true>), dim3((unsigned)rows), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((shared_merge_kernel<T, D, false>), dim3((unsigned)((rows * (D / 4) + 255) / 256)), dim3(256), 0, s, a);
  PA_LAUNCH_CHECK("shared_merge_kernel");
  return PA_OK;
}

}  // namespace
}  // namespace pa
