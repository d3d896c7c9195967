// The kernels of attention over a paged cache whose requests share prefixes, and their launch.
//
// One grid takes the prefixes, each read once for the rows of all its requests, and every request's own keys:
// the tiles of many rows first, whose MFMAs the loads of the others then run beside.  A second launch merges the
// states that they leave, a row at a time, in the order of the prefix's shares and the own keys last.  (The two
// parts one after the other, a part's shares merged by its last work-group and the prefix's state taken up
// by the own part: 64 requests behind 8192 tokens 41 and 29 us, 87 with the plan.)
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
  if (id < a.pre_rows.grid)
    rows_body<T, D, kPrefix>(a, id, smem, &flag);
  else
    rows_body<T, D, kOwn>(a, id - a.pre_rows.grid, smem, &flag);
}

// D / 4 lanes to a row of the groups' rows.
template <typename T, int D>
__global__ __launch_bounds__(256) void shared_merge_kernel(const PagedK a) {
  constexpr int LPR = D / 4, STATE = state_floats(D) / 4;
  const int col = (int)threadIdx.x % LPR;
  const int Hq = a.Hkv * a.G;
  const int64_t id = (int64_t)blockIdx.x * (256 / LPR) + (int)threadIdx.x / LPR;
  // (a sharing of another step: rows past the requests' last stay, and states are read from within their memory)
  const int32_t rows = imin(imax(a.share.start[a.R], 0), a.T), end = imin(imax(a.q_start[a.R], 0), a.T);
  const int32_t i = (int32_t)(id / Hq), head = (int32_t)(id - (int64_t)i * Hq);
  if (i >= rows) return;
  const int32_t tok = a.share.rows[i];
  if (tok < 0 || tok >= end) return;
  StatesAt at = a.at[id];
  if (at.n < 0 || at.n > (1 << 20) || ((int64_t)at.first + (int64_t)at.step * imax(at.n - 1, 0) + STATE) * 4 > a.n_states) at.n = 0;
  const f32x4* state = reinterpret_cast<const f32x4*>(a.states) + at.first;
  const f32x4* own = reinterpret_cast<const f32x4*>(a.own) + ((int64_t)tok * Hq + head) * STATE;
  const f32x4 oml = own[D / 4];
  f32x4 x = own[col];
  // the largest maximum, then the sums
  float m = oml[0], rest = oml[1];
#pragma unroll 4
  for (int s = 0; s < at.n; ++s) {
    const f32x4 ml = state[(int64_t)s * at.step + D / 4];
    rest = ml[0] > m ? ml[1] : ml[0] == m ? nan_max(rest, ml[1]) : rest;
    m = nan_max(m, ml[0]);
  }
  const float base = base_of(m);
  const float f0 = __builtin_amdgcn_exp2f((oml[0] - base) + (oml[1] - rest));
  f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 4
  for (int s = 0; s < at.n; ++s) {
    const f32x4 ml = state[(int64_t)s * at.step + D / 4], y = state[(int64_t)s * at.step + col];
    const float f = __builtin_amdgcn_exp2f((ml[0] - base) + (ml[1] - rest));
    l += f * ml[2];
    sum += f * y;
  }
  l += f0 * oml[2];
  sum += f0 * x;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  Mma<T>::store4(a.o + (int64_t)tok * a.o_st + (int64_t)head * a.o_sh + 4 * (int)sizeof(T) * col, sum * inv);
  if (a.lse && col == 0)
    a.lse[(int64_t)tok * a.lse_st + (int64_t)head * a.lse_sh] = l == 0.f ? -INFINITY : (m + (log2f(l) + rest)) * kLn2;
}

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
  hipLaunchKernelGGL((shared_merge_kernel<T, D>), dim3((unsigned)((rows * (D / 4) + 255) / 256)), dim3(256), 0, s, a);
  PA_LAUNCH_CHECK("shared_merge_kernel");
  return PA_OK;
}

}  // namespace
}  // namespace pa
