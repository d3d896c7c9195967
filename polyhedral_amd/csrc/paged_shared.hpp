// The kernels of attention over a paged cache whose requests share prefixes, and their launch: first the
// prefixes, each read once for the rows of all its requests, then each request's own keys, whose rows
// take up the states that the first launch has left.
#pragma once

#include "paged_rows.hpp"
#include "paged_tile.hpp"

namespace pa {
namespace {

template <typename T, int D, int PART>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2)))
void shared_rows_kernel(const PagedK a) {
  __shared__ __attribute__((aligned(256))) char smem[RowsShape<T, D>::SMEM];
  __shared__ int32_t flag;
  rows_body<T, D, PART>(a, (int32_t)blockIdx.x, smem, &flag);
}

template <typename T, int D, int PART>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void shared_both_kernel(const PagedK a) {
  constexpr int A = RowsShape<T, D>::SMEM, B = TileShape<T, D>::SMEM;
  __shared__ __attribute__((aligned(2 * TileShape<T, D>::SLOT))) char smem[A > B ? A : B];
  __shared__ int32_t flag;
  const int32_t id = (int32_t)blockIdx.x;
  if (id < a.tiles.grid)
    tile_body<T, D, PART>(a, id, smem, &flag);
  else
    rows_body<T, D, PART>(a, id - a.tiles.grid, smem, &flag);
}

template <typename T, int D, int PART>
int launch_part(const PagedK& a, hipStream_t s) {
  const int64_t grid = (int64_t)a.tiles.grid + a.rows.grid;
  if constexpr (sizeof(T) == 2) {
    if (a.tiles.grid) {
      hipLaunchKernelGGL((shared_both_kernel<T, D, PART>), dim3((unsigned)grid), dim3(256), 0, s, a);
      PA_LAUNCH_CHECK("shared_both_kernel");
      return PA_OK;
    }
  }
  hipLaunchKernelGGL((shared_rows_kernel<T, D, PART>), dim3((unsigned)grid), dim3(64 * kWaves), 0, s, a);
  PA_LAUNCH_CHECK("shared_rows_kernel");
  return PA_OK;
}

template <typename T, int D>
int launch_shared_t(const PagedK& pre, const PagedK& a, hipStream_t s) {
  if (int rc = launch_part<T, D, kPrefix>(pre, s)) return rc;
  return launch_part<T, D, kOwn>(a, s);
}

}  // namespace
}  // namespace pa
