// The kernels of attention over a paged cache and their launch.
//
// A call whose requests have few rows each (single tokens) runs the rows' body alone.  Any other
// call of the 2-byte types runs both in one grid, chunks' tiles first (they are the longer), then the
// tiles of the requests with few rows: a batch that mixes the two is one launch, in which the loads
// of the ones run beside the MFMAs of the others.
#pragma once

#include "paged_rows.hpp"
#include "paged_tile.hpp"

namespace pa {
namespace {

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2)))
void paged_rows_kernel(const PagedK a) {
  __shared__ __attribute__((aligned(256))) char smem[RowsShape<T, D>::SMEM];
  __shared__ int32_t flag;
  rows_body<T, D>(a, (int32_t)blockIdx.x, smem, &flag);
}

template <typename T, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void paged_both_kernel(const PagedK a) {
  constexpr int A = RowsShape<T, D>::SMEM, B = TileShape<T, D>::SMEM;
  __shared__ __attribute__((aligned(2 * TileShape<T, D>::SLOT))) char smem[A > B ? A : B];
  __shared__ int32_t flag;
  const int32_t id = (int32_t)blockIdx.x;
  if (id < a.tiles.grid)
    tile_body<T, D>(a, id, smem, &flag);
  else
    rows_body<T, D>(a, id - a.tiles.grid, smem, &flag);
}

template <typename T, int D>
int launch_paged_t(const PagedK& a, hipStream_t s) {
  const int64_t grid = (int64_t)a.tiles.grid + a.rows.grid;
  if constexpr (sizeof(T) == 2) {
    if (a.tiles.grid) {
      hipLaunchKernelGGL((paged_both_kernel<T, D>), dim3((unsigned)grid), dim3(256), 0, s, a);
      PA_LAUNCH_CHECK("paged_both_kernel");
      return PA_OK;
    }
  }
  hipLaunchKernelGGL((paged_rows_kernel<T, D>), dim3((unsigned)grid), dim3(64 * kWaves), 0, s, a);
  PA_LAUNCH_CHECK("paged_rows_kernel");
  return PA_OK;
}

}  // namespace
}  // namespace pa
