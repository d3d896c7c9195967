// Attention over a paged cache: the f32 kernels.
#include "paged_launch.hpp"

namespace pa {
int launch_paged_f32(const PagedK& a, int D, hipStream_t s) {
  return D == 64 ? launch_paged_t<float, 64>(a, s) : launch_paged_t<float, 128>(a, s);
}
}  // namespace pa
