// Attention over a paged cache: the f16 kernels.
#include "paged_launch.hpp"

namespace pa {
int launch_paged_f16(const PagedK& a, int D, hipStream_t s) {
  return D == 64 ? launch_paged_t<_Float16, 64>(a, s) : launch_paged_t<_Float16, 128>(a, s);
}
}  // namespace pa
