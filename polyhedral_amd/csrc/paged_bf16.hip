// Attention over a paged cache: the bf16 kernels.
#include "paged_launch.hpp"

namespace pa {
int launch_paged_bf16(const PagedK& a, int D, hipStream_t s) {
  return D == 64 ? launch_paged_t<__bf16, 64>(a, s) : launch_paged_t<__bf16, 128>(a, s);
}
}  // namespace pa
