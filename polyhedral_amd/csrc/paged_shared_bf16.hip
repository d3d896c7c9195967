// Attention over a paged cache whose requests share prefixes: the bf16 kernels.
#include "paged_shared.hpp"

namespace pa {
int launch_shared_bf16(const PagedK& a, int D, hipStream_t s) {
  return D == 64 ? launch_shared_t<__bf16, 64>(a, s) : launch_shared_t<__bf16, 128>(a, s);
}
}  // namespace pa
