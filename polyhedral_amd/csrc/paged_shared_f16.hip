// Attention over a paged cache whose requests share prefixes: the f16 kernels.
#include "paged_shared.hpp"

namespace pa {
int launch_shared_f16(const PagedK& a, int D, hipStream_t s) {
  return D == 64 ? launch_shared_t<_Float16, 64>(a, s) : launch_shared_t<_Float16, 128>(a, s);
}
}  // namespace pa
