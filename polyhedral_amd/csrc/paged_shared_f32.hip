// Attention over a paged cache whose requests share prefixes: the f32 kernels.
#include "paged_shared.hpp"

namespace pa {
int launch_shared_f32(const PagedK& a, int D, hipStream_t s) {
  return D == 64 ? launch_shared_t<float, 64>(a, s) : launch_shared_t<float, 128>(a, s);
}
}  // namespace pa
