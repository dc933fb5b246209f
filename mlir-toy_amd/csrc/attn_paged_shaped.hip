// attn_paged_shaped.hip — attn_paged_kernel.h's kernels of capped, biased or windowed
// scores over 16-bit and E4M3 pools.
#include "attn_paged_kernel.h"

namespace neptune {

hipError_t launch_attn_paged_shaped(const PagedAttnLaunch &L, hipStream_t s) {
  const PagedArgs a = paged_args(L);
  if (L.pool == E4M3)
    return L.head_dim == 64 ? launch_t<Bf16Tag, 64, E4M3, true>(a, L, s)
                            : launch_t<Bf16Tag, 128, E4M3, true>(a, L, s);
  if (L.dtype == 2)
    return L.head_dim == 64 ? launch_t<Bf16Tag, 64, WIDE, true>(a, L, s)
                            : launch_t<Bf16Tag, 128, WIDE, true>(a, L, s);
  return L.head_dim == 64 ? launch_t<F16Tag, 64, WIDE, true>(a, L, s)
                          : launch_t<F16Tag, 128, WIDE, true>(a, L, s);
}

}  // namespace neptune
