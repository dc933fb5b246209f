// attn_paged_mx.hip — attn_paged_kernel.h's kernels over MXFP4 pools, of plain scores
// and of capped, biased or windowed ones.
#include "attn_paged_kernel.h"

namespace neptune {

hipError_t launch_attn_paged_mx(const PagedAttnLaunch &L, hipStream_t s) {
  const PagedArgs a = paged_args(L);
  auto go = [&](auto e, auto d) {
    typedef decltype(e) E;
    constexpr int HD = decltype(d)::value;
    return shaped(L) ? launch_t<E, HD, MXFP4, true>(a, L, s) : launch_t<E, HD, MXFP4, false>(a, L, s);
  };
  typedef std::integral_constant<int, 64> d64;
  typedef std::integral_constant<int, 128> d128;
  if (L.dtype == 2) return L.head_dim == 64 ? go(Bf16Tag{}, d64{}) : go(Bf16Tag{}, d128{});
  return L.head_dim == 64 ? go(F16Tag{}, d64{}) : go(F16Tag{}, d128{});
}

}  // namespace neptune
