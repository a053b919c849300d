// The packed / paged attention kernels with a window and sinks: the same kernels as without, instantiated apart so that both
// sets compile at once, and so that calls without a window run the code that they ran before.
#include "window.h"

namespace bsk {

cudaError_t window_allow() { return allow_attention<true>(); }

cudaError_t window_fwd(int kind, bool f16, int dim, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                       const VarFwdWindowArgs& a, unsigned grid, cudaStream_t s) {
  if (kind == kPacked) return varattn_fwd_launch<kPacked, true>(f16, dim, tq, tk, tv, a, grid, s);
  if (kind == kCache16) return varattn_fwd_launch<kCache16, true>(f16, dim, tq, tk, tv, a, grid, s);
  return varattn_fwd_launch<kCacheE4m3, true>(f16, dim, tq, tk, tv, a, grid, s);
}

cudaError_t window_bwd(bool f16, int dim, const VarPrepArgs& p, const VarBwdArgs& a, const VarJoinArgs& j,
                       const CUtensorMap& tq,
                       const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo, const VarBwdGrids& g,
                       cudaStream_t s) {
  return varattn_bwd_launch<true>(f16, dim, p, a, j, tq, tk, tv, tdo, g, s);
}

cudaError_t window_decode(bool f16, int dim, bool e4m3, const PagedArgs& a, const PagedGrid& g, cudaStream_t s) {
  return paged_decode_launch<true>(f16, dim, e4m3, a, g, s);
}

}  // namespace bsk
