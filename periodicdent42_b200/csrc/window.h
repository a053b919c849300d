// Launches of the packed / paged attention kernels with a window (window.cu), called by capi.cu.
#pragma once

#include "attention_launch.cuh"

namespace bsk {

#define BSK_INTERNAL __attribute__((visibility("hidden")))
BSK_INTERNAL cudaError_t window_allow();  // shared memory of the kernels, once per device
BSK_INTERNAL cudaError_t window_fwd(int kind, bool f16, int dim, const CUtensorMap& tq, const CUtensorMap& tk,
                                    const CUtensorMap& tv, const VarFwdWindowArgs& a, unsigned grid, cudaStream_t s);
BSK_INTERNAL cudaError_t window_bwd(bool f16, int dim, const VarPrepArgs& p, const VarBwdArgs& a, const VarJoinArgs& j,
                       const CUtensorMap& tq,
                                    const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo, const VarBwdGrids& g,
                                    cudaStream_t s);
BSK_INTERNAL cudaError_t window_decode(bool f16, int dim, bool e4m3, const PagedArgs& a, const PagedGrid& g, cudaStream_t s);

}  // namespace bsk
