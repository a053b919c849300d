// Launches of the norm + rotation kernels (norm_rotary.cu), called by capi.cu.
#pragma once

#include <cuda_runtime.h>

#include "norm_rotary.cuh"

namespace bsk {

// Blocks of the backward and the floats of its partial sums.
__attribute__((visibility("hidden"))) int64_t norm_rotary_partials(int tokens, int heads, int kv_heads, int dim, int sm_count);
// dtype 0 bf16, 1 f16, 2 f32. `a` holds the tensors, sizes and scalars; the launch shape is chosen here.
__attribute__((visibility("hidden"))) cudaError_t norm_rotary_fwd(int dtype, bool interleaved, NormRotaryArgs a, int sm_count,
                                                                  cudaStream_t s);
__attribute__((visibility("hidden"))) cudaError_t norm_rotary_bwd(int dtype, bool interleaved, NormRotaryArgs a, void* dwq, void* dwk,
                                                                  int sm_count, cudaStream_t s);
// The rotation alone, a.sign the sign of the angles (-1: the gradient).
__attribute__((visibility("hidden"))) cudaError_t rotary_axes_turn(int dtype, bool interleaved, NormRotaryArgs a, int sm_count,
                                                                   cudaStream_t s);

}  // namespace bsk
