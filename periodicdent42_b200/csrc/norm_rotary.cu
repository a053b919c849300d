// Norm + rotation kernels: instantiation by type, vector width and layout, and their launch shapes.
#include "norm_rotary.h"

#include <algorithm>

namespace bsk {
namespace {

int lanes_for(int units) {
  int g = 1;
  while (g < units) g *= 2;
  return g;
}

// Blocks that the backward gives Q (w = 0) and K: about two rounds of what an SM holds, by their shares of the heads.
int bwd_blocks(const int (&heads)[2], int w, int sm_count) {
  if (!heads[w]) return 0;
  const int64_t all = (int64_t)heads[0] + heads[1];
  return (int)std::max<int64_t>(1, (int64_t)4 * sm_count * heads[w] / all);
}

template <class T, int kVec, int kUnits, bool kInter>
cudaError_t launch(NormRotaryArgs& a, bool backward, int sm_count, cudaStream_t s) {
  a.units = a.dim / (2 * kVec);
  a.group = lanes_for((a.units + kUnits - 1) / kUnits);
  const int groups = kNormThreads / a.group;
  // A row's lanes keep to one token. Few tokens: as many of its heads at once as there are groups, so that a token takes one
  // step; many: four heads a group (the loads of a batch, forward), and the groups left over take other tokens.
  const bool few = a.tokens <= 4 * sm_count;
  if (!backward) {
    const int all = a.heads[0] + a.heads[1];
    a.at_once[0] = std::min(groups, few ? all : (all + kNormBatch - 1) / kNormBatch);
    a.per_block[0] = few ? 1 : groups / a.at_once[0];
    const int64_t grid = ((int64_t)a.tokens + a.per_block[0] - 1) / a.per_block[0];
    norm_rotary_kernel<T, kVec, kUnits, kInter>
        <<<(unsigned)grid, kNormThreads, a.per_block[0] * (a.rotary_dim / 2) * sizeof(float2), s>>>(a);
    return cudaGetLastError();
  }
  for (int w = 0; w < 2; ++w) {
    a.at_once[w] = std::max(1, std::min(groups, few ? a.heads[w] : (a.heads[w] + 3) / 4));
    a.per_block[w] = few ? 1 : groups / a.at_once[w];
  }
  a.blocks_q = bwd_blocks(a.heads, 0, sm_count);
  const int grid = a.blocks_q + bwd_blocks(a.heads, 1, sm_count);
  // (angles of per_block tokens, or the groups' sums: both fit)
  norm_rotary_bwd_kernel<T, kVec, kUnits, kInter><<<grid, kNormThreads, groups * a.dim * sizeof(float), s>>>(a);
  return cudaGetLastError();
}

template <class T, int kVec, int kUnits>
cudaError_t launch(NormRotaryArgs& a, bool inter, bool backward, int sm_count, cudaStream_t s) {
  return inter ? launch<T, kVec, kUnits, true>(a, backward, sm_count, s) : launch<T, kVec, kUnits, false>(a, backward, sm_count, s);
}

// Whether every row can be read and written in pieces of kVec elements, `bytes` wide.
bool fits(const NormRotaryArgs& a, bool inter, bool backward, int vec, int elem, int bytes) {
  const int r = a.rotary_dim;
  if ((a.dim - r) % (2 * vec) || (inter ? r % (2 * vec) : (r / 2) % vec)) return false;
  const auto on = [&](const void* p) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
  for (int w = 0; w < 2; ++w) {
    if (!a.heads[w]) continue;
    if (!on(a.x[w]) || !on(a.y[w]) || a.token_stride[w] * elem % bytes || a.head_stride[w] * elem % bytes ||
        (int64_t)a.dim * elem % bytes)
      return false;
    if (backward && (!on(a.dy[w]) || a.dy_token_stride[w] * elem % bytes || a.dy_head_stride[w] * elem % bytes)) return false;
  }
  return true;
}

// 16-byte pieces where rows and halves allow them, else 4-byte ones, else single elements (dim 80, 40 elements turned, bf16:
// half of a pair's elements starts at a multiple of 40 bytes).
template <class T>
cudaError_t pick(NormRotaryArgs& a, bool inter, bool backward, int sm_count, cudaStream_t s) {
  constexpr int kWide = 16 / sizeof(T), kElem = sizeof(T);
  a.aligned32 = fits(a, inter, backward, kWide, kElem, 32);
  if (fits(a, inter, backward, kWide, kElem, 16)) {
    if constexpr (kElem == 4)
      if (a.dim > 2 * kWide * 32) return launch<T, kWide, 2>(a, inter, backward, sm_count, s);
    return launch<T, kWide, 1>(a, inter, backward, sm_count, s);
  }
  a.aligned32 = 0;
  if constexpr (kElem == 2)
    if (fits(a, inter, backward, 2, kElem, 4))
      return a.dim <= 128 ? launch<T, 2, 1>(a, inter, backward, sm_count, s) : launch<T, 2, 4>(a, inter, backward, sm_count, s);
  return launch<T, 1, 8>(a, inter, backward, sm_count, s);
}

cudaError_t by_type(int dtype, bool inter, NormRotaryArgs& a, bool backward, int sm_count, cudaStream_t s) {
  if (dtype == 0) return pick<__nv_bfloat16>(a, inter, backward, sm_count, s);
  if (dtype == 1) return pick<__half>(a, inter, backward, sm_count, s);
  return pick<float>(a, inter, backward, sm_count, s);
}

template <class T>
cudaError_t launch_weights(const NormWeightArgs& n, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((n.dim + 31) / 32, 2, 1);
  cfg.blockDim = dim3(32 * kNormWeightRows, 1, 1);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, norm_weight_kernel<T>, n);
}

}  // namespace

int64_t norm_rotary_partials(int tokens, int heads, int kv_heads, int dim, int sm_count) {
  const int h[2] = {heads, kv_heads};
  return (int64_t)(bwd_blocks(h, 0, sm_count) + bwd_blocks(h, 1, sm_count)) * dim;
}

cudaError_t norm_rotary_fwd(int dtype, bool interleaved, NormRotaryArgs a, int sm_count, cudaStream_t s) {
  return by_type(dtype, interleaved, a, false, sm_count, s);
}

cudaError_t norm_rotary_bwd(int dtype, bool interleaved, NormRotaryArgs a, void* dwq, void* dwk, int sm_count, cudaStream_t s) {
  cudaError_t e = by_type(dtype, interleaved, a, true, sm_count, s);
  if (e != cudaSuccess || (!dwq && !dwk)) return e;
  NormWeightArgs n{};
  n.partial = a.partial;
  n.dw[0] = dwq;
  n.dw[1] = dwk;
  n.count[0] = n.first[1] = bwd_blocks(a.heads, 0, sm_count);
  n.count[1] = bwd_blocks(a.heads, 1, sm_count);
  n.dim = a.dim;
  n.w_f32 = a.w_f32;
  if (dtype == 0) return launch_weights<__nv_bfloat16>(n, s);
  if (dtype == 1) return launch_weights<__half>(n, s);
  return launch_weights<float>(n, s);
}

}  // namespace bsk
