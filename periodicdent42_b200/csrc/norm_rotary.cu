// Norm + rotation kernels: instantiation by type, vector width and layout, and their launch shapes.
#include "norm_rotary.h"

#include <algorithm>
#include <atomic>

namespace bsk {
namespace {

int lanes_for(int units) {
  int g = 1;
  while (g < units) g *= 2;
  return g;
}

// Launch of a kernel that takes more shared memory than the default limit, raised on its first call on a device (`ready`).
template <class K>
cudaError_t run(K kernel, std::atomic<uint64_t>& ready, int most, int grid, int smem, const NormRotaryArgs& a, cudaStream_t s) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = uint64_t{1} << (device & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit, std::memory_order_release);
  }
  kernel<<<grid, kNormThreads, smem, s>>>(a);
  return cudaGetLastError();
}

// Blocks that Q (w = 0) and K get of `per_sm` on each SM, by what their rows and a token's angles cost (the angles about what
// six heads do), and no more than there are chunks.
int blocks_of(const int (&heads)[2], int w, int per_sm, int64_t chunks, int sm_count) {
  if (!heads[w]) return 0;
  const auto cost = [&](int i) { return heads[i] ? (int64_t)heads[i] + 6 : 0; };
  return (int)std::max<int64_t>(1, std::min(chunks, per_sm * sm_count * cost(w) / (cost(0) + cost(1))));
}

enum class Pass { kForward, kBackward, kTurn };  // kTurn: the rotation alone

template <class T, int kVec, int kUnits, bool kInter, int kLanes, Pass kPass>
cudaError_t launch(NormRotaryArgs& a, int sm_count, cudaStream_t s) {
  using Sh = NormShape<T, kVec, kUnits, kPass == Pass::kBackward>;
  const int groups = kNormThreads / a.group;
  // A row's lanes keep to one token. Few tokens: as many of its heads at once as there are groups, so that a token takes one
  // step; many: four heads a group, and the groups left over take other tokens.
  const bool few = a.tokens <= 4 * sm_count;
  int grid = 0;
  for (int w = 0; w < 2; ++w) {
    a.at_once[w] = std::max(1, std::min(groups, few ? a.heads[w] : (a.heads[w] + 3) / 4));
    a.per_block[w] = few ? 1 : groups / a.at_once[w];
    grid += blocks_of(a.heads, w, Sh::kBlocksPerSm, ((int64_t)a.tokens + a.per_block[w] - 1) / a.per_block[w], sm_count);
    if (w == 0) a.blocks_q = grid;
  }
  a.grid = grid;
  static std::atomic<uint64_t> ready{0};
  if constexpr (kPass == Pass::kBackward)
    return run(norm_rotary_bwd_kernel<T, kVec, kUnits, kInter, kLanes>, ready, Sh::kMostSmem, grid, Sh::smem_bytes(a), a, s);
  else
    return run(norm_rotary_kernel<T, kVec, kUnits, kInter, kLanes, kPass == Pass::kForward>, ready, Sh::kMostSmem, grid,
               Sh::smem_bytes(a), a, s);
}

// The lanes of a row are a power of two; for 16-byte pieces their number is known to the compiler (whose sums it unrolls).
template <class T, int kVec, int kUnits, bool kInter, Pass kPass>
cudaError_t launch_lanes(NormRotaryArgs& a, int sm_count, cudaStream_t s) {
  a.units = a.dim / (2 * kVec);
  a.group = lanes_for((a.units + kUnits - 1) / kUnits);
  if constexpr (kVec * sizeof(T) == 16 && kUnits == 1 && kPass != Pass::kTurn) {
    a.group = std::max(a.group, 4);
    if (a.group == 4) return launch<T, kVec, kUnits, kInter, 4, kPass>(a, sm_count, s);
    if (a.group == 8) return launch<T, kVec, kUnits, kInter, 8, kPass>(a, sm_count, s);
    if (a.group == 16) return launch<T, kVec, kUnits, kInter, 16, kPass>(a, sm_count, s);
    return launch<T, kVec, kUnits, kInter, 32, kPass>(a, sm_count, s);
  } else {
    return launch<T, kVec, kUnits, kInter, 0, kPass>(a, sm_count, s);
  }
}

template <class T, int kVec, int kUnits, Pass kPass>
cudaError_t launch_layout(NormRotaryArgs& a, bool inter, int sm_count, cudaStream_t s) {
  return inter ? launch_lanes<T, kVec, kUnits, true, kPass>(a, sm_count, s) : launch_lanes<T, kVec, kUnits, false, kPass>(a, sm_count, s);
}
template <class T, int kVec, int kUnits>
cudaError_t launch_any(NormRotaryArgs& a, bool inter, Pass pass, int sm_count, cudaStream_t s) {
  if (pass == Pass::kTurn) return launch_layout<T, kVec, kUnits, Pass::kTurn>(a, inter, sm_count, s);
  if (pass == Pass::kBackward) return launch_layout<T, kVec, kUnits, Pass::kBackward>(a, inter, sm_count, s);
  return launch_layout<T, kVec, kUnits, Pass::kForward>(a, inter, sm_count, s);
}

// Whether every row can be read and written in pieces of `vec` elements of `elem` bytes.
bool fits(const NormRotaryArgs& a, bool inter, bool backward, int vec, int elem) {
  const int r = a.rotary_dim, bytes = vec * elem;
  if (a.dim % (2 * vec) || (inter ? r % vec : (r / 2) % vec)) return false;
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

// 16-byte pieces where rows and halves allow them, else 8- and 4-byte ones, else single elements (dim 80, 40 elements turned, bf16:
// the second halves of the pairs start 40 bytes in, at a multiple of 8; 16383 tokens, 32 + 8 heads, with gradients: 253 us in
// 8-byte pieces and four blocks on an SM, 677 us in 4-byte ones and one block).
template <class T>
cudaError_t pick(NormRotaryArgs& a, bool inter, Pass pass, int sm_count, cudaStream_t s) {
  const bool backward = pass == Pass::kBackward;
  constexpr int kWide = 16 / sizeof(T), kElem = sizeof(T);
  if (fits(a, inter, backward, kWide, kElem)) {
    if constexpr (kElem == 4)
      if (a.dim > 2 * kWide * 32) return launch_any<T, kWide, 2>(a, inter, pass, sm_count, s);
    return launch_any<T, kWide, 1>(a, inter, pass, sm_count, s);
  }
  if constexpr (kElem == 2) {
    if (a.dim <= 256 && fits(a, inter, backward, 4, kElem)) return launch_any<T, 4, 1>(a, inter, pass, sm_count, s);
    if (fits(a, inter, backward, 2, kElem))
      return a.dim <= 128 ? launch_any<T, 2, 1>(a, inter, pass, sm_count, s) : launch_any<T, 2, 4>(a, inter, pass, sm_count, s);
  }
  return launch_any<T, 1, 8>(a, inter, pass, sm_count, s);
}

cudaError_t by_type(int dtype, bool inter, NormRotaryArgs& a, Pass pass, int sm_count, cudaStream_t s) {
  if (dtype == 0) return pick<__nv_bfloat16>(a, inter, pass, sm_count, s);
  if (dtype == 1) return pick<__half>(a, inter, pass, sm_count, s);
  return pick<float>(a, inter, pass, sm_count, s);
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
  // (Q and K get one block each at least)
  return tokens > 0 ? ((int64_t)kNormMostBlocks * sm_count + 2) * dim : 0;
}

cudaError_t norm_rotary_fwd(int dtype, bool interleaved, NormRotaryArgs a, int sm_count, cudaStream_t s) {
  a.sign = 1.0f;
  return by_type(dtype, interleaved, a, Pass::kForward, sm_count, s);
}

cudaError_t rotary_axes_turn(int dtype, bool interleaved, NormRotaryArgs a, int sm_count, cudaStream_t s) {
  return by_type(dtype, interleaved, a, Pass::kTurn, sm_count, s);
}

cudaError_t norm_rotary_bwd(int dtype, bool interleaved, NormRotaryArgs a, void* dwq, void* dwk, int sm_count, cudaStream_t s) {
  a.sign = 1.0f;
  cudaError_t e = by_type(dtype, interleaved, a, Pass::kBackward, sm_count, s);
  if (e != cudaSuccess || (!dwq && !dwk)) return e;
  NormWeightArgs n{};
  n.partial = a.partial;
  n.dw[0] = dwq;
  n.dw[1] = dwk;
  n.count[0] = n.first[1] = a.blocks_q;
  n.count[1] = a.grid - a.blocks_q;
  n.dim = a.dim;
  n.w_f32 = a.w_f32;
  if (dtype == 0) return launch_weights<__nv_bfloat16>(n, s);
  if (dtype == 1) return launch_weights<__half>(n, s);
  return launch_weights<float>(n, s);
}

}  // namespace bsk
