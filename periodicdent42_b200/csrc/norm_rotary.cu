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

enum class Pass { kForward, kBackward, kTurn };  // kTurn: the rotation alone

// How a tensor's heads and tokens are dealt to a block's groups, and what a chunk of it costs.
struct Deal {
  int at_once, per_block;
  int64_t chunks, cost;
};
// `most` heads of a token for each group. Costs in eighths of a row's, by the instructions counted for each: what a chunk takes
// per thread beside its rows (angles and weights to registers), and an element of the angles.
Deal deal(const NormRotaryArgs& a, int w, int groups, int rows, int most, Pass pass) {
  const int at_once = std::max(1, std::min(groups, (a.heads[w] + most - 1) / most)), per_block = groups / at_once;
  const int64_t steps = (a.heads[w] + rows * at_once - 1) / (rows * at_once);
  const int64_t elements = ((int64_t)per_block * (a.rotary_dim / 2) + kNormThreads - 1) / kNormThreads;
  const int chunk = pass == Pass::kForward ? 11 : pass == Pass::kBackward ? 3 : 5, angle = 6;
  return {at_once, per_block, ((int64_t)a.tokens + per_block - 1) / per_block, steps * rows * 8 + chunk + elements * angle};
}

// The blocks of Q and of K out of `most` together, and how each is dealt: what ends first by the costs, where every block takes
// whole chunks. Few tokens: as many heads of a token at once as there are groups, so that a token takes one step. Measured (us,
// 16383 tokens, 32 + 8 heads of 128 with gradients; four heads a group and blocks by the heads / up to 8 / up to 16, by costs):
// bf16 179 / 171 / 162, three axes without the norm 135 / 121 / 133 (long chunks of angles leave the copies idle), fp32 266 (four
// heads by costs) / 291 / 299; 16 + 4 heads of 256 230 / 218 / 202; 4096 tokens 58 / 55 / 55, 2048 32 / 33 / 34.
void deal_blocks(NormRotaryArgs& a, int groups, int rows, int most, int widest, bool few, Pass pass) {
  if (few || !a.heads[0] || !a.heads[1]) {
    const Deal d[2] = {deal(a, 0, groups, rows, few ? 1 : 8, pass), deal(a, 1, groups, rows, few ? 1 : 8, pass)};
    int blocks[2] = {0, 0};
    for (int w = 0; w < 2; ++w) {
      a.at_once[w] = d[w].at_once;
      a.per_block[w] = few ? 1 : d[w].per_block;
      const int64_t chunks = few ? a.tokens : d[w].chunks, work[2] = {a.heads[0] ? a.heads[0] + 6 : 0, a.heads[1] ? a.heads[1] + 6 : 0};
      if (a.heads[w]) blocks[w] = (int)std::max<int64_t>(1, std::min(chunks, most * work[w] / (work[0] + work[1])));
    }
    a.blocks_q = blocks[0];
    a.grid = blocks[0] + blocks[1];
    return;
  }
  int64_t least = INT64_MAX;
  for (int i = 4; i <= widest; i *= 2)
    for (int j = 4; j <= widest; j *= 2) {
      const Deal q = deal(a, 0, groups, rows, i, pass), k = deal(a, 1, groups, rows, j, pass);
      const double share = (double)(q.chunks * q.cost) / (double)(q.chunks * q.cost + k.chunks * k.cost);
      const int64_t about = std::max<int64_t>(1, (int64_t)((double)most * share));
      for (int64_t r = std::max<int64_t>(1, (q.chunks + about - 1) / about - 1), n = 0; n < 3; ++r, ++n) {  // rounds of Q
        const int64_t blocks = (q.chunks + r - 1) / r, left = most - blocks;
        if (left < 1) continue;
        const int64_t time = std::max(r * q.cost, (k.chunks + left - 1) / left * k.cost);
        if (time >= least) continue;
        least = time;
        a.at_once[0] = q.at_once;
        a.at_once[1] = k.at_once;
        a.per_block[0] = q.per_block;
        a.per_block[1] = k.per_block;
        a.blocks_q = (int)blocks;
        a.grid = (int)(blocks + std::min(left, k.chunks));
      }
    }
}

template <class T, int kVec, int kUnits, bool kInter, int kLanes, Pass kPass>
cudaError_t launch(NormRotaryArgs& a, int sm_count, cudaStream_t s) {
  using Sh = NormShape<T, kVec, kUnits, kPass == Pass::kBackward>;
  // (a row's lanes keep to one token)
  constexpr int kWidest = sizeof(T) == 4 ? 4 : kPass == Pass::kTurn ? 8 : 16;
  deal_blocks(a, kNormThreads / a.group, Sh::kRows, Sh::kBlocksPerSm * sm_count, kWidest, a.tokens <= 4 * sm_count, kPass);
  static std::atomic<uint64_t> ready{0};
  if constexpr (kPass == Pass::kBackward)
    return run(norm_rotary_bwd_kernel<T, kVec, kUnits, kInter, kLanes>, ready, Sh::kMostSmem, a.grid, Sh::smem_bytes(a), a, s);
  else
    return run(norm_rotary_kernel<T, kVec, kUnits, kInter, kLanes, kPass == Pass::kForward>, ready, Sh::kMostSmem, a.grid,
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
// the second halves of the pairs start 40 bytes in, at a multiple of 8; 16383 tokens, 32 + 8 heads, with gradients: 223 us in
// 8-byte pieces and four blocks on an SM; when it was 253, 677 us in 4-byte ones and one block).
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
