// Launches of the packed / paged attention kernels by element type, head dimension, kind of K / V and whether a window applies
// (kWin). The library's two source files share them: capi.cu has the kernels without a window, window.cu those with one,
// compiled at the same time.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include "gemm_sm100.cuh"  // (numbers the kernels for the error word)
#include "paged_decode_sm100.cuh"
#include "varattn_bwd_sm100.cuh"
#include "varattn_sm100.cuh"

namespace bsk {

template <class K>
cudaError_t allow_smem(K kernel, int bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

// Shared memory of the paged decode kernels of 8 * kNQ rows.
template <bool kF16, int kD, bool kFp8, int kNQ, bool kWin>
cudaError_t allow_paged_one() {
  const auto k = paged_decode_kernel<kF16, kD, kFp8, kNQ, kWin>;
  using Sh = PagedShape<kD, kFp8, kNQ>;
  static_assert(Sh::smem_bytes(Sh::kMaxWarps) <= 232448, "shared memory above the 227 KB per-CTA limit");
  return allow_smem(k, Sh::smem_bytes(Sh::kMaxWarps));
}
template <int kNQ, bool kWin>
cudaError_t allow_paged() {
  const cudaError_t e[] = {
      allow_paged_one<false, 128, false, kNQ, kWin>(), allow_paged_one<false, 128, true, kNQ, kWin>(),
      allow_paged_one<false, 64, false, kNQ, kWin>(),  allow_paged_one<false, 64, true, kNQ, kWin>(),
      allow_paged_one<true, 128, false, kNQ, kWin>(),  allow_paged_one<true, 128, true, kNQ, kWin>(),
      allow_paged_one<true, 64, false, kNQ, kWin>(),   allow_paged_one<true, 64, true, kNQ, kWin>()};
  for (cudaError_t x : e)
    if (x != cudaSuccess) return x;
  return cudaSuccess;
}

// The packed / paged attention kernels of one type and head dim.
template <bool kF16, int kD, bool kWin>
cudaError_t allow_varattn() {
  const cudaError_t e[] = {
      allow_smem(varattn_fwd_kernel<kF16, kD, kPacked, kWin>, VarShape<kF16, kD, kPacked>::kSmemBytes),
      allow_smem(varattn_fwd_kernel<kF16, kD, kCache16, kWin>, VarShape<kF16, kD, kCache16>::kSmemBytes),
      allow_smem(varattn_fwd_kernel<kF16, kD, kCacheE4m3, kWin>, VarShape<kF16, kD, kCacheE4m3>::kSmemBytes),
      allow_smem(varattn_bwd_dq_kernel<kF16, kD, kWin>, BwdDqShape<kF16, kD>::kSmemBytes),
      allow_smem(varattn_bwd_dkdv_kernel<kF16, kD, kWin>, BwdDkdvShape<kF16, kD>::kSmemBytes)};
  for (cudaError_t x : e)
    if (x != cudaSuccess) return x;
  return cudaSuccess;
}

// Shared memory of all of them.
template <bool kWin>
cudaError_t allow_attention() {
  const cudaError_t e[] = {allow_paged<1, kWin>(),           allow_paged<2, kWin>(),          allow_paged<4, kWin>(),
                           allow_varattn<false, 64, kWin>(), allow_varattn<false, 128, kWin>(),
                           allow_varattn<true, 64, kWin>(),  allow_varattn<true, 128, kWin>()};
  for (cudaError_t x : e)
    if (x != cudaSuccess) return x;
  return cudaSuccess;
}

// Instantiation by element type, head dim and cache type.
#define BSK_BY_TYPE(KERNEL, f16, dim, fp8, ...)                             \
  do {                                                                      \
    if (f16) {                                                              \
      if (dim == 128) { if (fp8) KERNEL<true, 128, true> __VA_ARGS__; else KERNEL<true, 128, false> __VA_ARGS__; } \
      else            { if (fp8) KERNEL<true, 64, true> __VA_ARGS__; else KERNEL<true, 64, false> __VA_ARGS__; }   \
    } else {                                                                \
      if (dim == 128) { if (fp8) KERNEL<false, 128, true> __VA_ARGS__; else KERNEL<false, 128, false> __VA_ARGS__; } \
      else            { if (fp8) KERNEL<false, 64, true> __VA_ARGS__; else KERNEL<false, 64, false> __VA_ARGS__; }   \
    }                                                                       \
  } while (0)

// Launch that may start before the kernel ahead of it in the stream has ended (the kernel waits for it by itself, after
// its own set-up).
template <class... KArgs, class... Args>
cudaError_t launch_overlapped(void (*kernel)(KArgs...), dim3 grid, int threads, int smem, cudaStream_t s, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int kKind, bool kWin>
cudaError_t varattn_fwd_launch(bool f16, int dim, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                               const VarFwdArgsOf<kWin>& a, unsigned grid, cudaStream_t s) {
  if (f16 && dim == 128)
    return launch_overlapped(varattn_fwd_kernel<true, 128, kKind, kWin>, grid, kAttnThreads,
                             VarShape<true, 128, kKind>::kSmemBytes, s, tq, tk, tv, a);
  if (f16)
    return launch_overlapped(varattn_fwd_kernel<true, 64, kKind, kWin>, grid, kAttnThreads,
                             VarShape<true, 64, kKind>::kSmemBytes, s, tq, tk, tv, a);
  if (dim == 128)
    return launch_overlapped(varattn_fwd_kernel<false, 128, kKind, kWin>, grid, kAttnThreads,
                             VarShape<false, 128, kKind>::kSmemBytes, s, tq, tk, tv, a);
  return launch_overlapped(varattn_fwd_kernel<false, 64, kKind, kWin>, grid, kAttnThreads,
                           VarShape<false, 64, kKind>::kSmemBytes, s, tq, tk, tv, a);
}

// Statistics (and work lists), then dK / dV, then dQ.
struct VarBwdGrids {
  unsigned prep, dkdv, dq;
  unsigned splits;  // kWin: split key blocks at most (0: none is split)
};
template <bool kF16, int kD, bool kWin>
cudaError_t varattn_bwd_launch_one(const VarPrepArgs& p, const VarBwdArgs& a, [[maybe_unused]] const VarJoinArgs& j, const CUtensorMap& tq, const CUtensorMap& tk,
                                   const CUtensorMap& tv, const CUtensorMap& tdo, const VarBwdGrids& g, cudaStream_t s) {
  varattn_bwd_prep_kernel<kF16, kD><<<g.prep, kPlanThreads, 0, s>>>(p);
  cudaError_t e = launch_overlapped(varattn_bwd_dkdv_kernel<kF16, kD, kWin>, g.dkdv, kBwdThreads,
                                    BwdDkdvShape<kF16, kD>::kSmemBytes, s, tq, tk, tv, tdo, a);
  if (e != cudaSuccess) return e;
  e = launch_overlapped(varattn_bwd_dq_kernel<kF16, kD, kWin>, g.dq, kBwdThreads, BwdDqShape<kF16, kD>::kSmemBytes, s, tq, tk, tv,
                        tdo, a);
  if constexpr (kWin)
    if (e == cudaSuccess && g.splits)
      e = launch_overlapped(varattn_bwd_join_kernel<kF16, kD>, dim3(g.splits, j.kv_heads, kVarBlk / kJoinRows), kJoinRows * kD / 2, 0, s,
                            j);
  return e;
}
template <bool kWin>
cudaError_t varattn_bwd_launch(bool f16, int dim, const VarPrepArgs& p, const VarBwdArgs& a, const VarJoinArgs& j, const CUtensorMap& tq,
                               const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo, const VarBwdGrids& g,
                               cudaStream_t s) {
  if (f16)
    return dim == 128 ? varattn_bwd_launch_one<true, 128, kWin>(p, a, j, tq, tk, tv, tdo, g, s)
                      : varattn_bwd_launch_one<true, 64, kWin>(p, a, j, tq, tk, tv, tdo, g, s);
  return dim == 128 ? varattn_bwd_launch_one<false, 128, kWin>(p, a, j, tq, tk, tv, tdo, g, s)
                    : varattn_bwd_launch_one<false, 64, kWin>(p, a, j, tq, tk, tv, tdo, g, s);
}

// Rows per tile (8 * nq), tiles, CTAs per tile and warps per CTA.
struct PagedGrid {
  int nq;
  unsigned tiles;
  int cluster, warps;
};
template <bool kF16, int kD, bool kFp8, int kNQ, bool kWin>
cudaError_t paged_decode_launch_rows(const PagedArgs& a, const PagedGrid& g, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = g.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(g.tiles * g.cluster, a.kv_heads, 1);
  using Sh = PagedShape<kD, kFp8, kNQ>;
  cfg.blockDim = dim3(32 * g.warps, 1, 1);
  cfg.dynamicSmemBytes = Sh::smem_bytes(g.warps);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_decode_kernel<kF16, kD, kFp8, kNQ, kWin>, a);
}
template <bool kWin>
struct PagedDecode {
  template <bool kF16, int kD, bool kFp8>
  static cudaError_t launch(const PagedArgs& a, const PagedGrid& g, cudaStream_t s) {
    if (g.nq == 1) return paged_decode_launch_rows<kF16, kD, kFp8, 1, kWin>(a, g, s);
    if (g.nq == 2) return paged_decode_launch_rows<kF16, kD, kFp8, 2, kWin>(a, g, s);
    return paged_decode_launch_rows<kF16, kD, kFp8, 4, kWin>(a, g, s);
  }
};
template <bool kWin>
cudaError_t paged_decode_launch(bool f16, int dim, bool e4m3, const PagedArgs& a, const PagedGrid& g, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  BSK_BY_TYPE(e = PagedDecode<kWin>::template launch, f16, dim, e4m3, (a, g, s));
  return e;
}

}  // namespace bsk
