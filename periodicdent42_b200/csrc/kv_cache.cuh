// Paged key/value cache for sm_100a: rows written (copied, or quantised to e4m3) and read back.
//
// A cache is [pages, page size, kv heads, D] with D = 64 or 128, addressed by flat slots (page * page size + offset);
// an e4m3 cache has one fp32 scale for each slot and head. Writing a row x of D elements:
//     scale = max |x| / 448,   code_d = e4m3(x_d / scale)      (448: the largest e4m3 value)
// with IEEE divisions, so a code is off by at most half an e4m3 step and never saturates; a row of zeros has scale 0 and
// codes 0, a row that holds a NaN has scale NaN. Reading back gives code * scale, rounded once.
//
// The quotients are taken by Markstein's method (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000
// processor", 1990): with y the correctly rounded reciprocal of the scale, q = x y, the residual r = q scale - x in one fused
// operation, and q - r y in another, three packed operations for two elements in place of a division each. The residual is
// exact but for 2 quotients in 1000, and the result is the correctly rounded x / scale for every pair of bf16 or fp16
// mantissas (compared in exact arithmetic; in this form of the signs also for x = -0).
//
// Bound: each row is read and written once, and few instructions are left beside that. Measured (16383 tokens of 8 heads,
// D 128, inputs larger than L2, in a graph; the memory's time at the rate of a copy in parentheses):
//   append as e4m3 26 us (16): instruction issue, 580 warp instructions for two K and two V rows of 8 elements a lane
//     (33 us with divisions);  append of 16 bits 23 us (20);
//   gather from e4m3 20 us (16), of 8191 tokens 10.8 (7.8), from 16 bits 12.5 (10.3): the loads' latency, slot -> codes, with
//     one row of K and of V a thread.
// One thread holds 8 elements of a K row and the same 8 of the V row (independent 16-byte loads; the append of one row when
// there are few, else of two); D / 8 neighbouring lanes share a row and take its maximum by shuffles.
// Slots outside [0, num_slots) are not touched: negative ones mark padding, others set the device error word.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "bsattn_bwd_sm100.cuh"

namespace bsk {

constexpr int kCacheThreads = 256;
constexpr uint32_t kKidKvCache = 9;

struct KvCacheArgs {
  const void* x[2];                          // K, V rows to write (append)
  int64_t token_stride[2], head_stride[2];   // of x, in elements
  void* y[2];                                // contiguous [tokens, heads, D] to read into (gather)
  void* cache[2];                            // k_cache, v_cache
  float* scale[2];                           // k_scale, v_scale (e4m3 caches)
  const void* slots;                         // int32 or int64 [tokens]
  int slots64;
  int tokens, heads;
  int heads_shift;                           // log2 of heads, -1 if it is no power of two
  int64_t num_slots;
  uint32_t* err;
};

__device__ __forceinline__ int64_t cache_slot(const KvCacheArgs& a, int t) {
  const int64_t s = a.slots64 ? static_cast<const int64_t*>(a.slots)[t] : static_cast<const int*>(a.slots)[t];
  if (s >= a.num_slots) {
    atomicCAS(a.err, 0u, kErrBounds | (kKidKvCache << 8) | (1u << 16));
    return -1;
  }
  return s;
}

template <bool kF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  return kF16 ? __half22float2(*reinterpret_cast<__half2*>(&w)) : __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w));
}
template <bool kF16>
__device__ __forceinline__ uint32_t round2(float lo, float hi) {
  if (kF16) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// kRows rows of K and of V per thread, kCacheThreads / (D / 8) rows apart: their loads are issued before any is used.
template <bool kF16, int kD, bool kFp8, int kRows>
__global__ void __launch_bounds__(kCacheThreads) kv_cache_append_kernel(const KvCacheArgs a) {
  constexpr int kTpr = kD / 8;  // lanes per row: 8 or 16
  // token * heads + head, below 2^31 (checked by the caller); a row's lanes are never split over two warps
  const uint32_t first = blockIdx.x * (kRows * (kCacheThreads / kTpr)) + threadIdx.x / kTpr;
  const uint32_t rows = static_cast<uint32_t>(a.tokens) * a.heads;
  const int c = threadIdx.x % kTpr;
  uint4 v[kRows][2];
  int64_t at[kRows];  // cache row, -1: none
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const uint32_t row = first + i * (kCacheThreads / kTpr);
    const bool live = row < rows;
    const uint32_t heads = static_cast<uint32_t>(a.heads);
    const int t = !live ? 0 : a.heads_shift >= 0 ? row >> a.heads_shift : row / heads;
    const int h = !live ? 0 : row - t * heads;
#pragma unroll
    for (int w = 0; w < 2; ++w) {  // (not behind the slot: the loads' latencies overlap)
      v[i][w] = make_uint4(0, 0, 0, 0);
      if (live)
        v[i][w] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x[w]) + t * a.token_stride[w] +
                                                       h * a.head_stride[w]) + c);
    }
    const int64_t slot = live ? cache_slot(a, t) : -1;
    at[i] = slot >= 0 ? slot * a.heads + h : -1;
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i)
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      if (!kFp8) {
        if (at[i] >= 0) static_cast<uint4*>(a.cache[w])[at[i] * kTpr + c] = v[i][w];
        continue;
      }
      const uint32_t words[4] = {v[i][w].x, v[i][w].y, v[i][w].z, v[i][w].w};
      float f[8];
      // largest |x| as bits: ordered like the values, a NaN above all of them (16-bit lanes until the row's is found)
      uint32_t top2 = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 p = unpack2<kF16>(words[k] ^ 0x80008000u);
        f[2 * k] = p.x;  // -x
        f[2 * k + 1] = p.y;
        top2 = __vmaxu2(top2, words[k] & 0x7fff7fffu);
      }
#pragma unroll
      for (int o = kTpr / 2; o > 0; o >>= 1) top2 = __vmaxu2(top2, __shfl_xor_sync(0xffffffffu, top2, o));
      const float top = unpack2<kF16>(max(top2 >> 16, top2 & 0xffffu)).x;
      const float scale = __fdiv_rn(top, 448.0f);
      uint2 codes = make_uint2(0, 0);
      if (scale > 0.0f) {
        if (scale > 0x1p-80f && scale < 0x1p80f) {  // nothing on the way leaves the normal range, but for elements of code 0
          const float ninv = -__frcp_rn(scale);
          const uint64_t ny2 = f2_pack(ninv, ninv), s2 = f2_pack(scale, scale);
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
            const uint64_t n2 = f2_pack(f[k], f[k + 1]), q2 = f2_mul(n2, ny2);
            f2_unpack(f2_fma(f2_fma(q2, s2, n2), ny2, q2), f[k], f[k + 1]);
          }
        } else {
#pragma unroll 1
          for (int k = 0; k < 8; ++k) f[k] = __fdiv_rn(-f[k], scale);
        }
        uint32_t q[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          q[k] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * k], f[2 * k + 1]), __NV_SATFINITE, __NV_E4M3);
        codes = make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
      }
      if (at[i] >= 0) {
        static_cast<uint2*>(a.cache[w])[at[i] * kTpr + c] = codes;
        if (c == 0) a.scale[w][at[i]] = scale;
      }
    }
}

template <bool kF16, int kD, bool kFp8>
__global__ void __launch_bounds__(kCacheThreads) kv_cache_gather_kernel(const KvCacheArgs a) {
  constexpr int kTpr = kD / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kCacheThreads + threadIdx.x;
  const uint32_t row = static_cast<uint32_t>(i / kTpr);  // below 2^31, as above
  if (row >= static_cast<uint32_t>(a.tokens) * a.heads) return;
  const int t = row / static_cast<uint32_t>(a.heads), h = row % static_cast<uint32_t>(a.heads);
  const int c = static_cast<int>(i % kTpr);
  const int64_t slot = cache_slot(a, t);
  const int64_t at = (slot * a.heads + h) * kTpr + c;
  uint4 out[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (slot >= 0) {
    if (!kFp8) {
#pragma unroll
      for (int w = 0; w < 2; ++w) out[w] = __ldg(static_cast<const uint4*>(a.cache[w]) + at);
    } else {
      uint2 q[2];
      float s[2];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        q[w] = __ldg(static_cast<const uint2*>(a.cache[w]) + at);
        s[w] = __ldg(a.scale[w] + slot * a.heads + h);
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint32_t r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t two = ((k < 2 ? q[w].x : q[w].y) >> (16 * (k & 1))) & 0xffffu;
          const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
          const float2 p = __half22float2(__half2(hr));  // exact: every e4m3 value is an fp16 value
          r[k] = round2<kF16>(p.x * s[w], p.y * s[w]);
        }
        out[w] = make_uint4(r[0], r[1], r[2], r[3]);
      }
    }
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) static_cast<uint4*>(a.y[w])[static_cast<int64_t>(row) * kTpr + c] = out[w];
}

}  // namespace bsk
