// Rotary positions for sm_100a: fp16, bf16 or fp32 rows of Q and K in one launch.
//
// Pair i of a head, (a, b) = (x[2i], x[2i+1]) in the interleaved layout or (x[i], x[i + r/2]) in the half layout, is
// turned by the angle t = position * inv_freq[i] and scaled:
//     y_a = s (a cos t - b sin t),   y_b = s (a sin t + b cos t);   elements from r on are copied.
// The gradient of a rotation is the rotation by -t with the same scale, so the backward pass is this kernel with
// `sign` = -1.
//
// Precision: a position of 10^6 leaves an fp32 angle 0.03 radians off, so the angle is taken in turns (t / 2 pi) in
// 64 bits, its whole turns are dropped there, and only the remaining fraction of a turn goes to sincospif. A 64-bit product
// would in turn be 2^-52 of its turns off (2^-14 radians at position 2^40), so what its roundings drop is kept as a second
// 64-bit number: the fraction is exact to 2^-43 of a turn for every 64-bit position. The rotation itself is fp32 and each
// result is rounded once.
//
// Bound: HBM, each row is read and written once. The angles cost one double product and one sincospif per (token,
// pair): they are taken once per token by the block, kept in shared memory and used by all heads of Q and K. The rows of
// a block (its tokens' heads of Q, then of K) are dealt out to groups of threads, a thread keeping its place within the
// head (its VEC pairs: 32 bytes of a 16-byte-aligned row); kRotaryBatch rows per thread are loaded before the angles
// are taken and before any is stored, so that enough loads are in flight, and neighbouring pieces move as one 32-byte
// access (16383 tokens of 32 + 8 heads, D 128, bf16, half of the head turned, interleaved: 60 us a pass, 5.6 TB/s; in
// 16-byte accesses 108; one row at a time 89; all of the head turned, either layout: 70..73, 4.7 TB/s).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx_sm100.cuh"

namespace bsk {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryMaxDim = 512;
constexpr int kRotaryBatch = 4;

struct RotaryArgs {
  const void* x[2];       // Q, K (K may be absent: heads[1] = 0)
  void* y[2];             // contiguous [tokens, heads, dim]
  int64_t token_stride[2], head_stride[2];  // of x, in elements
  int heads[2];
  const void* positions;  // int32 or int64 [tokens]
  int positions64;
  const float* inv_freq;  // [rotary_dim / 2]
  int tokens, dim, rotary_dim;
  float scale, sign;
  int aligned32;          // every row of x and y starts at a multiple of 32 bytes
};

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// position * frequency / 2 pi without its whole turns, in (-1, 1). Each number is a 64-bit one and what its rounding dropped.
__device__ __forceinline__ double turn_fraction(int64_t position, float frequency) {
  constexpr double kInv2Pi = 0.15915494309189535, kInv2PiLow = -9.839338337591243e-18;  // 1 / 2 pi to 107 bits
  const double f = frequency;
  const double g = f * kInv2Pi, g_low = fma(f, kInv2PiLow, fma(f, kInv2Pi, -g));  // turns per position
  const double p = static_cast<double>(position);
  // (positions above 2^53; the largest ones round to 2^63, which no int64 holds)
  const double p_low = p < 0x1p63 ? static_cast<double>(position - static_cast<int64_t>(p))
                                  : static_cast<double>(position - INT64_MAX) - 1.0;
  const double t = p * g, t_low = fma(p_low, g, fma(p, g_low, fma(p, g, -t)));
  return (t - rint(t)) + (t_low - rint(t_low));
}

template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// A thread's two pieces of a row: 16 bytes each, one 32-byte access where they are neighbours and aligned to it.
template <class P>
__device__ __forceinline__ void load_pair(const void* x0, const void* x1, bool joined, P& p, P& q) {
  if constexpr (sizeof(P) == 16) {
    if (joined) {
      uint32_t r[8];
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                   : "l"(x0)
                   : "memory");
      memcpy(&p, r, 16);
      memcpy(&q, r + 4, 16);
      return;
    }
  }
  p = *static_cast<const P*>(x0);
  q = *static_cast<const P*>(x1);
}
template <class P>
__device__ __forceinline__ void store_pair(void* y0, void* y1, bool joined, const P& p, const P& q) {
  if constexpr (sizeof(P) == 16) {
    if (joined) {
      uint32_t r[8];
      memcpy(r, &p, 16);
      memcpy(r + 4, &q, 16);
      st_global_v8(y0, r);
      return;
    }
  }
  *static_cast<P*>(y0) = p;
  *static_cast<P*>(y1) = q;
}

// kVec pairs per thread: 16 / sizeof(T) where rows, strides and the halves allow 16-byte accesses, else 1.
template <class T, int kVec, bool kInterleaved>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryArgs a, int tokens_per_block) {
  extern __shared__ float2 rot[];  // [tokens_per_block][rotary_dim / 2] (cos, sin) * scale
  const int half = a.rotary_dim / 2;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * tokens_per_block;
  const int nt = static_cast<int>(min(static_cast<int64_t>(tokens_per_block), a.tokens - t0));

  using P = Pack<T, kVec>;
  const int units = a.dim / (2 * kVec);           // threads per head row
  const int groups = kRotaryThreads / units;      // rows in flight per block
  const int u = threadIdx.x % units, g0 = threadIdx.x / units;
  const int all_heads = a.heads[0] + a.heads[1];
  const int rows = g0 < groups ? nt * all_heads : 0;  // (threads left over have none)
  const int pair = u * kVec;                      // first pair (or first pair-sized piece of the copied part)
  const bool turned = pair < half;
  const int e0 = (kInterleaved || !turned) ? 2 * pair : pair;
  const int e1 = (kInterleaved || !turned) ? e0 + kVec : pair + half;

  const bool joined = a.aligned32 && (kInterleaved || !turned);
  P p[kRotaryBatch], q[kRotaryBatch];
  auto load = [&](int first) {
#pragma unroll
    for (int b = 0; b < kRotaryBatch; ++b) {
      const int row = first + b * groups;
      if (row >= rows) break;
      const int it = row / all_heads, h = row - it * all_heads, w = h >= a.heads[0];
      const T* x = static_cast<const T*>(a.x[w]) + (t0 + it) * a.token_stride[w] + (w ? h - a.heads[0] : h) * a.head_stride[w];
      load_pair(x + e0, x + e1, joined, p[b], q[b]);
    }
  };
  load(g0);
  for (int i = threadIdx.x; i < nt * half; i += kRotaryThreads) {
    const int64_t t = t0 + i / half;
    const int64_t at = a.positions64 ? static_cast<const int64_t*>(a.positions)[t] : static_cast<const int*>(a.positions)[t];
    const double turn = turn_fraction(at, a.inv_freq[i % half]);
    float s, c;
    sincospif(2.0f * static_cast<float>(turn), &s, &c);
    rot[i] = make_float2(c * a.scale, a.sign * s * a.scale);
  }
  __syncthreads();

  for (int first = g0; first < rows; first += kRotaryBatch * groups) {
    if (first != g0) load(first);
#pragma unroll
    for (int b = 0; b < kRotaryBatch; ++b) {
      const int row = first + b * groups;
      if (row >= rows) break;
      const int it = row / all_heads, h = row - it * all_heads, w = h >= a.heads[0];
      T* y = static_cast<T*>(a.y[w]) + ((t0 + it) * a.heads[w] + (w ? h - a.heads[0] : h)) * a.dim;
      P po = p[b], qo = q[b];
      if (turned) {
        T in[2 * kVec], out[2 * kVec];
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          in[k] = p[b].v[k];
          in[kVec + k] = q[b].v[k];
        }
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          const float2 r = rot[it * half + pair + k];
          const int ia = kInterleaved ? 2 * k : k, ib = kInterleaved ? 2 * k + 1 : kVec + k;
          const float va = to_f32<T>(in[ia]), vb = to_f32<T>(in[ib]);
          out[ia] = from_f32<T>(va * r.x - vb * r.y);
          out[ib] = from_f32<T>(va * r.y + vb * r.x);
        }
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          po.v[k] = out[k];
          qo.v[k] = out[kVec + k];
        }
      }
      store_pair(y + e0, y + e1, joined, po, qo);
    }
  }
}

}  // namespace bsk
