// Rotary positions for sm_100a: fp16, bf16 or fp32 rows of Q and K in one launch.
//
// Pair i of a head, (a, b) = (x[2i], x[2i+1]) in the interleaved layout or (x[i], x[i + r/2]) in the half layout, is
// turned by the angle t = position * inv_freq[i] and scaled:
//     y_a = s (a cos t - b sin t),   y_b = s (a sin t + b cos t);   elements from r on are copied.
// The gradient of a rotation is the rotation by -t with the same scale, so the backward pass is this kernel with
// `sign` = -1.
//
// Precision: a position of 10^6 leaves an fp32 angle 0.03 radians off, so the angle is taken in turns (t / 2 pi) in
// 64 bits, its whole turns are dropped there, and only the remaining fraction of a turn goes to sincospif. The
// rotation itself is fp32 and each result is rounded once.
//
// Bound: HBM, each row is read and written once. The angles cost one double product and one sincospif per (token,
// pair): they are taken once per token by the block, kept in shared memory and used by all heads of Q and K. A thread
// keeps its place within the head (its VEC pairs: 32 bytes of a 16-byte-aligned row) and walks over heads, so the
// cosines stay in registers and there is no division in the loop.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx_sm100.cuh"

namespace bsk {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryMaxDim = 512;

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

template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// kVec pairs per thread: 16 / sizeof(T) where rows, strides and the halves allow 16-byte accesses, else 1.
template <class T, int kVec, bool kInterleaved>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryArgs a, int tokens_per_block) {
  extern __shared__ float2 rot[];  // [tokens_per_block][rotary_dim / 2] (cos, sin) * scale
  const int half = a.rotary_dim / 2;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * tokens_per_block;
  const int nt = static_cast<int>(min(static_cast<int64_t>(tokens_per_block), a.tokens - t0));
  for (int i = threadIdx.x; i < nt * half; i += kRotaryThreads) {
    const int64_t t = t0 + i / half;
    const double pos = a.positions64 ? static_cast<double>(static_cast<const int64_t*>(a.positions)[t])
                                     : static_cast<double>(static_cast<const int*>(a.positions)[t]);
    const double turns = pos * (static_cast<double>(a.inv_freq[i % half]) * 0.15915494309189533577);  // 1 / 2 pi
    float s, c;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
    rot[i] = make_float2(c * a.scale, a.sign * s * a.scale);
  }
  __syncthreads();

  using P = Pack<T, kVec>;
  const int units = a.dim / (2 * kVec);          // threads per head row
  const int rows = kRotaryThreads / units;       // heads in flight per block
  const int u = threadIdx.x % units, h0 = threadIdx.x / units;
  if (h0 >= rows) return;
  const int pair = u * kVec;                     // first pair (or first pair-sized piece of the copied part)
  const bool turned = pair < half;
  const int e0 = (kInterleaved || !turned) ? 2 * pair : pair;
  const int e1 = (kInterleaved || !turned) ? e0 + kVec : pair + half;
  for (int it = 0; it < nt; ++it) {
    const int64_t t = t0 + it;
    float c[kVec], s[kVec];
    if (turned) {
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        const float2 r = rot[it * half + pair + k];
        c[k] = r.x;
        s[k] = r.y;
      }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const T* x = static_cast<const T*>(a.x[w]) + t * a.token_stride[w];
      T* y = static_cast<T*>(a.y[w]) + t * a.heads[w] * a.dim;
#pragma unroll 4
      for (int h = h0; h < a.heads[w]; h += rows) {
        const T* xr = x + h * a.head_stride[w];
        T* yr = y + static_cast<int64_t>(h) * a.dim;
        P p = *reinterpret_cast<const P*>(xr + e0), q = *reinterpret_cast<const P*>(xr + e1);
        if (turned) {
          T in[2 * kVec], out[2 * kVec];
#pragma unroll
          for (int k = 0; k < kVec; ++k) {
            in[k] = p.v[k];
            in[kVec + k] = q.v[k];
          }
#pragma unroll
          for (int k = 0; k < kVec; ++k) {
            const int ia = kInterleaved ? 2 * k : k, ib = kInterleaved ? 2 * k + 1 : kVec + k;
            const float va = to_f32<T>(in[ia]), vb = to_f32<T>(in[ib]);
            out[ia] = from_f32<T>(va * c[k] - vb * s[k]);
            out[ib] = from_f32<T>(va * s[k] + vb * c[k]);
          }
#pragma unroll
          for (int k = 0; k < kVec; ++k) {
            p.v[k] = out[k];
            q.v[k] = out[kVec + k];
          }
        }
        *reinterpret_cast<P*>(yr + e0) = p;
        *reinterpret_cast<P*>(yr + e1) = q;
      }
    }
  }
}

}  // namespace bsk
