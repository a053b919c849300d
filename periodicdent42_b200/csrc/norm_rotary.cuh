// RMS norm of each head of Q and K with the rotation of its pairs in the same pass, and the gradients, for sm_100a: fp16, bf16
// or fp32 rows, weights in the rows' type or fp32.
//
//     xhat = x / rms,  rms = sqrt(mean(x^2) + eps),   z = w xhat,   y = R z    (rotary.cuh: pairs turned by t and scaled by s)
//     dz = R^T dy (turned by -t, the same scale),   g = w dz,   dx = (g - xhat mean(g xhat)) / rms,   dw = sum over rows dz xhat
//
// Everything is fp32 from the loads on; y and dx are rounded once, dw after its sum. The squares of a row may pass fp32's range
// (bf16 and fp32 rows beyond 10^19): then the row is multiplied by 2^-100 first, which changes its rms alone.
//
// A row is held by a group of 4 .. 32 lanes, each with its pairs' both elements, so the two sums of a row are shuffles and the
// row is read once. A group keeps to one token: the angles' sines and cosines and the weights stay in its lanes' registers for
// all of its heads, of which kNormBatch rows are loaded before any is used (and before the angles are taken). The backward
// gives Q and K blocks of their own, so that a thread adds up dw of one weight, walks the tokens with a fixed stride and
// leaves one partial row of dw per block; a second kernel adds those up in a fixed order (no atomics).
//
// Bound: HBM, x read and y written once (backward: x and dy read, dx written).
#pragma once

#include <type_traits>

#include "rotary.cuh"

namespace bsk {

constexpr int kNormThreads = 256;
constexpr int kNormBatch = 4;      // rows of a thread in flight, forward
constexpr int kNormBatchBwd = 2;   // backward: rows of x and of dy

struct NormRotaryArgs {
  const void* x[2];                // Q, K (either may be absent: 0 heads)
  void* y[2];                      // forward: results; backward: dx; contiguous [tokens, heads, dim]
  const void* dy[2];               // backward: gradients of the results
  const void* w[2];                // [dim]
  int64_t token_stride[2], head_stride[2];        // of x, in elements
  int64_t dy_token_stride[2], dy_head_stride[2];  // of dy
  int heads[2];
  int w_f32;                       // weights are fp32 (else of the rows' type)
  const void* positions;
  int positions64;
  const int* axes;
  int num_axes;
  const float* inv_freq;
  int tokens, dim, rotary_dim;
  float scale, eps;
  int aligned32;                   // every row starts at a multiple of 32 bytes
  int group, units;                // lanes and units of a row
  int at_once[2], per_block[2];    // heads of a token side by side, tokens of a block (forward: [0], for Q and K together)
  float* partial;                  // backward: [blocks of Q, then of K][dim]
  int blocks_q;
  uint32_t* err;
};

// Unit u of a head: kVec pairs (or, in the part that is not turned, 2 kVec elements), as two pieces of kVec elements.
template <int kVec, bool kInter>
struct NormUnit {
  int e0, e1, pair;
  bool turned, live, joined;  // joined: the two pieces are neighbours
  __device__ __forceinline__ NormUnit(int u, int units, int half) {
    live = u < units;
    pair = live ? u * kVec : 0;
    turned = live && pair < half;
    joined = kInter || !turned;
    e0 = joined ? 2 * pair : pair;
    e1 = joined ? e0 + kVec : pair + half;
  }
};

__device__ __forceinline__ float group_sum(float v, int group) {
  for (int o = group >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <class T, int kVec>
__device__ __forceinline__ void unpack_pieces(const Pack<T, kVec>& p, const Pack<T, kVec>& q, float (&f)[2 * kVec]) {
#pragma unroll
  for (int k = 0; k < kVec; ++k) {
    f[k] = to_f32<T>(p.v[k]);
    f[kVec + k] = to_f32<T>(q.v[k]);
  }
}

// Turned pairs of a unit in place: (a, b) -> (a c - b s, a s + b c); kBack: the other way.
template <int kVec, bool kInter, bool kBack>
__device__ __forceinline__ void turn_pieces(float (&f)[2 * kVec], const float2 (&rot)[kVec]) {
#pragma unroll
  for (int k = 0; k < kVec; ++k) {
    const int ia = kInter ? 2 * k : k, ib = kInter ? 2 * k + 1 : kVec + k;
    const float va = f[ia], vb = f[ib], c = rot[k].x, s = kBack ? -rot[k].y : rot[k].y;
    f[ia] = va * c - vb * s;
    f[ib] = va * s + vb * c;
  }
}

template <class T>
__device__ __forceinline__ float weight_at(const NormRotaryArgs& a, int w, int e) {
  return a.w_f32 ? __ldg(static_cast<const float*>(a.w[w]) + e) : to_f32<T>(static_cast<const T*>(a.w[w])[e]);
}

// (cos, sin) * scale of `count` tokens from t0 on: [token][pair].
__device__ __forceinline__ void norm_angles(const NormRotaryArgs& a, int64_t t0, int count, float2* rot) {
  const int half = a.rotary_dim / 2;
  for (int i = threadIdx.x; i < count * half; i += kNormThreads) {
    const int it = i / half, pair = i - it * half;
    const int64_t at = position_of(a.positions, a.positions64, a.axes, a.num_axes, a.tokens, t0 + it, pair, a.err);
    float s, c;
    sincospif(2.0f * static_cast<float>(turn_fraction(at, a.inv_freq[pair])), &s, &c);
    rot[i] = make_float2(c * a.scale, s * a.scale);
  }
}

// Rows whose squares pass fp32's range are scaled down by this first.
constexpr float kNormDown = 0x1p-100f;

// kUnits units per lane: units group * p + lane for p < kUnits.
template <class T, int kVec, int kUnits, bool kInter>
__global__ void __launch_bounds__(kNormThreads) norm_rotary_kernel(const __grid_constant__ NormRotaryArgs a) {
  extern __shared__ float2 rot_s[];
  using P = Pack<T, kVec>;
  using Unit = NormUnit<kVec, kInter>;
  const int half = a.rotary_dim / 2;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.per_block[0];
  const int nt = static_cast<int>(min(static_cast<int64_t>(a.per_block[0]), a.tokens - t0));
  const int lane = threadIdx.x & (a.group - 1), g = threadIdx.x / a.group;
  const int at_once = a.at_once[0], it = g / at_once, h0 = g - it * at_once;
  const int all_heads = a.heads[0] + a.heads[1];
  const int rows = it < nt ? all_heads : 0;
  P p[kNormBatch][kUnits], q[kNormBatch][kUnits];
  auto load = [&](int first) {
#pragma unroll
    for (int b = 0; b < kNormBatch; ++b) {
      const int row = first + b * at_once;
      const int w = row >= a.heads[0], h = w ? row - a.heads[0] : row;
      const T* x = static_cast<const T*>(a.x[w]) + (t0 + it) * a.token_stride[w] + h * a.head_stride[w];
#pragma unroll
      for (int n = 0; n < kUnits; ++n) {
        const Unit u(a.group * n + lane, a.units, half);
        if (row < rows && u.live) {
          load_pair(x + u.e0, x + u.e1, a.aligned32 && u.joined, p[b][n], q[b][n]);
        } else {
          p[b][n] = P{};
          q[b][n] = P{};
        }
      }
    }
  };
  load(h0);
  norm_angles(a, t0, nt, rot_s);
  __syncthreads();
  float2 rot[kUnits][kVec];
  float weight[2][kUnits][2 * kVec];
#pragma unroll
  for (int n = 0; n < kUnits; ++n) {
    const Unit u(a.group * n + lane, a.units, half);
#pragma unroll
    for (int k = 0; k < kVec; ++k) rot[n][k] = u.turned && rows ? rot_s[it * half + u.pair + k] : make_float2(1.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        weight[w][n][k] = a.heads[w] && u.live ? weight_at<T>(a, w, u.e0 + k) : 0.0f;
        weight[w][n][kVec + k] = a.heads[w] && u.live ? weight_at<T>(a, w, u.e1 + k) : 0.0f;
      }
  }
  const float inv_dim = 1.0f / static_cast<float>(a.dim);
  // (every lane of a warp takes part in every sum: the loop's length is the same for all)
  const int rounds = (all_heads + kNormBatch * at_once - 1) / (kNormBatch * at_once);
  for (int round = 0; round < rounds; ++round) {
    const int first = h0 + round * kNormBatch * at_once;
    if (round) load(first);
#pragma unroll
    for (int b = 0; b < kNormBatch; ++b) {
      const int row = first + b * at_once;
      const int w = row >= a.heads[0], h = w ? row - a.heads[0] : row;
      float f[kUnits][2 * kVec], ss = 0.0f;
#pragma unroll
      for (int n = 0; n < kUnits; ++n) {
        unpack_pieces<T, kVec>(p[b][n], q[b][n], f[n]);
#pragma unroll
        for (int k = 0; k < 2 * kVec; ++k) ss = fmaf(f[n][k], f[n][k], ss);
      }
      ss = group_sum(ss, a.group);
      float eps = a.eps;
      if constexpr (sizeof(T) != 2 || !std::is_same<T, __half>::value) {
        const bool far = !(ss <= 3.0e38f);
        if (__any_sync(0xffffffffu, far)) {
          const float down = far ? kNormDown : 1.0f;
          ss = 0.0f;
#pragma unroll
          for (int n = 0; n < kUnits; ++n)
#pragma unroll
            for (int k = 0; k < 2 * kVec; ++k) {
              f[n][k] *= down;
              ss = fmaf(f[n][k], f[n][k], ss);
            }
          ss = group_sum(ss, a.group);
          if (far) eps = 0.0f;
        }
      }
      const float inv = rsqrtf(fmaf(ss, inv_dim, eps));
      if (row >= rows) continue;
      T* y = static_cast<T*>(a.y[w]) + ((t0 + it) * a.heads[w] + h) * a.dim;
#pragma unroll
      for (int n = 0; n < kUnits; ++n) {
        const Unit u(a.group * n + lane, a.units, half);
        if (!u.live) continue;
#pragma unroll
        for (int k = 0; k < 2 * kVec; ++k) f[n][k] *= inv * (w ? weight[1][n][k] : weight[0][n][k]);
        if (u.turned) turn_pieces<kVec, kInter, false>(f[n], rot[n]);
        P po, qo;
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          po.v[k] = from_f32<T>(f[n][k]);
          qo.v[k] = from_f32<T>(f[n][kVec + k]);
        }
        store_pair(y + u.e0, y + u.e1, a.aligned32 && u.joined, po, qo);
      }
    }
  }
}

template <class T, int kVec, int kUnits, bool kInter>
__global__ void __launch_bounds__(kNormThreads) norm_rotary_bwd_kernel(const __grid_constant__ NormRotaryArgs a) {
  extern __shared__ float2 rot_s[];  // (cos, sin) of a chunk's tokens; at the end the groups' sums of dw
  ptx::grid_launch_dependents();
  using P = Pack<T, kVec>;
  using Unit = NormUnit<kVec, kInter>;
  const int half = a.rotary_dim / 2;
  const int w = static_cast<int>(blockIdx.x) >= a.blocks_q;
  const int block = w ? blockIdx.x - a.blocks_q : blockIdx.x, blocks = w ? gridDim.x - a.blocks_q : a.blocks_q;
  const int heads = a.heads[w];
  const int lane = threadIdx.x & (a.group - 1), g = threadIdx.x / a.group, groups = kNormThreads / a.group;
  const int at_once = a.at_once[w], tokens_per_block = a.per_block[w];
  const int it = g / at_once, h0 = g - it * at_once;
  const T* xs = static_cast<const T*>(a.x[w]);
  const T* dys = static_cast<const T*>(a.dy[w]);
  float weight[kUnits][2 * kVec], dw[kUnits][2 * kVec];
#pragma unroll
  for (int n = 0; n < kUnits; ++n) {
    const Unit u(a.group * n + lane, a.units, half);
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      weight[n][k] = u.live ? weight_at<T>(a, w, u.e0 + k) : 0.0f;
      weight[n][kVec + k] = u.live ? weight_at<T>(a, w, u.e1 + k) : 0.0f;
      dw[n][k] = dw[n][kVec + k] = 0.0f;
    }
  }
  const float inv_dim = 1.0f / static_cast<float>(a.dim);
  const int rounds = (heads + kNormBatchBwd * at_once - 1) / (kNormBatchBwd * at_once);
  const int64_t chunks = (static_cast<int64_t>(a.tokens) + tokens_per_block - 1) / tokens_per_block;
  for (int64_t chunk = block; chunk < chunks; chunk += blocks) {
    const int64_t t0 = chunk * tokens_per_block, t = t0 + it;
    const int nt = static_cast<int>(min(static_cast<int64_t>(tokens_per_block), a.tokens - t0));
    const int rows = it < nt ? heads : 0;
    P xp[kNormBatchBwd][kUnits], xq[kNormBatchBwd][kUnits], dp[kNormBatchBwd][kUnits], dq[kNormBatchBwd][kUnits];
    auto load = [&](int first) {
#pragma unroll
      for (int b = 0; b < kNormBatchBwd; ++b) {
        const int h = first + b * at_once;
        const T* x = xs + t * a.token_stride[w] + h * a.head_stride[w];
        const T* dy = dys + t * a.dy_token_stride[w] + h * a.dy_head_stride[w];
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
          const Unit u(a.group * n + lane, a.units, half);
          if (h < rows && u.live) {
            load_pair(x + u.e0, x + u.e1, a.aligned32 && u.joined, xp[b][n], xq[b][n]);
            load_pair(dy + u.e0, dy + u.e1, a.aligned32 && u.joined, dp[b][n], dq[b][n]);
          } else {
            xp[b][n] = xq[b][n] = dp[b][n] = dq[b][n] = P{};
          }
        }
      }
    };
    load(h0);
    __syncthreads();  // the chunk before has read its angles
    norm_angles(a, t0, nt, rot_s);
    __syncthreads();
    float2 rot[kUnits][kVec];
#pragma unroll
    for (int n = 0; n < kUnits; ++n) {
      const Unit u(a.group * n + lane, a.units, half);
#pragma unroll
      for (int k = 0; k < kVec; ++k) rot[n][k] = u.turned && rows ? rot_s[it * half + u.pair + k] : make_float2(1.0f, 0.0f);
    }
    for (int round = 0; round < rounds; ++round) {
      const int first = h0 + round * kNormBatchBwd * at_once;
      if (round) load(first);
#pragma unroll
      for (int b = 0; b < kNormBatchBwd; ++b) {
        const int h = first + b * at_once;
        float x[kUnits][2 * kVec], dz[kUnits][2 * kVec], ss = 0.0f, dot = 0.0f;
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
          const Unit u(a.group * n + lane, a.units, half);
          unpack_pieces<T, kVec>(xp[b][n], xq[b][n], x[n]);
          unpack_pieces<T, kVec>(dp[b][n], dq[b][n], dz[n]);
          if (u.turned) turn_pieces<kVec, kInter, true>(dz[n], rot[n]);
#pragma unroll
          for (int k = 0; k < 2 * kVec; ++k) ss = fmaf(x[n][k], x[n][k], ss);
        }
        ss = group_sum(ss, a.group);
        float eps = a.eps, down = 1.0f;
        if constexpr (sizeof(T) != 2 || !std::is_same<T, __half>::value) {
          const bool far = !(ss <= 3.0e38f);
          if (__any_sync(0xffffffffu, far)) {
            down = far ? kNormDown : 1.0f;
            ss = 0.0f;
#pragma unroll
            for (int n = 0; n < kUnits; ++n)
#pragma unroll
              for (int k = 0; k < 2 * kVec; ++k) {
                x[n][k] *= down;
                ss = fmaf(x[n][k], x[n][k], ss);
              }
            ss = group_sum(ss, a.group);
            if (far) eps = 0.0f;
          }
        }
        const float inv = rsqrtf(fmaf(ss, inv_dim, eps));
#pragma unroll
        for (int n = 0; n < kUnits; ++n)
#pragma unroll
          for (int k = 0; k < 2 * kVec; ++k) {
            x[n][k] *= inv;  // xhat
            dw[n][k] = fmaf(dz[n][k], x[n][k], dw[n][k]);
            dz[n][k] *= weight[n][k];  // g
            dot = fmaf(dz[n][k], x[n][k], dot);
          }
        dot = group_sum(dot, a.group) * inv_dim;
        if (h >= rows) continue;
        T* y = static_cast<T*>(a.y[w]) + (t * heads + h) * a.dim;
        const float out = inv * down;
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
          const Unit u(a.group * n + lane, a.units, half);
          if (!u.live) continue;
          P po, qo;
#pragma unroll
          for (int k = 0; k < kVec; ++k) {
            po.v[k] = from_f32<T>((dz[n][k] - x[n][k] * dot) * out);
            qo.v[k] = from_f32<T>((dz[n][kVec + k] - x[n][kVec + k] * dot) * out);
          }
          store_pair(y + u.e0, y + u.e1, a.aligned32 && u.joined, po, qo);
        }
      }
    }
  }
  // the groups' sums, added in order
  float* sums = reinterpret_cast<float*>(rot_s);
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kUnits; ++n) {
    const Unit u(a.group * n + lane, a.units, half);
    if (!u.live) continue;
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      sums[g * a.dim + u.e0 + k] = dw[n][k];
      sums[g * a.dim + u.e1 + k] = dw[n][kVec + k];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.dim; e += kNormThreads) {
    float s = 0.0f;
    for (int i = 0; i < groups; ++i) s += sums[i * a.dim + e];
    a.partial[static_cast<int64_t>(blockIdx.x) * a.dim + e] = s;
  }
}

// dw: the blocks' rows added up in a fixed order, 32 columns per block, 16 threads a column.
struct NormWeightArgs {
  const float* partial;
  void* dw[2];           // may be nullptr
  int first[2], count[2];  // rows of partial
  int dim, w_f32;
};
constexpr int kNormWeightRows = 16;

template <class T>
__global__ void __launch_bounds__(32 * kNormWeightRows) norm_weight_kernel(const NormWeightArgs a) {
  __shared__ float part[kNormWeightRows][33];
  ptx::grid_dependency_wait();
  const int w = blockIdx.y, e = blockIdx.x * 32 + threadIdx.x % 32, r0 = threadIdx.x / 32;
  if (!a.dw[w]) return;
  float s = 0.0f;
  if (e < a.dim)
    for (int r = r0; r < a.count[w]; r += kNormWeightRows) s += a.partial[static_cast<int64_t>(a.first[w] + r) * a.dim + e];
  part[r0][threadIdx.x % 32] = s;
  __syncthreads();
  if (r0 || e >= a.dim) return;
  s = 0.0f;
#pragma unroll
  for (int r = 0; r < kNormWeightRows; ++r) s += part[r][threadIdx.x];
  if (a.w_f32) static_cast<float*>(a.dw[w])[e] = s;
  else static_cast<T*>(a.dw[w])[e] = from_f32<T>(s);
}

}  // namespace bsk
