// Attention over packed sequences with grouped heads, forward and backward: one warp per row, written for clearness.
//   forward  (per query row):  s_j = scale q.k_j,  O = sum_j softmax(s)_j v_j,  lse = log sum_j e^{s_j}
//   dQ       (per query row):  dS_j = P_j (dO.v_j - dO.O),  dQ = scale sum_j dS_j k_j
//   dK, dV   (per key row of one kv head): the sums over the rows of all heads of its group and all queries that see it
#pragma once

#include "paged_decode_sm100.cuh"

namespace bsk {

struct VarlenArgs {
  const void *Q, *K, *V, *dO, *O_in;
  void *O, *dQ, *dK, *dV;
  float* lse;  // [tokens, heads] natural log
  const int* cu;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, do_ts, do_hs;
  int tokens, batch, heads, kv_heads, group, causal;
  float scale;
  uint32_t* err;
};

template <bool kF16, int N>
__device__ __forceinline__ void load_row(const void* p, int64_t off, float (&f)[N]) {
  const uint16_t* x = static_cast<const uint16_t*>(p) + off;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 v = unpack2<kF16>(*reinterpret_cast<const uint32_t*>(x + i));
    f[i] = v.x;
    f[i + 1] = v.y;
  }
}
template <int N>
__device__ __forceinline__ float dot_row(const float (&a)[N], const float (&b)[N]) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) s = fmaf(a[i], b[i], s);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
template <bool kF16, int N>
__device__ __forceinline__ void store_row(void* p, int64_t off, const float (&f)[N], float mul) {
  uint16_t* x = static_cast<uint16_t*>(p) + off;
#pragma unroll
  for (int i = 0; i < N; i += 2) *reinterpret_cast<uint32_t*>(x + i) = round2<kF16>(f[i] * mul, f[i + 1] * mul);
}

// mode 0: forward, 1: dQ, 2: dK and dV
template <bool kF16, int kD, int kMode>
__global__ void __launch_bounds__(128) varlen_simple_kernel(const VarlenArgs a) {
  constexpr int N = kD / 32;
  const int lane = threadIdx.x & 31;
  const int nh = kMode == 2 ? a.kv_heads : a.heads;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (w >= static_cast<int64_t>(a.tokens) * nh) return;
  const int t = static_cast<int>(w / nh), h = static_cast<int>(w % nh);
  int seq = 0;
  while (seq < a.batch && t >= __ldg(&a.cu[seq + 1])) ++seq;
  int lo = 0, hi = 0;
  bool bad = false;
  if (seq < a.batch) seq_rows(a.cu, seq, a.tokens, lo, hi, bad);
  if (w == 0)
    for (int i = lane; i < a.batch; i += 32) {
      int x, y;
      bool wrong;
      seq_rows(a.cu, i, a.tokens, x, y, wrong);
      if (wrong) paged_flag(a.err, 4);
    }
  const int d = lane * N;
  if (kMode == 0) {
    float q[N], o[N] = {}, m = -INFINITY, l = 0.0f;
    load_row<kF16>(a.Q, t * a.q_ts + h * a.q_hs + d, q);
    const int g = h / a.group, end = a.causal ? min(t + 1, hi) : hi;
    for (int j = lo; j < end; ++j) {
      float k[N], v[N];
      load_row<kF16>(a.K, j * a.k_ts + g * a.k_hs + d, k);
      load_row<kF16>(a.V, j * a.v_ts + g * a.v_hs + d, v);
      const float s = dot_row(q, k) * a.scale;
      const float mn = fmaxf(m, s), al = expf(m - mn), p = expf(s - mn);
      m = mn;
      l = l * al + p;
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = fmaf(p, v[i], o[i] * al);
    }
    store_row<kF16>(a.O, (static_cast<int64_t>(t) * a.heads + h) * kD + d, o, l > 0.0f ? 1.0f / l : 0.0f);
    if (a.lse && lane == 0) a.lse[static_cast<int64_t>(t) * a.heads + h] = l > 0.0f ? m + logf(l) : -INFINITY;
  } else if (kMode == 1) {
    float q[N], go[N], o[N], dq[N] = {};
    const int64_t at = static_cast<int64_t>(t) * a.heads + h;
    load_row<kF16>(a.Q, t * a.q_ts + h * a.q_hs + d, q);
    load_row<kF16>(a.dO, t * a.do_ts + h * a.do_hs + d, go);
    load_row<kF16>(a.O_in, at * kD + d, o);
    const float delta = dot_row(go, o), lse = a.lse[at];
    const int g = h / a.group, end = a.causal ? min(t + 1, hi) : hi;
    for (int j = lo; j < end; ++j) {
      float k[N], v[N];
      load_row<kF16>(a.K, j * a.k_ts + g * a.k_hs + d, k);
      load_row<kF16>(a.V, j * a.v_ts + g * a.v_hs + d, v);
      const float ds = expf(dot_row(q, k) * a.scale - lse) * (dot_row(go, v) - delta);
#pragma unroll
      for (int i = 0; i < N; ++i) dq[i] = fmaf(ds, k[i], dq[i]);
    }
    store_row<kF16>(a.dQ, at * kD + d, dq, a.scale);
  } else {
    float k[N], v[N], dk[N] = {}, dv[N] = {};
    load_row<kF16>(a.K, t * a.k_ts + h * a.k_hs + d, k);
    load_row<kF16>(a.V, t * a.v_ts + h * a.v_hs + d, v);
    for (int j = a.causal ? t : lo; j < hi; ++j)
      for (int x = h * a.group; x < (h + 1) * a.group; ++x) {
        float q[N], go[N], o[N];
        const int64_t at = static_cast<int64_t>(j) * a.heads + x;
        load_row<kF16>(a.Q, j * a.q_ts + x * a.q_hs + d, q);
        load_row<kF16>(a.dO, j * a.do_ts + x * a.do_hs + d, go);
        load_row<kF16>(a.O_in, at * kD + d, o);
        const float p = expf(dot_row(q, k) * a.scale - a.lse[at]), ds = p * (dot_row(go, v) - dot_row(go, o));
#pragma unroll
        for (int i = 0; i < N; ++i) {
          dk[i] = fmaf(ds, q[i], dk[i]);
          dv[i] = fmaf(p, go[i], dv[i]);
        }
      }
    const int64_t at = (static_cast<int64_t>(t) * a.kv_heads + h) * kD + d;
    store_row<kF16>(a.dK, at, dk, a.scale);
    store_row<kF16>(a.dV, at, dv, 1.0f);
  }
}

}  // namespace bsk
