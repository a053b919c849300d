// RMS norm of each head of Q and K with the rotation of its pairs in the same pass, and the gradients, for sm_100a: fp16, bf16
// or fp32 rows, weights in the rows' type or fp32.
//
//     xhat = x / rms,  rms = sqrt(mean(x^2) + eps),   z = w xhat,   y = R z    (rotary.cuh: pairs turned by t and scaled by s)
//     dz = R^T dy (turned by -t, the same scale),   g = w dz,   dx = (g - xhat mean(g xhat)) / rms,   dw = sum over rows dz xhat
//
// Everything is fp32 from the loads on; y and dx are rounded once, dw after its sum. The squares of a row may pass fp32's range
// (bf16 and fp32 rows beyond 10^19): then the row is multiplied by 2^-100 first, which changes its rms alone.
//
// The same kernel without the norm (kNorm) turns by positions on several axes. (The one-axis rotation has rotary.cuh's kernel,
// whose results it keeps bit for bit where all axes agree.)
//
// A row is held by a group of 1 .. 32 lanes, each with its pairs' both elements, so the two sums of a row are shuffles and the
// row is read once. A group keeps to one token: the angles' sines and cosines and the weights stay in its lanes' registers for
// all of its heads. The blocks are as many as fit on the SMs, some for Q and the others for K; each walks the tokens with a fixed
// stride. Rows come through a ring of asynchronous copies in shared memory that each thread fills for itself, kNormBatch rows
// (backward: kNormBatchBwd of x and of dy) a stage: the next stages, of the next token too, are on their way while one is used,
// and no thread waits for another's. A thread adds up dw of its own weights and a block leaves one partial row; a second kernel
// adds those up in a fixed order (no atomics).
//
// Bound: HBM at first, x read and y written once (backward: x and dy read, dx written), then issue slots: the packed two-float
// instructions halve the arithmetic, and what is left still takes about half of all slots. 16383 tokens, 32 + 8 heads of 128, us
// (TB/s): bf16 forward 64 (5.2), both ways 163 (5.2); the rotation alone on three axes 60 (5.6); fp32 both ways 266 (6.3).
#pragma once

#include <type_traits>

#include "gemm_sm100.cuh"
#include "bsattn_bwd_sm100.cuh"
#include "rotary.cuh"

namespace bsk {

constexpr int kNormThreads = 256;
constexpr int kNormMostBlocks = 6;  // on an SM
constexpr int kNormBatch = 4;     // rows of a thread's step, forward
constexpr int kNormBatchBwd = 2;  // backward: rows of x and of dy

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
  float scale, sign, eps;          // sign: of the angles
  int group, units;                // lanes and units of a row
  int at_once[2], per_block[2];    // heads of a token side by side, tokens of a chunk
  int grid, blocks_q;              // blocks, and those of them that take Q; the others take K
  float* partial;                  // backward: [blocks][dim]
  uint32_t* err;
};

// Unit u of a head: kVec pairs (or, in the part that is not turned, 2 kVec elements), as two pieces of kVec elements, each beside
// the neighbouring lanes' ones. Half layout: the pairs' first elements and their second ones. Interleaved: kVec / 2 pairs from
// either half of the head (single elements: a pair).
template <int kVec, bool kInter>
struct NormUnit {
  static constexpr int kFirst = kInter && kVec > 1 ? kVec / 2 : kVec;  // pairs of the first piece
  int e0, e1, pair0, pair1;  // first elements of the pieces; the unit's pairs are pair0 + k, from k = kFirst on pair1 + k - kFirst
  bool live, turned0, turned1;
  __device__ __forceinline__ NormUnit(int u, int units, int half) {
    live = u < units;
    const int n = live ? u : 0;
    if constexpr (kInter && kVec > 1) {
      e0 = n * kVec;
      e1 = (units + n) * kVec;
      pair0 = e0 / 2;
      pair1 = e1 / 2;
      turned0 = live && pair0 < half;
      turned1 = live && pair1 < half;
    } else {
      pair0 = pair1 = n * kVec;
      turned0 = turned1 = live && pair0 < half;
      e0 = kInter || !turned0 ? 2 * pair0 : pair0;
      e1 = kInter || !turned0 ? e0 + kVec : pair0 + half;
    }
  }
};

// Arithmetic on N floats, two at a time where N is even (one instruction for both).
template <int N>
__device__ __forceinline__ void v_mul(float (&d)[N], const float (&a)[N], const float (&b)[N]) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int k = 0; k < N; k += 2) f2_unpack(f2_mul(f2_pack(a[k], a[k + 1]), f2_pack(b[k], b[k + 1])), d[k], d[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) d[k] = a[k] * b[k];
  }
}
template <int N>
__device__ __forceinline__ void v_scale(float (&d)[N], float c) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int k = 0; k < N; k += 2) f2_unpack(f2_mul(f2_pack(d[k], d[k + 1]), f2_pack(c, c)), d[k], d[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) d[k] *= c;
  }
}
// d = a b + c
template <int N>
__device__ __forceinline__ void v_fma(float (&d)[N], const float (&a)[N], const float (&b)[N], const float (&c)[N]) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int k = 0; k < N; k += 2)
      f2_unpack(f2_fma(f2_pack(a[k], a[k + 1]), f2_pack(b[k], b[k + 1]), f2_pack(c[k], c[k + 1])), d[k], d[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) d[k] = fmaf(a[k], b[k], c[k]);
  }
}
// d = c - a b
template <int N>
__device__ __forceinline__ void v_nfma(float (&d)[N], const float (&a)[N], const float (&b)[N], const float (&c)[N]) {
  float m[N];
#pragma unroll
  for (int k = 0; k < N; ++k) m[k] = -b[k];
  v_fma(d, a, m, c);
}
// d = a c + b
template <int N>
__device__ __forceinline__ void v_axpy(float (&d)[N], const float (&a)[N], float c, const float (&b)[N]) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int k = 0; k < N; k += 2)
      f2_unpack(f2_fma(f2_pack(a[k], a[k + 1]), f2_pack(c, c), f2_pack(b[k], b[k + 1])), d[k], d[k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) d[k] = fmaf(a[k], c, b[k]);
  }
}
// A unit's elements, the pairs' first ones and second ones (of a part that is not turned: the even and the odd ones, or the
// two pieces; it makes no difference there).
template <int kVec>
struct Halves {
  float a[kVec], b[kVec];
};

template <int kVec>
__device__ __forceinline__ float dot(const Halves<kVec>& x, const Halves<kVec>& y) {
  float s;
  if constexpr (kVec % 2 == 0) {
    uint64_t sa = 0, sb = 0;
#pragma unroll
    for (int k = 0; k < kVec; k += 2) {
      sa = f2_fma(f2_pack(x.a[k], x.a[k + 1]), f2_pack(y.a[k], y.a[k + 1]), sa);
      sb = f2_fma(f2_pack(x.b[k], x.b[k + 1]), f2_pack(y.b[k], y.b[k + 1]), sb);
    }
    float lo, hi;
    f2_unpack(f2_add(sa, sb), lo, hi);
    s = lo + hi;
  } else {
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < kVec; ++k) s = fmaf(x.b[k], y.b[k], fmaf(x.a[k], y.a[k], s));
  }
  return s;
}

// Element k of the halves' a (b) is element `first` (`second`) of the unit's two pieces, one behind the other.
template <int kVec, bool kInter>
__device__ __forceinline__ constexpr int first_of(int k) { return kInter ? 2 * k : k; }
template <int kVec, bool kInter>
__device__ __forceinline__ constexpr int second_of(int k) { return kInter ? 2 * k + 1 : kVec + k; }

template <class T, int kVec, bool kInter>
__device__ __forceinline__ void unpack_pieces(const Pack<T, kVec>& p, const Pack<T, kVec>& q, Halves<kVec>& f) {
  float e[2 * kVec];
  if constexpr (std::is_same<T, __nv_bfloat16>::value && kVec % 2 == 0) {  // a shift and a mask for two elements
    uint32_t w[kVec];
    memcpy(w, &p, sizeof(p));
    memcpy(w + kVec / 2, &q, sizeof(q));
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      e[2 * k] = __uint_as_float(w[k] << 16);
      e[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      e[k] = to_f32<T>(p.v[k]);
      e[kVec + k] = to_f32<T>(q.v[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < kVec; ++k) {
    f.a[k] = e[first_of<kVec, kInter>(k)];
    f.b[k] = e[second_of<kVec, kInter>(k)];
  }
}

template <class T, int kVec, bool kInter>
__device__ __forceinline__ void pack_pieces(const Halves<kVec>& f, Pack<T, kVec>& p, Pack<T, kVec>& q) {
  float e[2 * kVec];
#pragma unroll
  for (int k = 0; k < kVec; ++k) {
    e[first_of<kVec, kInter>(k)] = f.a[k];
    e[second_of<kVec, kInter>(k)] = f.b[k];
  }
  if constexpr (sizeof(T) == 2 && kVec % 2 == 0) {
    constexpr bool kF16 = std::is_same<T, __half>::value;
    uint32_t w[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k) w[k] = pack2<kF16>(e[2 * k], e[2 * k + 1]);
    memcpy(&p, w, sizeof(p));
    memcpy(&q, w + kVec / 2, sizeof(q));
  } else {
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      p.v[k] = from_f32<T>(e[k]);
      q.v[k] = from_f32<T>(e[kVec + k]);
    }
  }
}

// Sines and cosines of a unit's pairs, times the scale.
template <int kVec>
struct Turn {
  float c[kVec], s[kVec];
};
// dz = R^T dy for pairs [kFrom, kTo)
template <int kFrom, int kTo, int kVec>
__device__ __forceinline__ void turn_back(Halves<kVec>& f, const Turn<kVec>& r) {
  constexpr int N = kTo - kFrom;
  if constexpr (N > 0) {
    float a[N], b[N], c[N], s[N], u[N], w[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      a[k] = f.a[kFrom + k];
      b[k] = f.b[kFrom + k];
      c[k] = r.c[kFrom + k];
      s[k] = r.s[kFrom + k];
    }
    v_mul(u, b, s);
    v_mul(w, b, c);
    v_fma(u, a, c, u);
    v_nfma(w, a, s, w);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      f.a[kFrom + k] = u[k];
      f.b[kFrom + k] = w[k];
    }
  }
}
// y = (a ca.c + b cb.s, a ca.s + b cb.c) for pairs [kFrom, kTo); not turned: (a ca.c, b cb.c)
template <int kFrom, int kTo, int kVec>
__device__ __forceinline__ void turn_ahead(const Halves<kVec>& f, const Turn<kVec>& ca, const Turn<kVec>& cb, bool turned, Halves<kVec>& y) {
  constexpr int N = kTo - kFrom;
  if constexpr (N > 0) {
    float a[N], b[N], ac[N], as[N], bc[N], bs[N], u[N], w[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      a[k] = f.a[kFrom + k];
      b[k] = f.b[kFrom + k];
      ac[k] = ca.c[kFrom + k];
      as[k] = ca.s[kFrom + k];
      bc[k] = cb.c[kFrom + k];
      bs[k] = cb.s[kFrom + k];
    }
    if (turned) {
      v_mul(u, b, bs);
      v_fma(u, a, ac, u);
      v_mul(w, b, bc);
      v_fma(w, a, as, w);
    } else {
      v_mul(u, a, ac);
      v_mul(w, b, bc);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      y.a[kFrom + k] = u[k];
      y.b[kFrom + k] = w[k];
    }
  }
}

// Sum over a row's lanes; kLanes 0: `group` of them.
template <int kLanes>
__device__ __forceinline__ float group_sum(float v, int group) {
  if constexpr (kLanes > 0) {
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  } else {
    for (int o = group >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

template <class T>
__device__ __forceinline__ float weight_at(const NormRotaryArgs& a, int w, int e) {
  return a.w_f32 ? __ldg(static_cast<const float*>(a.w[w]) + e) : to_f32<T>(static_cast<const T*>(a.w[w])[e]);
}

// Weights in shared memory as the lanes take them: 16 bytes of a unit (8 for kVec 1) beside those of the next, so that the
// lanes of a row read neighbouring ones.
template <int kVec>
struct WeightChunk {
  static constexpr int kFloats = kVec == 1 ? 2 : 4, kChunks = 2 * kVec / kFloats;
  using V = typename std::conditional<kVec == 1, float2, float4>::type;
};
template <class T, int kVec, bool kInter>
__device__ __forceinline__ void stage_weights(const NormRotaryArgs& a, int w, float* dst) {
  using C = WeightChunk<kVec>;
  const int half = a.rotary_dim / 2;
  for (int i = threadIdx.x; i < a.dim; i += kNormThreads) {
    const int x = i % C::kFloats, u = i / C::kFloats % a.units, c = i / C::kFloats / a.units;
    const int at = c * C::kFloats + x;  // of the unit's halves: a, then b
    const NormUnit<kVec, kInter> unit(u, a.units, half);
    const int e = at < kVec ? first_of<kVec, kInter>(at) : second_of<kVec, kInter>(at - kVec);
    dst[i] = weight_at<T>(a, w, e < kVec ? unit.e0 + e : unit.e1 + e - kVec);
  }
}
template <int kVec>
__device__ __forceinline__ void read_weights(const float* src, int unit, int units, Halves<kVec>& f) {
  using C = WeightChunk<kVec>;
  float v[2 * kVec];
#pragma unroll
  for (int c = 0; c < C::kChunks; ++c) {
    const typename C::V x = reinterpret_cast<const typename C::V*>(src)[c * units + unit];
    memcpy(v + c * C::kFloats, &x, sizeof(x));
  }
#pragma unroll
  for (int k = 0; k < kVec; ++k) {
    f.a[k] = v[k];
    f.b[k] = v[kVec + k];
  }
}

// (cos, sin) * scale of a chunk's tokens, [token][pair], element i by thread i % kNormThreads. Where the pairs divide the threads
// (dim 128: 64 of 256), a thread's pair is the same throughout and its rate is taken once; and most positions are small, exact in
// 64 bits (both together: three axes, 16383 tokens, both ways, 144.6 us -> 134.7).
struct NormAngles {
  int it0, pair0;        // this thread's first token and pair
  int tokens, pairs;     // what its next element is further
  TurnRate rate;
  int64_t start;         // of the positions of its axis
  __device__ __forceinline__ NormAngles(const NormRotaryArgs& a) {
    const int half = a.rotary_dim / 2;
    it0 = threadIdx.x / half;
    pair0 = threadIdx.x % half;
    tokens = kNormThreads / half;
    pairs = kNormThreads % half;
    pick(a, pair0);
  }
  __device__ __forceinline__ void pick(const NormRotaryArgs& a, int pair) {
    rate = turn_rate(a.inv_freq[pair]);
    start = axis_start(a.axes, a.num_axes, a.tokens, pair, a.err);
  }
  __device__ __forceinline__ void take(const NormRotaryArgs& a, int64_t t0, int count, float2* rot) {
    const int half = a.rotary_dim / 2;
    for (int it = it0, pair = pair0, i = threadIdx.x; it < count; i += kNormThreads) {
      if (pairs) pick(a, pair);
      const int64_t t = start + t0 + it;
      const int64_t at = a.positions64 ? static_cast<const int64_t*>(a.positions)[t] : static_cast<const int*>(a.positions)[t];
      const int low = static_cast<int>(at);
      const double turn = low == at ? turn_fraction(static_cast<double>(low), 0.0, rate) : turn_fraction(at, rate);
      float s, c;
      sincospif(2.0f * static_cast<float>(turn), &s, &c);
      rot[i] = make_float2(c * a.scale, a.sign * s * a.scale);
      it += tokens;
      pair += pairs;
      if (pair >= half) {
        pair -= half;
        ++it;
      }
    }
  }
};

// A row whose squares pass fp32's range is multiplied by this first.
constexpr float kNormDown = 0x1p-100f;

template <int kVec, int kUnits, bool kInter>
__device__ __forceinline__ void read_turns(const NormRotaryArgs& a, const float2* rot, int group, int lane, bool any,
                                           Turn<kVec> (&t)[kUnits]) {
#pragma unroll
  for (int n = 0; n < kUnits; ++n) {
    const NormUnit<kVec, kInter> u(group * n + lane, a.units, a.rotary_dim / 2);
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      const bool second = k >= NormUnit<kVec, kInter>::kFirst, turned = second ? u.turned1 : u.turned0;
      const int pair = second ? u.pair1 + k - NormUnit<kVec, kInter>::kFirst : u.pair0 + k;
      const float2 r = turned && any ? rot[pair] : make_float2(1.0f, 0.0f);
      t[n].c[k] = r.x;
      t[n].s[k] = r.y;
    }
  }
}

// A thread's rows on their way: rings of kStages steps in shared memory, each of kPieces pieces of a thread's own, [step][piece]
// [thread], so that nobody waits for another thread's. Pieces of 4 bytes and more are copied asynchronously.
template <class P, int kPieces>
struct NormRing {
  static constexpr int kStepBytes = kPieces * kNormThreads * (int)sizeof(P);
  static constexpr int kStages = kStepBytes <= 32768 ? 3 : 2;
  static constexpr int kBytes = kStages * kStepBytes;
  static constexpr bool kAsync = sizeof(P) >= 4;
  static __device__ __forceinline__ uint8_t* at(uint8_t* ring, int stage, int piece) {
    return ring + stage * kStepBytes + (piece * kNormThreads + threadIdx.x) * sizeof(P);
  }
  static __device__ __forceinline__ void fetch(uint8_t* dst, const void* src, bool live) {
    if constexpr (kAsync) {
      const uint32_t n = live ? sizeof(P) : 0u;  // 0: zeros, src is not read
      if constexpr (sizeof(P) == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(dst)), "l"(src), "r"(n) : "memory");
      else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(ptx::smem_u32(dst)), "l"(src), "r"(n), "n"(sizeof(P)) : "memory");
    } else {
      *reinterpret_cast<P*>(dst) = live ? *static_cast<const P*>(src) : P{};
    }
  }
  static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory"); }
};

// Chunks of per_block tokens are walked with a stride of the blocks, a chunk's heads in rounds of kRows rows a thread; a step is a
// round of a chunk. Where this thread's next step to be fetched, or to be worked on, stands.
struct NormStep {
  int64_t chunk;
  int round, stage;
  __device__ __forceinline__ void next(int rounds, int64_t blocks, int stages) {
    if (++round == rounds) {
      round = 0;
      chunk += blocks;
    }
    if (++stage == stages) stage = 0;
  }
};

// kUnits units per lane: units group * p + lane for p < kUnits. kLanes: the group's width, 0 where it is known at run time only.
template <class T, int kVec, int kUnits, bool kBackward>
struct NormShape {
  using P = Pack<T, kVec>;
  static constexpr int kRows = kBackward ? kNormBatchBwd : kNormBatch;
  static constexpr int kTensors = kBackward ? 2 : 1;
  using Ring = NormRing<P, kRows * kUnits * 2 * kTensors>;
  // by registers and shared memory: about as much on its way in an SM whatever a piece's size
  static constexpr int kBlocksPerSm = kUnits > 1 ? 1 : 32 / (kVec * (int)sizeof(T)) < kNormMostBlocks ? 32 / (kVec * (int)sizeof(T)) : kNormMostBlocks;
  static constexpr int kMostSmem = Ring::kBytes + 20 * 1024;
  // the ring (at the end the groups' sums of dw), a chunk's angles, the weights
  static __host__ __device__ int weights_at(const NormRotaryArgs& a) {
    const int per_block = a.per_block[0] > a.per_block[1] ? a.per_block[0] : a.per_block[1];
    const int loop = Ring::kBytes + per_block * (a.rotary_dim / 2) * (int)sizeof(float2);
    const int sums = kBackward ? kNormThreads / a.group * a.dim * (int)sizeof(float) : 0;
    return ((loop > sums ? loop : sums) + 15) / 16 * 16;
  }
  static int smem_bytes(const NormRotaryArgs& a) { return weights_at(a) + a.dim * (int)sizeof(float); }
};

// Blocks [0, blocks_q) take Q, the others K, each with the tokens blocks * per_block apart.
struct NormBlock {
  int w, heads, at_once, per_block, it, h0, rounds;
  int64_t first, blocks, chunks;
  __device__ __forceinline__ NormBlock(const NormRotaryArgs& a, int g, int rows_a_step) {
    w = static_cast<int>(blockIdx.x) >= a.blocks_q;
    first = w ? blockIdx.x - a.blocks_q : blockIdx.x;
    blocks = w ? gridDim.x - a.blocks_q : a.blocks_q;
    heads = a.heads[w];
    at_once = a.at_once[w];
    per_block = a.per_block[w];
    it = g / at_once;
    h0 = g - it * at_once;
    rounds = (heads + rows_a_step * at_once - 1) / (rows_a_step * at_once);
    chunks = (static_cast<int64_t>(a.tokens) + per_block - 1) / per_block;
  }
  // heads of this thread's token of a chunk, 0 where it has none
  __device__ __forceinline__ int rows(const NormRotaryArgs& a, int64_t chunk) const {
    return it < per_block && chunk * per_block + it < a.tokens ? heads : 0;
  }
};

// kNorm: else the rotation alone (without weights, eps and the norm; the part that is not turned is copied).
template <class T, int kVec, int kUnits, bool kInter, int kLanes, bool kNorm>
__global__ void __launch_bounds__(kNormThreads, NormShape<T, kVec, kUnits, false>::kBlocksPerSm)
    norm_rotary_kernel(const __grid_constant__ NormRotaryArgs a) {
  extern __shared__ float4 norm_smem[];
  using P = Pack<T, kVec>;
  using Sh = NormShape<T, kVec, kUnits, false>;
  using Ring = typename Sh::Ring;
  using Unit = NormUnit<kVec, kInter>;
  uint8_t* ring = reinterpret_cast<uint8_t*>(norm_smem);
  float2* rot = reinterpret_cast<float2*>(ring + Ring::kBytes);  // [tokens][pairs]
  float* w_s = reinterpret_cast<float*>(ring + Sh::weights_at(a));
  const int half = a.rotary_dim / 2, group = kLanes > 0 ? kLanes : a.group;
  const int lane = threadIdx.x & (group - 1);
  const NormBlock blk(a, threadIdx.x / group, kNormBatch);
  const int w = blk.w;
  const T* xs = static_cast<const T*>(a.x[w]);
  const int64_t x_step = blk.at_once * a.head_stride[w], y_step = static_cast<int64_t>(blk.at_once) * a.dim;
  NormStep ahead{blk.first, 0, 0};
  auto fetch = [&]() {
    if (ahead.chunk < blk.chunks) {
      const int rows = blk.rows(a, ahead.chunk), h = blk.h0 + ahead.round * kNormBatch * blk.at_once;
      const T* x0 = xs + (ahead.chunk * blk.per_block + blk.it) * a.token_stride[w] + h * a.head_stride[w];
#pragma unroll
      for (int n = 0; n < kUnits; ++n) {
        const Unit u(group * n + lane, a.units, half);
        const T* x = x0 + u.e0;  // (not read where the row or the unit is not there)
#pragma unroll
        for (int b = 0; b < kNormBatch; ++b, x += x_step) {
          const bool live = h + b * blk.at_once < rows && u.live;
          Ring::fetch(Ring::at(ring, ahead.stage, (b * kUnits + n) * 2), x, live);
          Ring::fetch(Ring::at(ring, ahead.stage, (b * kUnits + n) * 2 + 1), x + (u.e1 - u.e0), live);
        }
      }
    }
    Ring::commit();
    ahead.next(blk.rounds, blk.blocks, Ring::kStages);
  };
#pragma unroll
  for (int i = 0; i < Ring::kStages - 1; ++i) fetch();
  if constexpr (kNorm) stage_weights<T, kVec, kInter>(a, w, w_s);
  const float inv_dim = 1.0f / static_cast<float>(a.dim);
  NormAngles angles(a);
  NormStep now{blk.first, 0, 0};
  while (now.chunk < blk.chunks) {
    const int64_t t0 = now.chunk * blk.per_block, t = t0 + blk.it;
    const int rows = blk.rows(a, now.chunk);
    __syncthreads();  // the chunk before has read its angles
    angles.take(a, t0, static_cast<int>(min(static_cast<int64_t>(blk.per_block), a.tokens - t0)), rot);
    __syncthreads();
    // Turn and weights in one: (a, b) -> (a ac + b bs, a as + b bc), bs with the other sign
    Turn<kVec> ca[kUnits], cb[kUnits];
    read_turns<kVec, kUnits, kInter>(a, rot + blk.it * half, group, lane, rows > 0, ca);
#pragma unroll
    for (int n = 0; n < kUnits; ++n) {
      cb[n] = ca[n];
      v_scale(cb[n].s, -1.0f);
      if constexpr (kNorm) {
        Halves<kVec> weight;
        const Unit u(group * n + lane, a.units, half);
        read_weights<kVec>(w_s, u.live ? group * n + lane : 0, a.units, weight);
        v_mul(cb[n].c, cb[n].c, weight.b);
        v_mul(cb[n].s, cb[n].s, weight.b);
        v_mul(ca[n].c, ca[n].c, weight.a);
        v_mul(ca[n].s, ca[n].s, weight.a);
      }
    }
    // (every lane of a warp takes part in every sum: the loop's length is the same for all)
    for (int round = 0; round < blk.rounds; ++round) {
      fetch();
      Ring::wait();
      const int h = blk.h0 + round * kNormBatch * blk.at_once;
      T* y = static_cast<T*>(a.y[w]) + (t * blk.heads + h) * a.dim;
#pragma unroll
      for (int b = 0; b < kNormBatch; ++b, y += y_step) {
        Halves<kVec> f[kUnits];
        float ss = 0.0f, eps = a.eps;
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
          unpack_pieces<T, kVec, kInter>(*reinterpret_cast<const P*>(Ring::at(ring, now.stage, (b * kUnits + n) * 2)),
                                         *reinterpret_cast<const P*>(Ring::at(ring, now.stage, (b * kUnits + n) * 2 + 1)), f[n]);
          if constexpr (kNorm) ss += dot(f[n], f[n]);
        }
        if constexpr (kNorm) ss = group_sum<kLanes>(ss, group);
        if constexpr (kNorm && !std::is_same<T, __half>::value) {
          const bool far = !(ss <= 3.0e38f);
          if (__any_sync(0xffffffffu, far)) {
            if (far) eps = 0.0f;
            ss = 0.0f;
#pragma unroll
            for (int n = 0; n < kUnits; ++n) {
              v_scale(f[n].a, far ? kNormDown : 1.0f);
              v_scale(f[n].b, far ? kNormDown : 1.0f);
              ss += dot(f[n], f[n]);
            }
            ss = group_sum<kLanes>(ss, group);
          }
        }
        const float inv = rsqrtf(fmaf(ss, inv_dim, eps));
        if (h + b * blk.at_once >= rows) continue;
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
          const Unit u(group * n + lane, a.units, half);
          if (!u.live) continue;
          Halves<kVec> y_f;
          P po, qo;
          if (kNorm || u.turned0 || u.turned1) {
            if constexpr (kNorm) {  // (before the turn: a large row times a large scale would pass fp32's range)
              v_scale(f[n].a, inv);
              v_scale(f[n].b, inv);
            }
            turn_ahead<0, Unit::kFirst>(f[n], ca[n], cb[n], u.turned0, y_f);
            turn_ahead<Unit::kFirst, kVec>(f[n], ca[n], cb[n], u.turned1, y_f);
            pack_pieces<T, kVec, kInter>(y_f, po, qo);
          }
          if constexpr (!kNorm) {  // what is not turned is copied as it is
            if (!u.turned0) po = *reinterpret_cast<const P*>(Ring::at(ring, now.stage, (b * kUnits + n) * 2));
            if (!u.turned1) qo = *reinterpret_cast<const P*>(Ring::at(ring, now.stage, (b * kUnits + n) * 2 + 1));
          }
          *reinterpret_cast<P*>(y + u.e0) = po;
          *reinterpret_cast<P*>(y + u.e1) = qo;
        }
      }
      now.next(blk.rounds, blk.blocks, Ring::kStages);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <class T, int kVec, int kUnits, bool kInter, int kLanes>
__global__ void __launch_bounds__(kNormThreads, NormShape<T, kVec, kUnits, true>::kBlocksPerSm)
    norm_rotary_bwd_kernel(const __grid_constant__ NormRotaryArgs a) {
  extern __shared__ float4 norm_smem[];
  ptx::grid_launch_dependents();
  using P = Pack<T, kVec>;
  using Sh = NormShape<T, kVec, kUnits, true>;
  using Ring = typename Sh::Ring;
  using Unit = NormUnit<kVec, kInter>;
  uint8_t* ring = reinterpret_cast<uint8_t*>(norm_smem);
  float2* rot = reinterpret_cast<float2*>(ring + Ring::kBytes);  // [tokens][pairs]
  float* w_s = reinterpret_cast<float*>(ring + Sh::weights_at(a));
  const int half = a.rotary_dim / 2, group = kLanes > 0 ? kLanes : a.group;
  const int lane = threadIdx.x & (group - 1), g = threadIdx.x / group, groups = kNormThreads / group;
  const NormBlock blk(a, g, kNormBatchBwd);
  const int w = blk.w;
  const T* xs = static_cast<const T*>(a.x[w]);
  const T* dys = static_cast<const T*>(a.dy[w]);
  const int64_t x_step = blk.at_once * a.head_stride[w], dy_step = blk.at_once * a.dy_head_stride[w],
                y_step = static_cast<int64_t>(blk.at_once) * a.dim;
  NormStep ahead{blk.first, 0, 0};
  auto fetch = [&]() {
    if (ahead.chunk < blk.chunks) {
      const int rows = blk.rows(a, ahead.chunk), h = blk.h0 + ahead.round * kNormBatchBwd * blk.at_once;
      const int64_t t = ahead.chunk * blk.per_block + blk.it;
      const T* x0 = xs + t * a.token_stride[w] + h * a.head_stride[w];
      const T* dy0 = dys + t * a.dy_token_stride[w] + h * a.dy_head_stride[w];
#pragma unroll
      for (int n = 0; n < kUnits; ++n) {
        const Unit u(group * n + lane, a.units, half);
        const T* x = x0 + u.e0;  // (not read where the row or the unit is not there)
        const T* dy = dy0 + u.e0;
#pragma unroll
        for (int b = 0; b < kNormBatchBwd; ++b, x += x_step, dy += dy_step) {
          const bool live = h + b * blk.at_once < rows && u.live;
          const int piece = (b * kUnits + n) * 4;
          Ring::fetch(Ring::at(ring, ahead.stage, piece), x, live);
          Ring::fetch(Ring::at(ring, ahead.stage, piece + 1), x + (u.e1 - u.e0), live);
          Ring::fetch(Ring::at(ring, ahead.stage, piece + 2), dy, live);
          Ring::fetch(Ring::at(ring, ahead.stage, piece + 3), dy + (u.e1 - u.e0), live);
        }
      }
    }
    Ring::commit();
    ahead.next(blk.rounds, blk.blocks, Ring::kStages);
  };
#pragma unroll
  for (int i = 0; i < Ring::kStages - 1; ++i) fetch();
  stage_weights<T, kVec, kInter>(a, w, w_s);
  Halves<kVec> dw[kUnits];
#pragma unroll
  for (int n = 0; n < kUnits; ++n)
#pragma unroll
    for (int k = 0; k < kVec; ++k) dw[n].a[k] = dw[n].b[k] = 0.0f;
  const float inv_dim = 1.0f / static_cast<float>(a.dim);
  NormAngles angles(a);
  NormStep now{blk.first, 0, 0};
  while (now.chunk < blk.chunks) {
    const int64_t t0 = now.chunk * blk.per_block, t = t0 + blk.it;
    const int rows = blk.rows(a, now.chunk);
    __syncthreads();  // the chunk before has read its angles
    angles.take(a, t0, static_cast<int>(min(static_cast<int64_t>(blk.per_block), a.tokens - t0)), rot);
    __syncthreads();
    Turn<kVec> turn[kUnits];
    read_turns<kVec, kUnits, kInter>(a, rot + blk.it * half, group, lane, rows > 0, turn);
    for (int round = 0; round < blk.rounds; ++round) {
      fetch();
      Ring::wait();
      const int h = blk.h0 + round * kNormBatchBwd * blk.at_once;
      T* y = static_cast<T*>(a.y[w]) + (t * blk.heads + h) * a.dim;
#pragma unroll
      for (int b = 0; b < kNormBatchBwd; ++b, y += y_step) {
        // dx = (g - x (sum(g x) / (dim rms^2))) / rms: both sums of a row at once
        Halves<kVec> x[kUnits], dz[kUnits];
        float ss = 0.0f, gx = 0.0f, eps = a.eps, down = 1.0f;
        auto sums = [&]() {
          ss = gx = 0.0f;
#pragma unroll
          for (int n = 0; n < kUnits; ++n) {
            Halves<kVec> p, weight;
            read_weights<kVec>(w_s, min(group * n + lane, a.units - 1), a.units, weight);
            v_mul(p.a, dz[n].a, x[n].a);
            v_mul(p.b, dz[n].b, x[n].b);
            ss += dot(x[n], x[n]);
            gx += dot(p, weight);
          }
          ss = group_sum<kLanes>(ss, group);
          gx = group_sum<kLanes>(gx, group);
        };
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
          const Unit u(group * n + lane, a.units, half);
          const int piece = (b * kUnits + n) * 4;
          unpack_pieces<T, kVec, kInter>(*reinterpret_cast<const P*>(Ring::at(ring, now.stage, piece)),
                                         *reinterpret_cast<const P*>(Ring::at(ring, now.stage, piece + 1)), x[n]);
          unpack_pieces<T, kVec, kInter>(*reinterpret_cast<const P*>(Ring::at(ring, now.stage, piece + 2)),
                                         *reinterpret_cast<const P*>(Ring::at(ring, now.stage, piece + 3)), dz[n]);
          if (u.turned0) turn_back<0, Unit::kFirst>(dz[n], turn[n]);
          if (u.turned1) turn_back<Unit::kFirst, kVec>(dz[n], turn[n]);
        }
        sums();
        if constexpr (!std::is_same<T, __half>::value) {
          const bool far = !(ss <= 3.0e38f);
          if (__any_sync(0xffffffffu, far)) {
            if (far) {
              down = kNormDown;
              eps = 0.0f;
            }
#pragma unroll
            for (int n = 0; n < kUnits; ++n) {
              v_scale(x[n].a, down);
              v_scale(x[n].b, down);
            }
            sums();
          }
        }
        const float inv = rsqrtf(fmaf(ss, inv_dim, eps));
        const float mean = gx * inv_dim * inv * inv, out = inv * down;
        const bool live_row = h + b * blk.at_once < rows;
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
          const Unit u(group * n + lane, a.units, half);
          Halves<kVec> g_f, weight;
          v_mul(g_f.a, dz[n].a, x[n].a);
          v_mul(g_f.b, dz[n].b, x[n].b);
          v_axpy(dw[n].a, g_f.a, inv, dw[n].a);
          v_axpy(dw[n].b, g_f.b, inv, dw[n].b);
          if (!live_row || !u.live) continue;
          read_weights<kVec>(w_s, group * n + lane, a.units, weight);
          v_mul(g_f.a, dz[n].a, weight.a);
          v_mul(g_f.b, dz[n].b, weight.b);
          v_axpy(g_f.a, x[n].a, -mean, g_f.a);
          v_axpy(g_f.b, x[n].b, -mean, g_f.b);
          v_scale(g_f.a, out);
          v_scale(g_f.b, out);
          P po, qo;
          pack_pieces<T, kVec, kInter>(g_f, po, qo);
          *reinterpret_cast<P*>(y + u.e0) = po;
          *reinterpret_cast<P*>(y + u.e1) = qo;
        }
      }
      now.next(blk.rounds, blk.blocks, Ring::kStages);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  // the groups' sums, added in order
  float* sums = reinterpret_cast<float*>(ring);
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kUnits; ++n) {
    const Unit u(group * n + lane, a.units, half);
    if (!u.live) continue;
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      const int i = first_of<kVec, kInter>(k), j = second_of<kVec, kInter>(k);
      sums[g * a.dim + (i < kVec ? u.e0 + i : u.e1 + i - kVec)] = dw[n].a[k];
      sums[g * a.dim + (j < kVec ? u.e0 + j : u.e1 + j - kVec)] = dw[n].b[k];
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
