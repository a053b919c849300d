// Attention of a few new tokens per sequence over a paged cache, for sm_100a (fp16 / bf16 queries; a cache of the
// queries' type or of e4m3 codes with one scale per slot and head).
//
// Rows: the (token, head) pairs of one sequence that share a kv head, token-major, in tiles of 16. A cluster of C CTAs
// takes one tile; the keys that the tile's last row may see are split evenly over the cluster, and within a CTA over
// its four warps, stage by stage. Every warp is on its own: it copies its stages of K and V rows (8 KB each, three in
// flight) with cp.async, multiplies them with mma.sync m16n8k16 and keeps its own running maximum, sum and 16 x D
// output in registers (one pass over the keys, softmax statistics and output in fp32). The partial results meet once
// at the end: four warps in shared memory, C CTAs through distributed shared memory, so a call is one launch without
// a workspace.
//
// Bound: HBM. A key and value are read once per tile and used by 16 rows (4 * 16 * D flops for 4 * D bytes), far below
// the tensor pipe's rate, so the tile is the smallest that mma.sync has, and 2 CTAs of 96 KB per SM keep about 128 KB
// of copies in flight. tcgen05's 128-row tile would leave 7/8 of its rows empty here.
//
// e4m3 caches: the contraction's order over D (for K) and the columns' order (for V) are permuted so that each thread
// reads its codes as 16-byte words and converts them in registers. K codes become the queries' type (exact: every e4m3
// value is an fp16 and a bf16 value) and the scale multiplies the scores; V codes become bf16 and the scale multiplies
// P before its rounding to bf16 -- also for fp16 queries, since P * scale may leave fp16's range: an error of 2^-9 a
// weight beside the 2^-4 of the codes.
//
// P is rounded to the queries' type for the second product (relative error 2^-9 bf16, 2^-12 fp16 a weight, the outputs'
// own rounding); its sum is taken in fp32 before the rounding.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "bsattn_sm100.cuh"
#include "kv_cache.cuh"

namespace bsk {

constexpr int kPagedThreads = 128;
constexpr int kPagedWarps = 4;
constexpr int kPagedStages = 3;
constexpr int kPagedStageBytes = 8192;  // K and V rows of one warp's stage
constexpr int kPagedRows = 16;          // rows of a tile (mma.sync M)
constexpr uint32_t kKidPaged = 10;

struct PagedArgs {
  const void* Q;              // [tokens, heads, D], strides in elements
  int64_t q_token_stride, q_head_stride;
  void* O;                    // contiguous [tokens, heads, D]
  const void* k_cache;        // [pages, page size, kv heads, D]
  const void* v_cache;
  const float* k_scale;       // [pages, page size, kv heads], e4m3 caches only
  const float* v_scale;
  const int* block_table;     // [batch, table_width] page numbers
  const int* kv_lens;         // [batch] cached tokens, the chunk's own among them
  const int* cu_seqlens;      // [batch + 1] first row of each sequence's new tokens
  int64_t table_stride;
  int tokens, batch, heads, kv_heads, group;  // group = heads / kv_heads
  int table_width, page_shift, num_pages;
  float scale_log2;           // softmax scale * log2(e)
  uint32_t* err;
};

__device__ __forceinline__ void paged_flag(uint32_t* err, uint32_t site) {
  atomicCAS(err, 0u, kErrBounds | (kKidPaged << 8) | (site << 16));
}

// Rows [lo, hi) of sequence i's new tokens, held within [0, tokens].
__device__ __forceinline__ void seq_rows(const int* cu, int i, int tokens, int& lo, int& hi, bool& bad) {
  const int a = i == 0 ? 0 : __ldg(&cu[i]), b = __ldg(&cu[i + 1]);
  lo = min(max(a, 0), tokens);
  hi = min(max(b, lo), tokens);
  bad = a != lo || b != hi || (i == 0 && __ldg(&cu[0]) != 0);
}

// Tiles of `rows` packed rows are numbered with base(i) = cu[i] * group / rows + i for sequence i (increasing, and
// base(i + 1) - base(i) covers sequence i's tiles). Warp-wide search: the last i in [0, batch] with base(i) <= tile,
// narrowed by a factor of 32 per step.
__device__ __forceinline__ int find_seq(const int* cu, int batch, int tokens, int group, int rows, int64_t tile) {
  int lo = 0, hi = batch + 1;  // base(lo) <= tile < base(hi)
  const int lane = ptx::lane_id();
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int i = min(lo + lane * step, hi);
    int64_t base = INT64_MAX;
    if (i < hi) base = static_cast<int64_t>(i == 0 ? 0 : min(max(__ldg(&cu[i]), 0), tokens)) * group / rows + i;
    const uint32_t below = __ballot_sync(0xffffffffu, base <= tile);
    const int last = below ? 31 - __clz(below) : 0;
    lo = lo + last * step;
    hi = min(lo + step, hi);
  }
  return lo;
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool full) {
  const uint32_t n = full ? 16u : 0u;  // 0: the 16 bytes are set to zero and src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src, bool full) {
  const uint32_t n = full ? 4u : 0u;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint4 lds_16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds_8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// D (16 x 8, fp32) += A (16 x 16) B (16 x 8), fp16 or bf16 operands.
template <bool kF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (kF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two e4m3 codes (low 16 bits) -> two 16-bit floats, exactly.
template <bool kF16>
__device__ __forceinline__ uint32_t e4m3x2(uint32_t two) {
  uint32_t h;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(h) : "r"(two));
  if (kF16) return h;
  const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h));
  return pack_bf16(f.x, f.y);
}

template <bool kF16, int kD, bool kFp8>
struct PagedShape {
  static constexpr int kRowBytes = kD * (kFp8 ? 1 : 2);
  static constexpr int kKeys = kPagedStageBytes / (2 * kRowBytes);  // keys per warp stage: 16, 32 or 64
  static constexpr int kChunks = kRowBytes / 16;                    // 16-byte chunks per row: 4, 8 or 16
  static constexpr int kScaleBytes = kFp8 ? 2 * kKeys * 4 : 0;
  static constexpr int kStage = kPagedStageBytes + kScaleBytes;
  static constexpr int kWarpBytes = kPagedStages * kStage;
  static constexpr int kMergeBytes = (kPagedWarps + 1) * (kPagedRows * kD + 2 * kPagedRows) * 4;
  static constexpr int kSmemBytes = kPagedWarps * kWarpBytes > kMergeBytes ? kPagedWarps * kWarpBytes : kMergeBytes;
};

template <bool kF16, int kD, bool kFp8>
__global__ void __launch_bounds__(kPagedThreads) paged_decode_kernel(const PagedArgs a) {
  using Sh = PagedShape<kF16, kD, kFp8>;
  constexpr int kKeys = Sh::kKeys, kChunks = Sh::kChunks, kRowBytes = Sh::kRowBytes;
  constexpr int kKS = kD / 16;       // k16 steps of Q K^T
  constexpr int kNT = kKeys / 8;     // n8 tiles of a stage's scores
  constexpr int kOT = kD / 8;        // n8 tiles of the output
  constexpr bool kPF16 = kF16 && !kFp8;  // type of P and V in the second product
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float m_all[kPagedWarps][kPagedRows], l_all[kPagedWarps][kPagedRows];
  __shared__ float m_cta[kPagedRows], l_cta[kPagedRows];

  uint32_t nrank, rank;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(nrank));
  asm volatile("mov.u32 %0, %%cluster_ctaid.x;" : "=r"(rank));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t4 = lane & 3, r8 = lane >> 2;
  const int64_t tile = blockIdx.x / nrank;
  const int hkv = blockIdx.y;

  // ---- which sequence and rows (the same for the whole cluster, so a return leaves nobody waiting)
  const int seq = find_seq(a.cu_seqlens, a.batch, a.tokens, a.group, kPagedRows, tile);
  if (seq == a.batch) {  // rows behind the last sequence are zero
    if (blockIdx.x == gridDim.x - 1 && hkv == 0)  // the last tile of the grid always comes here
      for (int i = threadIdx.x; i < a.batch; i += kPagedThreads) {
        int lo, hi;
        bool bad;
        seq_rows(a.cu_seqlens, i, a.tokens, lo, hi, bad);
        if (bad) paged_flag(a.err, 1);
      }
    const int end = min(max(__ldg(&a.cu_seqlens[a.batch]), 0), a.tokens);
    const int64_t base = static_cast<int64_t>(end) * a.group / kPagedRows + a.batch;
    const int64_t first = static_cast<int64_t>(end) * a.group + (tile - base) * kPagedRows;
    constexpr int kOc = kD / 8;
    for (int i = threadIdx.x + rank * kPagedThreads; i < kPagedRows * kOc; i += kPagedThreads * nrank) {
      const int64_t row = first + i / kOc;
      if (row < static_cast<int64_t>(a.tokens) * a.group) {
        const int64_t t = row / a.group;
        const int h = hkv * a.group + static_cast<int>(row % a.group);
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.O) + (t * a.heads + h) * kD)[i % kOc] = make_uint4(0, 0, 0, 0);
      }
    }
    return;
  }
  int lo, hi;
  bool bad;
  seq_rows(a.cu_seqlens, seq, a.tokens, lo, hi, bad);
  const int64_t base = static_cast<int64_t>(lo) * a.group / kPagedRows + seq;
  const int64_t row0 = (tile - base) * kPagedRows;                     // first packed row of the tile
  const int64_t rows = static_cast<int64_t>(hi - lo) * a.group;        // packed rows of the sequence
  if (row0 >= rows) return;
  int kv_len = __ldg(&a.kv_lens[seq]);
  const int64_t room = static_cast<int64_t>(a.table_width) << a.page_shift;
  if (kv_len < 0 || kv_len > room) {
    if (threadIdx.x == 0) paged_flag(a.err, 2);
    kv_len = kv_len < 0 ? 0 : static_cast<int>(room);
  }
  const int first_pos = kv_len - (hi - lo);  // position of the chunk's first token (negative: rows without keys)
  const int last_row = static_cast<int>(min(row0 + kPagedRows, rows) - 1);
  const int keys_end = max(first_pos + last_row / a.group + 1, 0);  // keys that the tile's last row sees

  // ---- this CTA's keys: whole sets of four warp stages
  constexpr int kSet = kKeys * kPagedWarps;
  const int sets = (keys_end + kSet - 1) / kSet;
  const int per = (sets + nrank - 1) / nrank;
  const int set_begin = min(static_cast<int>(rank) * per, sets), set_end = min(set_begin + per, sets);
  const int n_stages = set_end - set_begin;

  // ---- queries as A fragments (rows r8 and r8 + 8 of the tile)
  uint32_t qf[kKS][4];
  int limit[2];  // keys at or beyond this position are masked
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int64_t row = row0 + r8 + 8 * x;
    const bool live = row < rows;
    const int tok = live ? static_cast<int>(row / a.group) : 0;
    const int head = hkv * a.group + (live ? static_cast<int>(row % a.group) : 0);
    limit[x] = live ? first_pos + tok + 1 : 0;
    const uint16_t* q = static_cast<const uint16_t*>(a.Q) + (lo + tok) * a.q_token_stride + head * a.q_head_stride;
#pragma unroll
    for (int k = 0; k < kKS; ++k) {
      // element pairs of k step k: {2 t4, 2 t4 + 1} and {+8, +9}; e4m3: four neighbours 64 h + 16 t4 + 4 w (k = 4 h + w)
      const int d0 = kFp8 ? 64 * (k >> 2) + 16 * t4 + 4 * (k & 3) : 16 * k + 2 * t4;
      const int d1 = kFp8 ? d0 + 2 : d0 + 8;
      qf[k][x] = live ? *reinterpret_cast<const uint32_t*>(q + d0) : 0u;
      qf[k][2 + x] = live ? *reinterpret_cast<const uint32_t*>(q + d1) : 0u;
    }
  }

  // ---- copies: stage s of this warp = keys [key0(s), key0(s) + kKeys)
  const uint32_t wbase = ptx::smem_u32(smem) + warp * Sh::kWarpBytes;
  const int* table = a.block_table + seq * a.table_stride;
  auto key0 = [&](int s) { return (set_begin + s) * kSet + warp * kKeys; };
  constexpr int kSl = (kKeys + 31) / 32;
  int64_t slot_of[kSl];  // lane l: slots of keys l (and l + 32) of the stage to be copied next, -1: none
  auto look_up = [&](int s) {
#pragma unroll
    for (int x = 0; x < kSl; ++x) {
      const int key = key0(s) + lane + 32 * x;
      slot_of[x] = -1;
      if (s < n_stages && lane + 32 * x < kKeys && key < keys_end) {
        const int page = __ldg(&table[key >> a.page_shift]);
        if (page < 0 || page >= a.num_pages)
          paged_flag(a.err, 3);
        else
          slot_of[x] = (static_cast<int64_t>(page) << a.page_shift) + (key & ((1 << a.page_shift) - 1));
      }
    }
  };
  // Swizzles (16-byte chunk index): 16-bit rows by the row for ldmatrix; e4m3 K so that two neighbouring rows, and V so
  // that rows 0, 2, 4, 6, fall into different banks for the reads below.
  auto k_chunk = [](int row, int c) -> int {
    if (!kFp8) return c ^ (row & 7);
    return kChunks == 8 ? c ^ ((row & 1) << 2) : c;
  };
  auto v_chunk = [](int row, int c) -> int {
    if (!kFp8) return c ^ (row & 7);
    return kChunks == 8 ? c ^ (row & 6) : c ^ ((row >> 1) & 3);
  };
  auto copy = [&](int s) {
    if (s < n_stages) {
      const uint32_t dst = wbase + (s % kPagedStages) * Sh::kStage;
      constexpr int kPer = 32 / kChunks;  // rows copied at once
#pragma unroll
      for (int r0 = 0; r0 < kKeys; r0 += kPer) {
        const int row = r0 + lane / kChunks, c = lane % kChunks;
        const int64_t slot = __shfl_sync(0xffffffffu, slot_of[r0 / 32], row & 31);
        const bool live = slot >= 0;
        const int64_t off = ((live ? slot : 0) * a.kv_heads + hkv) * kRowBytes + 16 * c;
        cp_async_16(dst + row * kRowBytes + 16 * k_chunk(row, c), static_cast<const uint8_t*>(a.k_cache) + off, live);
        cp_async_16(dst + kPagedStageBytes / 2 + row * kRowBytes + 16 * v_chunk(row, c),
                    static_cast<const uint8_t*>(a.v_cache) + off, live);
      }
      if (kFp8) {
#pragma unroll
        for (int x = 0; x < kSl; ++x) {
          const bool live = slot_of[x] >= 0;
          const int64_t off = (live ? slot_of[x] : 0) * a.kv_heads + hkv;
          const uint32_t sdst = dst + kPagedStageBytes + (lane + 32 * x) * 4;
          cp_async_4(sdst, a.k_scale + off, live);
          cp_async_4(sdst + kKeys * 4, a.v_scale + off, live);
        }
      }
    }
    cp_async_commit();
  };

  float o[kOT][4];
#pragma unroll
  for (int j = 0; j < kOT; ++j)
#pragma unroll
    for (int x = 0; x < 4; ++x) o[j][x] = 0.0f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};

#pragma unroll
  for (int s = 0; s < kPagedStages - 1; ++s) {
    look_up(s);
    copy(s);
  }
  look_up(kPagedStages - 1);
  for (int s = 0; s < n_stages; ++s) {
    __syncwarp();  // every lane is done with the buffer that the next copy overwrites
    copy(s + kPagedStages - 1);
    look_up(s + kPagedStages);
    cp_async_wait<kPagedStages - 1>();
    __syncwarp();
    const uint32_t kb = wbase + (s % kPagedStages) * Sh::kStage, vb = kb + kPagedStageBytes / 2;

    float sc[kNT][4];
#pragma unroll
    for (int j = 0; j < kNT; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) sc[j][x] = 0.0f;
    if constexpr (!kFp8) {
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int k = 0; k < kKS; k += 2) {
          const int row = 8 * j + (lane & 7), c = 2 * k + (lane >> 3);
          uint32_t b[4];
          ldmatrix_x4(kb + row * kRowBytes + 16 * k_chunk(row, c), b);
          mma_16816<kF16>(sc[j], qf[k], b[0], b[1]);
          mma_16816<kF16>(sc[j], qf[k + 1], b[2], b[3]);
        }
    } else {
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        const int row = 8 * j + r8;
#pragma unroll
        for (int h = 0; h < kD / 64; ++h) {
          const uint4 w4 = lds_16(kb + row * kRowBytes + 16 * k_chunk(row, t4 + 4 * h));
          const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_16816<kF16>(sc[j], qf[4 * h + k], e4m3x2<kF16>(w[k] & 0xffffu), e4m3x2<kF16>(w[k] >> 16));
        }
      }
    }

    // ---- scores in log2 units, mask, running maximum
    const int kbase = key0(s);
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
      float ks[2] = {a.scale_log2, a.scale_log2};
      if constexpr (kFp8) {
        const uint2 u = lds_8(kb + kPagedStageBytes + (8 * j + 2 * t4) * 4);
        ks[0] *= __uint_as_float(u.x);
        ks[1] *= __uint_as_float(u.y);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int key = kbase + 8 * j + 2 * t4 + (x & 1);
        sc[j][x] = key < limit[x >> 1] ? sc[j][x] * ks[x & 1] : -INFINITY;
        mx[x >> 1] = fmaxf(mx[x >> 1], sc[j][x]);
      }
    }
    float sub[2];
    bool moved = false;
    float alpha[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
      mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
      const float m_new = fmaxf(m_run[x], mx[x]);
      sub[x] = m_new == -INFINITY ? 0.0f : m_new;  // no key so far: P = 0, no NaN
      alpha[x] = ex2_approx(m_run[x] - sub[x]);
      moved |= m_new != m_run[x];
      m_run[x] = m_new;
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int x = 0; x < 2; ++x) l_run[x] *= alpha[x];
#pragma unroll
      for (int j = 0; j < kOT; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[j][x] *= alpha[x >> 1];
    }
#pragma unroll
    for (int j = 0; j < kNT; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        sc[j][x] = ex2_approx(sc[j][x] - sub[x >> 1]);
        l_run[x >> 1] += sc[j][x];
      }

    // ---- O += P V
#pragma unroll
    for (int kk = 0; kk < kKeys / 16; ++kk) {
      if constexpr (kFp8) {
        const uint2 u0 = lds_8(kb + kPagedStageBytes + (kKeys + 16 * kk + 2 * t4) * 4);
        const uint2 u1 = lds_8(kb + kPagedStageBytes + (kKeys + 16 * kk + 8 + 2 * t4) * 4);
        const float vs[4] = {__uint_as_float(u0.x), __uint_as_float(u0.y), __uint_as_float(u1.x), __uint_as_float(u1.y)};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          sc[2 * kk][x] *= vs[x & 1];
          sc[2 * kk + 1][x] *= vs[2 + (x & 1)];
        }
      }
      const uint32_t p[4] = {pack2<kPF16>(sc[2 * kk][0], sc[2 * kk][1]), pack2<kPF16>(sc[2 * kk][2], sc[2 * kk][3]),
                             pack2<kPF16>(sc[2 * kk + 1][0], sc[2 * kk + 1][1]),
                             pack2<kPF16>(sc[2 * kk + 1][2], sc[2 * kk + 1][3])};
      if constexpr (!kFp8) {
#pragma unroll
        for (int j = 0; j < kOT; j += 2) {
          const int row = 16 * kk + (lane & 15), c = j + (lane >> 4);
          uint32_t b[4];
          ldmatrix_x4_trans(vb + row * kRowBytes + 16 * v_chunk(row, c), b);
          mma_16816<kPF16>(o[j], p, b[0], b[1]);
          mma_16816<kPF16>(o[j + 1], p, b[2], b[3]);
        }
      } else {
        // output tile j holds columns r8 * (D / 8) + j: each thread reads D / 8 neighbouring codes of its four keys
        uint32_t w[4][kD / 32];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int row = 16 * kk + 2 * t4 + (x & 1) + 8 * (x >> 1);
          if constexpr (kD == 128) {
            const uint4 v4 = lds_16(vb + row * kRowBytes + 16 * v_chunk(row, r8));
            w[x][0] = v4.x; w[x][1] = v4.y; w[x][2] = v4.z; w[x][3] = v4.w;
          } else {
            const uint2 v2 = lds_8(vb + row * kRowBytes + 16 * v_chunk(row, r8 >> 1) + 8 * (r8 & 1));
            w[x][0] = v2.x; w[x][1] = v2.y;
          }
        }
#pragma unroll
        for (int q = 0; q < kD / 32; ++q)
#pragma unroll
          for (int b = 0; b < 4; ++b)
            mma_16816<kPF16>(o[4 * q + b], p, e4m3x2<kPF16>(__byte_perm(w[0][q], w[1][q], b | ((4 + b) << 4)) & 0xffffu),
                             e4m3x2<kPF16>(__byte_perm(w[2][q], w[3][q], b | ((4 + b) << 4)) & 0xffffu));
      }
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l_run[x] += __shfl_xor_sync(0xffffffffu, l_run[x], 1);
    l_run[x] += __shfl_xor_sync(0xffffffffu, l_run[x], 2);
  }

  // ---- the four warps' results meet in shared memory
  __syncthreads();  // the stages are no longer read
  float* part = reinterpret_cast<float*>(smem);             // [warps][16][D]
  float* cta = part + kPagedWarps * kPagedRows * kD;        // [16][D] of this CTA
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int row = r8 + 8 * x;
    if (t4 == 0) {
      m_all[warp][row] = m_run[x];
      l_all[warp][row] = l_run[x];
    }
#pragma unroll
    for (int j = 0; j < kOT; ++j)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int n = 2 * t4 + y;
        const int col = kFp8 ? n * (kD / 8) + j : 8 * j + n;
        part[(warp * kPagedRows + row) * kD + col] = o[j][2 * x + y];
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kPagedRows * kD; i += kPagedThreads) {
    const int row = i / kD;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) m = fmaxf(m, m_all[w][row]);
    const float ms = m == -INFINITY ? 0.0f : m;
    float acc = 0.0f, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) {
      const float f = ex2_approx(m_all[w][row] - ms);
      acc += part[w * kPagedRows * kD + i] * f;
      l += l_all[w][row] * f;
    }
    cta[i] = acc;
    if (i % kD == 0) {
      m_cta[row] = m;
      l_cta[row] = l;
    }
  }
  // ---- the cluster's results meet through distributed shared memory: each CTA finishes a part of the rows' elements
  if (nrank > 1) ptx::cluster_sync();
  else __syncthreads();
  const uint32_t cta_s = ptx::smem_u32(cta), m_s = ptx::smem_u32(m_cta), l_s = ptx::smem_u32(l_cta);
  auto remote = [&](uint32_t addr, uint32_t r) -> float {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ptx::mapa_shared(addr, r)) : "memory");
    return v;
  };
  for (int i = 2 * (threadIdx.x + rank * kPagedThreads); i < kPagedRows * kD; i += 2 * kPagedThreads * nrank) {
    const int row = i / kD, col = i % kD;
    if (row0 + row >= rows) continue;
    float m = -INFINITY;
    for (uint32_t r = 0; r < nrank; ++r) m = fmaxf(m, remote(m_s + 4 * row, r));
    const float ms = m == -INFINITY ? 0.0f : m;
    float a0 = 0.0f, a1 = 0.0f, l = 0.0f;
    for (uint32_t r = 0; r < nrank; ++r) {
      const float f = ex2_approx(remote(m_s + 4 * row, r) - ms);
      l += remote(l_s + 4 * row, r) * f;
      a0 += remote(cta_s + 4 * i, r) * f;
      a1 += remote(cta_s + 4 * i + 4, r) * f;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a row without keys is zero
    const int64_t t = lo + (row0 + row) / a.group;
    const int h = hkv * a.group + static_cast<int>((row0 + row) % a.group);
    *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.O) + (t * a.heads + h) * kD + col) = pack2<kF16>(a0 * inv, a1 * inv);
  }
  if (nrank > 1) ptx::cluster_sync();  // no CTA leaves while another may read its shared memory
}

}  // namespace bsk
