// Attention of a few new tokens per sequence over a paged cache, for sm_100a (fp16 / bf16 queries; a cache of the
// queries' type or of e4m3 codes with one scale per slot and head).
//
// Rows: the (token, head) pairs of one sequence that share a kv head, token-major, in tiles of 8, 16 or 32. A cluster of C
// CTAs takes one tile; the keys that the tile's last row may see are split over the cluster, and each CTA deals its part
// out to its warps, stage by stage. Every warp is on its own: it copies its stages of K and V rows (8 KB each, two
// buffers) with cp.async, multiplies them with mma.sync m16n8k16 and keeps its own running maxima, sums and outputs in
// registers (one pass over the keys, softmax statistics and output in fp32). The partial results meet once at the end:
// the warps in shared memory, C CTAs through distributed shared memory, so a call is one launch without a workspace.
//
// Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T: keys (and the columns of V) fill the 16 rows of the
// instruction and the query rows its 8 columns, so 8 rows cost half of what they do as a half-empty 16-row operand --
// products, exponentials, masks and output registers -- and a larger tile uses each K / V fragment for all its rows. P^T
// goes from the first product's accumulators to the second's operand by movmatrix.
//
// Bound: HBM. A key and value are read once per tile (4 * rows * D flops for 4 * D bytes), far below the tensor pipe's
// rate; 12 warps per SM keep about 100 KB of copies in flight (three buffers for 8 warps: 135 us where this takes 121, a
// batch of 64 over e4m3 caches of 97..8192). tcgen05's 128-row tile would stay mostly empty here.
//
// e4m3 caches: the contraction's order over D (for K) and the columns' order (for V) are permuted so that each thread
// reads its codes as 16-byte words and converts them in registers, to fp16 (exact, one instruction for two codes; to bf16
// it takes five, and the conversions then are half of the kernel's instructions). So both products are fp16 products:
//   - bf16 queries are brought into fp16's range by a power of two per row, which goes back into the scores together with the
//     keys' scales: the largest element to [2^15, 2^16) (in bf16 at most 65280, below fp16's 65504), so elements down to 2^-32
//     of it stay exact and the error of the others is at most 2^-40 of it;
//   - the values' scales enter the exponent: w_j = 2^(s_j + log2 scale_j - m_w) with a running maximum m_w of its own, so
//     the rounded weights span (0, 1] whatever the scales are, and O = sum_j w_j code_j 2^(m_w) beside l = sum_j p_j 2^m.
//
// P (or w) is rounded to 16 bits for the second product (half a step: 2^-8 of a weight in bf16, 2^-11 in fp16, the
// outputs' own rounding or finer); its sum is taken in fp32 before the rounding.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "bsattn_sm100.cuh"
#include "kv_cache.cuh"

namespace bsk {

constexpr int kPagedStages = 2;
constexpr int kPagedStageBytes = 8192;  // K and V rows of one warp's stage
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
// An 8 x 8 tile of 16-bit values, spread over the warp like an accumulator, transposed.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// D (16 x 8, fp32) += A (16 x 16) B (16 x 8), fp16 or bf16 operands.
template <bool kF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (kF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four e4m3 codes -> two pairs of fp16 values, exactly.
__device__ __forceinline__ void e4m3x4(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}

__device__ __forceinline__ float log2f_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int kD, bool kFp8, int kNQ>
struct PagedShape {
  static constexpr int kRows = 8 * kNQ;                             // query rows of a tile
  static constexpr int kRowBytes = kD * (kFp8 ? 1 : 2);
  static constexpr int kKeys = kPagedStageBytes / (2 * kRowBytes);  // keys per warp stage: 16, 32 or 64
  static constexpr int kChunks = kRowBytes / 16;                    // 16-byte chunks per row: 4, 8 or 16
  static constexpr int kScaleBytes = kFp8 ? 2 * kKeys * 4 : 0;
  static constexpr int kStage = kPagedStageBytes + kScaleBytes;
  static constexpr int kWarpBytes = kPagedStages * kStage;
  static constexpr int kPitch = kD + 4;  // floats per row of the merge area: neighbouring rows in different banks
  static constexpr int kMaxWarps = kNQ == 1 ? 12 : 8;  // by registers
  static constexpr int smem_bytes(int warps) {
    const int merge = (warps + 1) * kRows * (kPitch + 4) * 4;
    return warps * kWarpBytes > merge ? warps * kWarpBytes : merge;
  }
};

template <bool kF16, int kD, bool kFp8, int kNQ>
__global__ void __launch_bounds__(32 * PagedShape<kD, kFp8, kNQ>::kMaxWarps) paged_decode_kernel(const PagedArgs a) {
  using Sh = PagedShape<kD, kFp8, kNQ>;
  constexpr int kRows = Sh::kRows, kKeys = Sh::kKeys, kChunks = Sh::kChunks, kRowBytes = Sh::kRowBytes;
  constexpr int kKS = kD / 16;          // k16 steps of K Q^T
  constexpr int kBlk = kKeys / 16;      // 16-key blocks of a stage
  constexpr int kMT = kD / 16;          // m16 tiles of O^T
  constexpr int kLd = kNQ == 4 ? 2 : 4;  // 16-bit fragments loaded together
  constexpr bool kMF16 = kF16 || kFp8;  // fp16 operands
  extern __shared__ __align__(128) uint8_t smem[];

  uint32_t nrank, rank;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(nrank));
  asm volatile("mov.u32 %0, %%cluster_ctaid.x;" : "=r"(rank));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_threads = blockDim.x, n_warps = n_threads >> 5;
  const int t4 = lane & 3, r8 = lane >> 2;
  const int64_t tile = blockIdx.x / nrank;
  const int hkv = blockIdx.y;

  // ---- which sequence and rows (the same for the whole cluster, so a return leaves nobody waiting)
  int seq, lo, hi, kv_len;
  if (a.batch < 32) {  // one round of loads: every lane has one sequence's bounds
    const int raw = __ldg(&a.cu_seqlens[min(lane, a.batch)]);
    kv_len = lane < a.batch ? __ldg(&a.kv_lens[lane]) : 0;
    const int start = lane == 0 ? 0 : min(max(raw, 0), a.tokens);
    const int64_t base = static_cast<int64_t>(start) * a.group / kRows + lane;
    seq = 31 - __clz(__ballot_sync(0xffffffffu, lane <= a.batch && base <= tile) | 1u);
    lo = __shfl_sync(0xffffffffu, start, seq);
    hi = min(max(__shfl_sync(0xffffffffu, raw, min(seq + 1, a.batch)), lo), a.tokens);
    kv_len = __shfl_sync(0xffffffffu, kv_len, seq);
  } else {
    seq = find_seq(a.cu_seqlens, a.batch, a.tokens, a.group, kRows, tile);
    bool bad;
    const int i = min(seq, a.batch - 1);
    seq_rows(a.cu_seqlens, i, a.tokens, lo, hi, bad);
    kv_len = __ldg(&a.kv_lens[i]);
  }
  if (seq == a.batch) {  // rows behind the last sequence are zero
    if (blockIdx.x == gridDim.x - 1 && hkv == 0)  // the last tile of the grid always comes here
      for (int i = threadIdx.x; i < a.batch; i += n_threads) {
        int r0, r1;
        bool bad;
        seq_rows(a.cu_seqlens, i, a.tokens, r0, r1, bad);
        if (bad) paged_flag(a.err, 1);
      }
    const int end = min(max(__ldg(&a.cu_seqlens[a.batch]), 0), a.tokens);
    const int64_t base = static_cast<int64_t>(end) * a.group / kRows + a.batch;
    const int64_t first = static_cast<int64_t>(end) * a.group + (tile - base) * kRows;
    constexpr int kOc = kD / 8;
    for (int i = threadIdx.x + rank * n_threads; i < kRows * kOc; i += n_threads * nrank) {
      const int64_t row = first + i / kOc;
      if (row < static_cast<int64_t>(a.tokens) * a.group) {
        const int64_t t = row / a.group;
        const int h = hkv * a.group + static_cast<int>(row % a.group);
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.O) + (t * a.heads + h) * kD)[i % kOc] = make_uint4(0, 0, 0, 0);
      }
    }
    return;
  }
  const int64_t base = static_cast<int64_t>(lo) * a.group / kRows + seq;
  const int64_t row0 = (tile - base) * kRows;                    // first packed row of the tile
  const int64_t rows = static_cast<int64_t>(hi - lo) * a.group;  // packed rows of the sequence
  if (row0 >= rows) return;
  const int64_t room = static_cast<int64_t>(a.table_width) << a.page_shift;
  if (kv_len < 0 || kv_len > room) {
    if (threadIdx.x == 0) paged_flag(a.err, 2);
    kv_len = kv_len < 0 ? 0 : static_cast<int>(room);
  }
  const int first_pos = kv_len - (hi - lo);  // position of the chunk's first token (negative: rows without keys)
  const int last_row = static_cast<int>(min(row0 + kRows, rows) - 1);
  const int keys_end = max(first_pos + last_row / a.group + 1, 0);                 // keys that the tile's last row sees
  const int clear = first_pos + static_cast<int>(row0 / a.group) + 1;              // keys that every row sees

  // ---- keys in pieces of kKeys: a run of them for each CTA of the cluster, dealt out to its warps
  const int pieces = (keys_end + kKeys - 1) / kKeys, per = (pieces + nrank - 1) / nrank;
  const int first_piece = min(static_cast<int>(rank) * per, pieces) + warp;
  const int end_piece = min(static_cast<int>(rank + 1) * per, pieces);
  const int n_stages = first_piece < end_piece ? (end_piece - first_piece + n_warps - 1) / n_warps : 0;

  // ---- copies: stage s of this warp = keys [key0(s), key0(s) + kKeys)
  const uint32_t wbase = ptx::smem_u32(smem) + warp * Sh::kWarpBytes;
  const int* table = a.block_table + seq * a.table_stride;
  auto key0 = [&](int s) { return (first_piece + s * n_warps) * kKeys; };
  constexpr int kSl = (kKeys + 31) / 32;
  int slot_of[kSl];  // lane l: slots of keys l (and l + 32) of the stage to be copied next, -1: none
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
          slot_of[x] = (page << a.page_shift) + (key & ((1 << a.page_shift) - 1));
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
  const int lane_row = lane / kChunks, lane_chunk = lane % kChunks;
  const uint8_t* k_src = static_cast<const uint8_t*>(a.k_cache) + hkv * kRowBytes + 16 * lane_chunk;
  const uint8_t* v_src = static_cast<const uint8_t*>(a.v_cache) + hkv * kRowBytes + 16 * lane_chunk;
  const int row_stride = a.kv_heads * kRowBytes;
  auto copy = [&](int s) {
    if (s < n_stages) {
      const uint32_t dst = wbase + (s % kPagedStages) * Sh::kStage;
      constexpr int kPer = 32 / kChunks;  // rows copied at once
#pragma unroll
      for (int r0 = 0; r0 < kKeys; r0 += kPer) {
        const int row = r0 + lane_row;
        const int slot = __shfl_sync(0xffffffffu, slot_of[r0 / 32], row & 31);
        const int64_t off = static_cast<int64_t>(max(slot, 0)) * row_stride;
        cp_async_16(dst + row * kRowBytes + 16 * k_chunk(row, lane_chunk), k_src + off, slot >= 0);
        cp_async_16(dst + kPagedStageBytes / 2 + row * kRowBytes + 16 * v_chunk(row, lane_chunk), v_src + off, slot >= 0);
      }
      if (kFp8) {
#pragma unroll
        for (int x = 0; x < kSl; ++x) {
          const int64_t off = static_cast<int64_t>(max(slot_of[x], 0)) * a.kv_heads + hkv;
          const uint32_t sdst = dst + kPagedStageBytes + (lane + 32 * x) * 4;
          cp_async_4(sdst, a.k_scale + off, slot_of[x] >= 0);
          cp_async_4(sdst + kKeys * 4, a.v_scale + off, slot_of[x] >= 0);
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < kPagedStages - 1; ++s) {
    look_up(s);
    copy(s);
  }
  look_up(kPagedStages - 1);

  // ---- queries as B fragments: row r8 (+ 8 q) of the tile
  uint32_t qf[kNQ][kKS][2];
  float row_up[kNQ];  // what row r8 + 8 q was divided by
#pragma unroll
  for (int q = 0; q < kNQ; ++q) {
    const int64_t row = row0 + r8 + 8 * q;
    const bool live = row < rows;
    const int tok = live ? static_cast<int>(row / a.group) : 0;
    const int head = hkv * a.group + (live ? static_cast<int>(row % a.group) : 0);
    const uint16_t* p = static_cast<const uint16_t*>(a.Q) + (lo + tok) * a.q_token_stride + head * a.q_head_stride;
#pragma unroll
    for (int k = 0; k < kKS; ++k) {
      // element pairs of k step k: {2 t4, 2 t4 + 1} and {+8, +9}; e4m3: four neighbours 64 h + 16 t4 + 4 w (k = 4 h + w)
      const int d0 = kFp8 ? 64 * (k >> 2) + 16 * t4 + 4 * (k & 3) : 16 * k + 2 * t4;
      const int d1 = kFp8 ? d0 + 2 : d0 + 8;
      qf[q][k][0] = live ? *reinterpret_cast<const uint32_t*>(p + d0) : 0u;
      qf[q][k][1] = live ? *reinterpret_cast<const uint32_t*>(p + d1) : 0u;
    }
    row_up[q] = 1.0f;
    if constexpr (kFp8 && !kF16) {  // bf16 -> fp16, the row's largest element brought to [2^15, 2^16)
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < kKS; ++k)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t w = qf[q][k][y] & 0x7fff7fffu;
          top = max(top, max(w >> 16, w & 0xffffu));
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = max(static_cast<int>(top >> 7), 40) - 142;  // exponent of the largest, less 15
      const float down = __int_as_float((127 - e) << 23);
      row_up[q] = __int_as_float((127 + e) << 23);
#pragma unroll
      for (int k = 0; k < kKS; ++k)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float2 f = unpack2<false>(qf[q][k][y]);
          qf[q][k][y] = pack_f16(f.x * down, f.y * down);
        }
    }
  }
  // This thread's columns of S^T are rows 8 q + 2 t4 + y: their limits (keys at or beyond are masked) and scales (softmax
  // scale * log2(e), times row_up, which the row's own lanes 4 r .. 4 r + 3 hold).
  int limit[kNQ][2];
  float row_scale[kNQ][2];
#pragma unroll
  for (int q = 0; q < kNQ; ++q)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int64_t row = row0 + 8 * q + 2 * t4 + y;
      limit[q][y] = row < rows ? first_pos + static_cast<int>(row / a.group) + 1 : 0;
      row_scale[q][y] = a.scale_log2;
      if constexpr (kFp8 && !kF16) row_scale[q][y] *= __shfl_sync(0xffffffffu, row_up[q], 4 * (2 * t4 + y));
    }

  float o[kMT][kNQ][4];
#pragma unroll
  for (int j = 0; j < kMT; ++j)
#pragma unroll
    for (int q = 0; q < kNQ; ++q)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[j][q][x] = 0.0f;
  // running maxima of the scores and of score + log2(value's scale) (the same without scales), and this thread's sums of P
  float m_run[kNQ][2], w_run[kNQ][2], l_run[kNQ][2];
#pragma unroll
  for (int q = 0; q < kNQ; ++q)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      m_run[q][y] = w_run[q][y] = -INFINITY;
      l_run[q][y] = 0.0f;
    }

  for (int s = 0; s < n_stages; ++s) {
    __syncwarp();  // every lane is done with the buffer that the next copy overwrites
    copy(s + kPagedStages - 1);
    look_up(s + kPagedStages);
    cp_async_wait<kPagedStages - 1>();
    __syncwarp();
    const uint32_t kb = wbase + (s % kPagedStages) * Sh::kStage, vb = kb + kPagedStageBytes / 2;
    const uint8_t* kp = smem + warp * Sh::kWarpBytes + (s % kPagedStages) * Sh::kStage;
    const uint8_t* vp = kp + kPagedStageBytes / 2;
    const float* ks_p = reinterpret_cast<const float*>(kp + kPagedStageBytes);  // e4m3: the keys' scales, the values' scales

    // ---- S^T: keys r8 and r8 + 8 of each 16-key block, rows 2 t4 and 2 t4 + 1 of each 8
    float sc[kBlk][kNQ][4];
#pragma unroll
    for (int j = 0; j < kBlk; ++j)
#pragma unroll
      for (int q = 0; q < kNQ; ++q)
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[j][q][x] = 0.0f;
    // (with 8 rows there are few products at once: two chains of them per block shorten their latency)
    constexpr int kChains = kNQ == 1 ? 2 : 1;
    float sc1[kBlk][kNQ][4];
    if constexpr (kChains == 2) {
#pragma unroll
      for (int j = 0; j < kBlk; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) sc1[j][0][x] = 0.0f;
    }
    if constexpr (!kFp8) {
#pragma unroll
      for (int j = 0; j < kBlk; ++j)
#pragma unroll
        for (int k0 = 0; k0 < kKS; k0 += kLd) {
          uint32_t f[kLd][4];  // loads first, so that they are in flight together
#pragma unroll
          for (int k = 0; k < kLd; ++k) {
            const int row = 16 * j + (lane & 15), c = 2 * (k0 + k) + (lane >> 4);
            ldmatrix_x4(kb + row * kRowBytes + 16 * k_chunk(row, c), f[k]);
          }
#pragma unroll
          for (int k = 0; k < kLd; ++k)
#pragma unroll
            for (int q = 0; q < kNQ; ++q)
              mma_16816<kMF16>(kChains == 2 && (k & 1) ? sc1[j][q] : sc[j][q], f[k], qf[q][k0 + k][0], qf[q][k0 + k][1]);
        }
    } else {
#pragma unroll
      for (int j = 0; j < kBlk; ++j) {
        const int row = 16 * j + r8;
#pragma unroll
        for (int h = 0; h < kD / 64; ++h) {
          const uint4 u4 = *reinterpret_cast<const uint4*>(kp + row * kRowBytes + 16 * k_chunk(row, t4 + 4 * h));
          const uint4 v4 = *reinterpret_cast<const uint4*>(kp + (row + 8) * kRowBytes + 16 * k_chunk(row + 8, t4 + 4 * h));
          const uint32_t u[4] = {u4.x, u4.y, u4.z, u4.w}, v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t f[4];
            e4m3x4(u[k], f[0], f[2]);
            e4m3x4(v[k], f[1], f[3]);
#pragma unroll
            for (int q = 0; q < kNQ; ++q)
              mma_16816<kMF16>(kChains == 2 && (k & 1) ? sc1[j][q] : sc[j][q], f, qf[q][4 * h + k][0], qf[q][4 * h + k][1]);
          }
        }
      }
    }
    if constexpr (kChains == 2) {
#pragma unroll
      for (int j = 0; j < kBlk; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[j][0][x] += sc1[j][0][x];
    }

    // ---- scores in log2 units, mask, running maxima
    float lv[kFp8 ? kBlk : 1][2];  // log2 of the values' scales of this thread's keys
    const int kbase = key0(s);
    const bool edge = kbase + kKeys > clear;  // some row does not see the whole stage
#pragma unroll
    for (int j = 0; j < kBlk; ++j) {
      float ks[2] = {1.0f, 1.0f};
      if constexpr (kFp8) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          ks[y] = ks_p[16 * j + r8 + 8 * y];
          lv[j][y] = log2f_approx(ks_p[kKeys + 16 * j + r8 + 8 * y]);
        }
      }
#pragma unroll
      for (int q = 0; q < kNQ; ++q)
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[j][q][x] *= kFp8 ? row_scale[q][x & 1] * ks[x >> 1] : row_scale[q][x & 1];
    }
    if (edge) {
#pragma unroll
      for (int j = 0; j < kBlk; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int key = kbase + 16 * j + r8 + 8 * (x >> 1);
#pragma unroll
          for (int q = 0; q < kNQ; ++q)
            if (key >= limit[q][x & 1]) sc[j][q][x] = -INFINITY;
          if constexpr (kFp8)  // a key that no row sees: its scale is not looked at
            if (key >= keys_end) lv[j][x >> 1] = -INFINITY;
        }
    }
    float m_sub[kNQ][2], w_sub[kNQ][2], alpha[kNQ][2], beta[kNQ][2];
    bool moved = false;
#pragma unroll
    for (int q = 0; q < kNQ; ++q)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float mx = fmaxf(sc[0][q][y], sc[0][q][2 + y]), wx = kFp8 ? fmaxf(sc[0][q][y] + lv[0][0], sc[0][q][2 + y] + lv[0][1]) : 0.0f;
#pragma unroll
        for (int j = 1; j < kBlk; ++j) {
          mx = fmaxf(mx, fmaxf(sc[j][q][y], sc[j][q][2 + y]));
          if constexpr (kFp8) wx = fmaxf(wx, fmaxf(sc[j][q][y] + lv[j][0], sc[j][q][2 + y] + lv[j][1]));
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          if constexpr (kFp8) wx = fmaxf(wx, __shfl_xor_sync(0xffffffffu, wx, d));
        }
        const float m_new = fmaxf(m_run[q][y], mx);
        m_sub[q][y] = m_new == -INFINITY ? 0.0f : m_new;  // no key so far: P = 0, no NaN
        alpha[q][y] = ex2_approx(m_run[q][y] - m_sub[q][y]);
        moved |= m_new != m_run[q][y];
        m_run[q][y] = m_new;
        if constexpr (kFp8) {
          const float w_new = fmaxf(w_run[q][y], wx);
          w_sub[q][y] = w_new == -INFINITY ? 0.0f : w_new;
          beta[q][y] = ex2_approx(w_run[q][y] - w_sub[q][y]);
          moved |= w_new != w_run[q][y];
          w_run[q][y] = w_new;
        } else {
          beta[q][y] = alpha[q][y];
        }
      }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int q = 0; q < kNQ; ++q) {
        l_run[q][0] *= alpha[q][0];
        l_run[q][1] *= alpha[q][1];
#pragma unroll
        for (int j = 0; j < kMT; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[j][q][x] *= beta[q][x & 1];
      }
    }

    // ---- O^T += V^T P^T, 16 keys at a time
#pragma unroll
    for (int j = 0; j < kBlk; ++j) {
      uint32_t pf[kNQ][2];
#pragma unroll
      for (int q = 0; q < kNQ; ++q) {
        float e[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float p = ex2_approx(sc[j][q][x] - m_sub[q][x & 1]);
          l_run[q][x & 1] += p;
          e[x] = kFp8 ? ex2_approx(sc[j][q][x] + lv[j][x >> 1] - w_sub[q][x & 1]) : p;
        }
        pf[q][0] = movmatrix_trans(pack2<kMF16>(e[0], e[1]));
        pf[q][1] = movmatrix_trans(pack2<kMF16>(e[2], e[3]));
      }
      if constexpr (!kFp8) {
#pragma unroll
        for (int m0 = 0; m0 < kMT; m0 += kLd) {
          uint32_t f[kLd][4];
#pragma unroll
          for (int mt = 0; mt < kLd; ++mt) {
            const int row = 16 * j + (lane & 7) + 8 * (lane >> 4), c = 2 * (m0 + mt) + ((lane >> 3) & 1);
            ldmatrix_x4_trans(vb + row * kRowBytes + 16 * v_chunk(row, c), f[mt]);
          }
#pragma unroll
          for (int mt = 0; mt < kLd; ++mt)
#pragma unroll
            for (int q = 0; q < kNQ; ++q) mma_16816<kMF16>(o[m0 + mt][q], f[mt], pf[q][0], pf[q][1]);
        }
      } else {
        // rows r8 and r8 + 8 of output tile mt are columns r8 * (D / 8) + 2 mt and the next: each thread reads D / 8
        // neighbouring codes of its four keys and pairs up the keys' bytes of a column
        uint32_t w[4][kD / 32];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int row = 16 * j + 2 * t4 + (x & 1) + 8 * (x >> 1);
          if constexpr (kD == 128) {
            const uint4 v4 = *reinterpret_cast<const uint4*>(vp + row * kRowBytes + 16 * v_chunk(row, r8));
            w[x][0] = v4.x; w[x][1] = v4.y; w[x][2] = v4.z; w[x][3] = v4.w;
          } else {
            const uint2 v2 = *reinterpret_cast<const uint2*>(vp + row * kRowBytes + 16 * v_chunk(row, r8 >> 1) + 8 * (r8 & 1));
            w[x][0] = v2.x; w[x][1] = v2.y;
          }
        }
#pragma unroll
        for (int i = 0; i < kD / 32; ++i)
#pragma unroll
          for (int b = 0; b < 2; ++b) {  // columns 2 b and 2 b + 1 of word i
            const uint32_t u = __byte_perm(w[0][i], w[1][i], b ? 0x7362 : 0x5140);
            const uint32_t v = __byte_perm(w[2][i], w[3][i], b ? 0x7362 : 0x5140);
            uint32_t f[4];
            e4m3x4(u, f[0], f[1]);
            e4m3x4(v, f[2], f[3]);
#pragma unroll
            for (int q = 0; q < kNQ; ++q) mma_16816<kMF16>(o[2 * i + b][q], f, pf[q][0], pf[q][1]);
          }
      }
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int q = 0; q < kNQ; ++q)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l_run[q][y] += __shfl_xor_sync(0xffffffffu, l_run[q][y], d);

  // ---- the warps' results meet in shared memory: [warps + 1][rows] of D sums, and of (m, l, m_w)
  __syncthreads();  // the stages are no longer read
  float* sums = reinterpret_cast<float*>(smem);
  constexpr int kPitch = Sh::kPitch;
  float4* stat = reinterpret_cast<float4*>(sums + (n_warps + 1) * kRows * kPitch);
#pragma unroll
  for (int q = 0; q < kNQ; ++q)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int row = warp * kRows + 8 * q + 2 * t4 + y;
      if (r8 == 0) stat[row] = make_float4(m_run[q][y], l_run[q][y], kFp8 ? w_run[q][y] : m_run[q][y], 0.0f);
      if constexpr (kFp8) {
#pragma unroll
        for (int j = 0; j < kMT; j += 2)
          *reinterpret_cast<float4*>(sums + row * kPitch + r8 * (kD / 8) + 2 * j) =
              make_float4(o[j][q][y], o[j][q][2 + y], o[j + 1][q][y], o[j + 1][q][2 + y]);
      } else {
#pragma unroll
        for (int j = 0; j < kMT; ++j) {
          sums[row * kPitch + 16 * j + r8] = o[j][q][y];
          sums[row * kPitch + 16 * j + 8 + r8] = o[j][q][2 + y];
        }
      }
    }
  __syncthreads();
  constexpr int kParts = kD / 4;                // float4 pieces of a row
  const int tpr = n_threads / kRows;            // threads per row
  {
    const int row = threadIdx.x / tpr;
    float m = -INFINITY, w = -INFINITY, l = 0.0f;
#pragma unroll 4
    for (int i = 0; i < n_warps; ++i) {
      const float4 st = stat[i * kRows + row];
      m = fmaxf(m, st.x);
      w = fmaxf(w, st.z);
    }
    const float ms = m == -INFINITY ? 0.0f : m, wsub = w == -INFINITY ? 0.0f : w;
    for (int c = threadIdx.x % tpr; c < kParts; c += tpr) {
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      l = 0.0f;
#pragma unroll 4
      for (int i = 0; i < n_warps; ++i) {
        const float4 st = stat[i * kRows + row], v = reinterpret_cast<const float4*>(sums + (i * kRows + row) * kPitch)[c];
        l += st.y * ex2_approx(st.x - ms);
        const float f = ex2_approx(st.z - wsub);
        acc.x += v.x * f;
        acc.y += v.y * f;
        acc.z += v.z * f;
        acc.w += v.w * f;
      }
      reinterpret_cast<float4*>(sums + (n_warps * kRows + row) * kPitch)[c] = acc;
    }
    if (threadIdx.x % tpr == 0) stat[n_warps * kRows + row] = make_float4(m, l, w, 0.0f);
  }
  // ---- the cluster's results meet through distributed shared memory: each CTA finishes a part of the tile
  if (nrank > 1) ptx::cluster_sync();
  else __syncthreads();
  const uint32_t sums_s = ptx::smem_u32(sums + n_warps * kRows * kPitch), stat_s = ptx::smem_u32(stat + n_warps * kRows);
  auto remote = [&](uint32_t addr, uint32_t r) -> float4 {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(ptx::mapa_shared(addr, r))
                 : "memory");
    return v;
  };
  for (int i = threadIdx.x + rank * n_threads; i < kRows * kParts; i += n_threads * nrank) {
    const int row = i / kParts, c = i % kParts;
    if (row0 + row >= rows) continue;
    float m = -INFINITY, w = -INFINITY;
#pragma unroll 4
    for (uint32_t r = 0; r < nrank; ++r) {
      const float4 st = remote(stat_s + 16 * row, r);
      m = fmaxf(m, st.x);
      w = fmaxf(w, st.z);
    }
    const float ms = m == -INFINITY ? 0.0f : m, wsub = w == -INFINITY ? 0.0f : w;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
#pragma unroll 4
    for (uint32_t r = 0; r < nrank; ++r) {
      const float4 st = remote(stat_s + 16 * row, r), v = remote(sums_s + (row * kPitch + 4 * c) * 4, r);
      l += st.y * ex2_approx(st.x - ms);
      const float f = ex2_approx(st.z - wsub);
      acc.x += v.x * f;
      acc.y += v.y * f;
      acc.z += v.z * f;
      acc.w += v.w * f;
    }
    // A row without keys is zero; so is one whose values' scales are all zero, whatever its scores are (m_w = -inf: every
    // weight was zero, and 2^-m may be infinite).
    const float up = w == -INFINITY ? 1.0f : ex2_approx(wsub - ms);
    const float inv = l == 0.0f ? 0.0f : up / l;
    const int64_t t = lo + (row0 + row) / a.group;
    const int h = hkv * a.group + static_cast<int>((row0 + row) % a.group);
    reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.O) + (t * a.heads + h) * kD)[c] =
        make_uint2(pack2<kF16>(acc.x * inv, acc.y * inv), pack2<kF16>(acc.z * inv, acc.w * inv));
  }
  if (nrank > 1) ptx::cluster_sync();  // no CTA leaves while another may read its shared memory
}

}  // namespace bsk
