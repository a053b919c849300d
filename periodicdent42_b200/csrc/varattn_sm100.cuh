// Attention over packed sequences, or of chunks of new tokens over a paged cache, for sm_100a (fp16 / bf16, head dim 64 or
// 128, grouped heads): forward, tcgen05.
//
// Work item = a tile of query rows -- TT = 128 / group tokens x the group's heads, so that the 128 rows of the tensor core's
// tile all use the same keys -- and its key blocks [b0, b1) of 128 keys (varattn_plan.cuh). For every key block
//     S_j = Q K_j^T                 tcgen05.mma 128x128x16 x (D/16) into TMEM S buffer j % 2
//     P_j = exp2(S_j * c - m)       online softmax, 16-bit P written back into the S buffer
//     O  += P_j V_j                 tcgen05.mma with A = P from TMEM, V an MN-major shared-memory operand
// and O / l (and the log-sum-exp) at the end. The CTA's shape and its softmax are those of the block-sparse forward
// (bsattn_sm100.cuh, where they are explained and measured): warp 0 TMA producer, warps 1 and 2 issue S and PV, warps 4-11
// softmax (two warps per row quarter, each half of the keys), warps 12-15 output. What differs:
//   - Q tiles come as 3-D boxes (64 columns x group heads x TT tokens) from any token / head stride, K and V tiles as boxes
//     of one head x 128 tokens, or, paged, as one 5-D box per page: a copy costs about 70 ns of the CTA's one copy engine
//     whatever its size, and pages of 16 rows need 16 of them per key block (2048 new tokens over 16384, 32 / 8 heads,
//     D 128: 744 us; with one copy per 64-column chunk of a page 1000; pages of 32 rows 625, of 64 and more 610).
//   - Keys that a row may not see are masked by position; only blocks that reach behind the tile's first row's limit
//     compare. A row without any key keeps its maximum at -inf and is written as zero.
//   - The last block of a sequence may hold foreign rows (the next sequence's, or stale page contents, NaN among them). Their
//     scores are replaced, but P = 0 does not stop a NaN in V: warp 3 sets those V rows to zero in shared memory between the
//     copy's arrival and the PV product (only such blocks take this detour).
//
// e4m3 caches (kKind 2): both products are fp16 products. Warps 12-15, which otherwise only write results, convert: codes
// arrive by the same copies in a staging ring, a thread takes a key's row and writes it as fp16 (one instruction for two
// codes, exact) to the K / V ring, rows behind the sequence as zeros. Warp 3 brings the blocks' scales. The keys' scales
// multiply the scores. The values' scales multiply P, brought near 1 by a power of two R of each row that follows the
// largest scale that the row has seen (O is rescaled when R grows), so that P * scale stays within fp16's range: values'
// scales down to 2^-20 of that keep P's full precision. Warp 3 divides the scales by the tile's largest power of two; in the
// last blocks, where a row may not see the key that it came from, the rest to the row's own goes into the exponent of P
// (done in every block, this took a sixth more time). bf16 queries are turned into fp16 in place, each row by its own power
// of two: exact for elements down to 2^-32 of the row's largest, the error of the others at most 2^-40 of it.
// Bound here: the conversion's one warp per sub-partition beside the softmax's two (8100 warp instructions a block where
// 16-bit caches take 4100), and instructions: the roles share the instruction cache, and with more code in their loops they
// wait for it. So the conversion's and the two issuers' loops are rolled (1024 new tokens over 30000, 32 / 8 heads, D 128:
// 1047 us; when it was 1033: conversion unrolled 1126, issuers unrolled 1189, both 1203; 16-bit cache 555).
//
// P is rounded to the operands' type (half a step: 2^-8 of a weight in bf16, 2^-11 in fp16), its sums are fp32 and taken before.
//
// Bound: each key block's own chain of steps -- scores, maximum, exchange between the two warps of a row, exponentials, P, with
// one query tile in flight per CTA; no pipe is at its limit (8192 tokens, 32 / 8 heads, D 128: tensor pipe 47 % of the time,
// issue 49 %, XU 35 %, DRAM 3 %; 552 us in short runs, 646 when repeated under the power cap). Packing the group's heads into
// the tile means a causal tile spans only TT tokens, so less of its last block is masked, and one K / V tile feeds the whole
// group.
#pragma once

#include "bsattn_bwd_sm100.cuh"
#include "varattn_plan.cuh"

namespace bsk {

// Maxima that pass a NaN on (a NaN score has to reach the row's result).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Rows of a [128 x D] tile that no copy fills (128 is no multiple of the group): zeroed once by the whole CTA.
__device__ __forceinline__ void zero_tile_rows(uint8_t* tile, int chunks, int first) {
  for (int i = threadIdx.x; i < (kVarBlk - first) * chunks * 8; i += blockDim.x) {
    const int r = first + i / (chunks * 8), c = i % (chunks * 8);
    *reinterpret_cast<uint4*>(tile + (c >> 3) * kAttnChunk + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
}

// Exponent fields that value scales count as (e4m3 caches): 2^(133 - field) and 2^(field - 133) are normal numbers. A row's
// reference is at most kScaleSpan below its tile's, so that 2^8 * 2^kScaleSpan, 64 times, is finite.
constexpr int kScaleLow = 20, kScaleHigh = 240, kScaleSpan = 110;

// Floor of the exponentials on the FMA pipe: weights below 2^-126 are zero, so that no masked or far key, however large its
// values are, adds to a row.
constexpr int kVarFloor = -127;

// Where the K / V rows come from.
enum : int { kPacked = 0, kCache16 = 1, kCacheE4m3 = 2 };

template <bool kF16, int kD, int kKind>
struct VarShape {
  static constexpr bool kE4m3 = kKind == kCacheE4m3;
  static constexpr int kTile = kVarBlk * kD * 2;
  static constexpr int kChunks = kD / 64;
  static constexpr int kSlots = kE4m3 && kD == 128 ? 3 : 5;  // K / V ring
  static constexpr int kStages = kE4m3 ? 3 : 0;              // staging ring of code tiles
  static constexpr int kStageBytes = kVarBlk * kD;
  // barriers 512 B, sums and maxima, and for e4m3, two of each: keys' and values' scales, exponents of the largest value scale
  // up to a key, rows' scales, rows' closing factors, the tile's exponent, the one before, its step
  static constexpr int kSmallBytes = 512 + 3 * 128 * 4 + (kE4m3 ? (5 * 256 + 6) * 4 : 0);
  static constexpr int kSmemBytes = 1024 + kTile * (2 + kSlots) + kStages * kStageBytes + kSmallBytes;
  static constexpr uint32_t kFmt = kF16 || kE4m3 ? 0u : 1u;  // tcgen05 kind::f16 operands: 0 f16, 1 bf16
  static_assert(kSmemBytes <= 232448, "shared memory above the 227 KB per-CTA limit");
};

struct VarFwdArgs {
  void* O;              // contiguous [tokens, heads, D]
  float* lse;           // optional [tokens, heads], natural log
  const VarItem* items;
  const int* count;     // entries of `items`
  float* part_o;        // split entries: [pieces][kv heads][128 rows][D], each piece's rows divided by its own sums
  float* part_lse;      // [pieces][kv heads][128], log2 of the piece's sum of 2^score (-inf: no key)
  const int* table;     // paged: block table
  int64_t table_stride;
  int page_shift, num_pages;
  const float* k_scale; // e4m3 caches: [pages, page size, kv heads]
  const float* v_scale;
  int heads, kv_heads, group, causal;
  float scale_log2;
  uint32_t* err;
  uint64_t timeout_ns;
};

template <bool kF16, int kD, int kKind>
__global__ void __launch_bounds__(kAttnThreads, 1)
    varattn_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const VarFwdArgs a) {
  using Sh = VarShape<kF16, kD, kKind>;
  constexpr bool kPaged = kKind != kPacked, kE4m3 = kKind == kCacheE4m3;
  constexpr bool kOpF16 = kF16 || kE4m3;  // type of the products' operands
  constexpr int kTile = Sh::kTile, kSlots = Sh::kSlots, kStages = Sh::kStages;
  constexpr int kHalfD = kD / 2;
  // K / V tiles in shared memory: atoms of 8 rows x 128 bytes. Packed: a 64-column chunk's 16 atoms, then the next chunk's
  // (one copy per chunk). Paged: the chunks of 8 rows together, so that one copy brings a whole page.
  constexpr int kGroupPitch = kKind == kCache16 ? 1024 * Sh::kChunks : 1024;  // from 8 rows to the next 8
  constexpr int kChunkPitch = kKind == kCache16 ? 1024 : kAttnChunk;          // from 64 columns to the next 64
  constexpr uint32_t IDESC_S = ptx::instr_desc(128, 128, Sh::kFmt, Sh::kFmt, 0, 0);
  constexpr uint32_t IDESC_PV = ptx::instr_desc(128, kD, Sh::kFmt, Sh::kFmt, 0, 1);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                      // [2] Q of alternate items
  uint8_t* sKV = sQ + 2 * kTile;           // [kSlots]
  uint8_t* sRaw = sKV + kSlots * kTile;    // [kStages] code tiles
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRaw + kStages * Sh::kStageBytes);
  uint64_t* q_full = bars + 0;                       // [2]
  uint64_t* q_empty = bars + 2;                      // [2]
  uint64_t* kv_full = bars + 4;                      // [kSlots]
  uint64_t* kv_empty = kv_full + kSlots;             // [kSlots]
  uint64_t* raw_full = kv_empty + kSlots;            // [kSlots] a V tile with foreign rows has arrived (16-bit)
  uint64_t* stg_full = raw_full;                     // [kStages] a code tile has arrived (e4m3)
  uint64_t* stg_empty = stg_full + kStages;          // [kStages] it has been converted (4 warps)
  uint64_t* q_raw = stg_empty + kStages;             // [2] Q as it was copied (e4m3)
  uint64_t* sc_full = q_raw + 2;                     // [2] a block's scales are in shared memory (4 warps; e4m3)
  constexpr int kMore = kE4m3 ? 2 * kStages + 4 : kSlots;
  uint64_t* s_full = raw_full + kMore;               // [2]
  uint64_t* s_free = s_full + 2;                     // [2]
  uint64_t* p_full = s_free + 2;                     // [2]
  uint64_t* o_done = p_full + 2;                     // [2]
  uint64_t* xbar = o_done + 2;                       // [8]
  uint64_t* drain = xbar + 8;                        // [2]
  uint64_t* l_ready = drain + 2;
  uint64_t* o_free = l_ready + 1;                    // [2]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(o_free + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert(4 + 2 * kSlots + kMore + 2 + 2 + 2 + 2 + 8 + 2 + 1 + 2 <= 63, "barrier area exceeds its 512 bytes");
  float* l_part = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 512);  // [2 halves][128 rows]
  float* m_row = l_part + 256;                                                       // [128 rows]
  float* k_sc = m_row + 128;  // e4m3: [2][128] keys' scales
  float* v_sc = k_sc + 256;   // [2][128] values' scales / 2^(exponent of the tile)
  float* q_sc = v_sc + 256;   // [2][128] what the query rows were divided by
  int* v_top = reinterpret_cast<int*>(q_sc + 256);  // [2][128] exponent field of the largest value scale up to key i
  float* r_end = reinterpret_cast<float*>(v_top + 256);  // [2][128] what the rows' O is multiplied by at the end of alternate items
  int* r_tile = reinterpret_cast<int*>(r_end + 256);     // [2] exponent field of the tile's largest value scale so far
  int* r_before = r_tile + 2;                            // [2] that before the block
  float* r_step = reinterpret_cast<float*>(r_tile + 4);  // [2] 2^(r_before - r_tile)

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int group = a.group, tt = kVarBlk / group;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(ptx::smem_u32(&q_full[s]), kE4m3 ? 4 : 1);
      ptx::mbar_init(ptx::smem_u32(&q_empty[s]), 1);
      if (kE4m3) {
        ptx::mbar_init(ptx::smem_u32(&q_raw[s]), 1);
        ptx::mbar_init(ptx::smem_u32(&sc_full[s]), 1);
      }
      ptx::mbar_init(ptx::smem_u32(&s_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&s_free[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&p_full[s]), 8);
      ptx::mbar_init(ptx::smem_u32(&drain[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&o_done[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&o_free[s]), 4);
    }
    for (int s = 0; s < kSlots; ++s) {
      ptx::mbar_init(ptx::smem_u32(&kv_full[s]), kE4m3 ? 4 : 1);
      ptx::mbar_init(ptx::smem_u32(&kv_empty[s]), 1);
      if (!kE4m3) ptx::mbar_init(ptx::smem_u32(&raw_full[s]), 1);
    }
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&stg_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&stg_empty[s]), 4);
    }
    ptx::mbar_init(ptx::smem_u32(l_ready), 8);
    for (int s = 0; s < 8; ++s) ptx::mbar_init(ptx::smem_u32(&xbar[s]), 2);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (tt * group < kVarBlk) {
    for (int s = 0; s < 2; ++s) zero_tile_rows(sQ + s * kTile, Sh::kChunks, tt * group);
    ptx::fence_proxy_async_smem();
  }
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&tmQ);
    ptx::prefetch_tmap(&tmK);
    ptx::prefetch_tmap(&tmV);
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_holder), kAttnTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  WaitCtl ctl{abort_flag, a.err, a.timeout_ns, kKidVarAttn};
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();  // the list; all of the above overlaps its construction
  const int n_items = *a.count * a.kv_heads;  // (entry, kv head), heads innermost
  const int cta = blockIdx.x, grid = gridDim.x;
  // Item k of this CTA; false behind the list's end.
  auto item_at = [&](int k, VarItem& it, int& hkv) -> bool {
    const int i = zigzag(k, cta, grid, n_items);
    if (i < 0) return false;
    const int e = i / a.kv_heads;
    hkv = i - e * a.kv_heads;
    const int4* p = reinterpret_cast<const int4*>(a.items + e);
    const int4 x = __ldg(p), y = __ldg(p + 1);
    it = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    return true;
  };
  // Keys of the sequence in the item's last block: below 128 its V tile holds foreign rows.
  auto tail_rows = [](const VarItem& it) { return it.kv_len - (it.b1 - 1) * kVarBlk; };
  // e4m3: the first block that may be the last one that some row sees keys of: that of the first token's own key, or the item's
  // last. The blocks before it are seen whole by every row that sees any key.
  auto first_edge = [](const VarItem& it) { return min(it.pos0 >> 7, it.b1 - 1); };

  static_assert(kAttnThreads == 512, "register split assumes 16 warps");
  if (warp < 4) ptx::setmaxnreg_dec<kAttnRegsLow>();
  if (warp >= 12) ptx::setmaxnreg_dec<kAttnRegsOut>();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    // Packed: one thread. Paged: lane i copies the block's box i (a page, or 128 rows of a larger one); its table entry is
    // read a block ahead, so the lookups cost neither latency nor a thread's turn per box (16 unrolled boxes in one thread
    // took 4.4 us a block).
    uint32_t slot = 0, slot_phase = 0, q_issued = 0, kv_issued = 0;
    bool ok = true;
    constexpr int kRing = kE4m3 ? kStages : kSlots;  // the ring that copies go to
    uint64_t* ring_full = kE4m3 ? stg_full : kv_full;
    uint64_t* ring_empty = kE4m3 ? stg_empty : kv_empty;
    const uint32_t kv0 = ptx::smem_u32(kE4m3 ? sRaw : sKV);
    if (kPaged || lane == 0) {
      const int page_rows = kPaged ? 1 << a.page_shift : 0;
      const int box_rows = kPaged ? min(page_rows, kVarBlk) : kVarBlk;
      const int pages_per_blk = kVarBlk / box_rows;
      auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t site) -> bool {
        return kPaged ? warp_wait_bounded<false, 512>(ptx::smem_u32(bar), parity, ctl, site)
                      : wait_bounded<false, 512>(ptx::smem_u32(bar), parity, ctl, site);
      };
      // Paged: this lane's table entry of key block b (-1: no box), and the first cache row it stands for; rows behind the
      // cache (a bad page) read as zeros, boxes wholly behind the sequence's end are not copied.
      auto entry = [&](const VarItem& it, int b) -> int {
        const int key = b * kVarBlk + lane * box_rows;
        return lane < pages_per_blk && key < it.kv_len ? __ldg(a.table + it.src * a.table_stride + (key >> a.page_shift)) : 0;
      };
      auto row_of = [&](const VarItem& it, int b, int page) -> int {
        const int key = b * kVarBlk + lane * box_rows;
        if (lane >= pages_per_blk || key >= it.kv_len) return -1;
        if (page < 0 || page >= a.num_pages) {
          atomicCAS(a.err, 0u, kErrBounds | (kKidVarAttn << 8) | (3u << 16));
          return a.num_pages << a.page_shift;
        }
        return (page << a.page_shift) + (key & (page_rows - 1));
      };
      auto push = [&](const CUtensorMap* m, const VarItem& it, int hkv, int b, bool is_v, int row) -> bool {
        if (!wait(&ring_empty[slot], slot_phase ^ 1, 2)) return false;
        const bool foreign = !kE4m3 && is_v && b == it.b1 - 1 && tail_rows(it) < kVarBlk;
        const uint32_t fb = ptx::smem_u32(foreign ? &raw_full[slot] : &ring_full[slot]);
        uint32_t dst = kv0 + slot * (kE4m3 ? Sh::kStageBytes : kTile);
        if (kPaged) dst += lane * (kE4m3 ? box_rows * kD : (box_rows >> 3) * kGroupPitch);
        if (lane == 0) {
          const int boxes = kPaged ? min(pages_per_blk, (it.kv_len - b * kVarBlk + box_rows - 1) / box_rows) : 1;
          ptx::mbar_arrive_expect_tx(fb, boxes * box_rows * kD * (kE4m3 ? 1 : 2));
        }
        if constexpr (kE4m3) {
          __syncwarp();
          if (row >= 0) ptx::tma_load_3d(dst, m, fb, 0, hkv, row);
        } else if constexpr (kPaged) {
          __syncwarp();
          if (row >= 0) ptx::tma_load_5d(dst, m, fb, 0, 0, 0, row >> 3, hkv);
        } else {
#pragma unroll
          for (int c = 0; c < Sh::kChunks; ++c) ptx::tma_load_3d(dst + c * kAttnChunk, m, fb, 64 * c, hkv, row);
        }
        ++kv_issued;
        if (++slot == kRing) { slot = 0; slot_phase ^= 1; }
        return true;
      };
      VarItem it;
      int hkv;
      for (int k = 0; ok && item_at(k, it, hkv); ++k) {
        if (it.b1 <= it.b0) continue;
        int ahead = 0;
        if constexpr (kPaged) ahead = entry(it, it.b0);
        const uint32_t qbuf = q_issued & 1;
        ok = wait(&q_empty[qbuf], ((q_issued >> 1) & 1) ^ 1, 1);
        if (!ok) break;
        if (lane == 0) {
          const uint32_t qf = ptx::smem_u32(kE4m3 ? &q_raw[qbuf] : &q_full[qbuf]);
          ptx::mbar_arrive_expect_tx(qf, tt * group * kD * 2);
#pragma unroll
          for (int c = 0; c < Sh::kChunks; ++c)
            ptx::tma_load_3d(ptx::smem_u32(sQ) + qbuf * kTile + c * kAttnChunk, &tmQ, qf, 64 * c, hkv * group, it.row0);
        }
        ++q_issued;
        int row = 0, prev = 0;
        for (int b = it.b0; b < it.b1 && ok; ++b) {
          if constexpr (kPaged) {
            row = row_of(it, b, ahead);
            if (b + 1 < it.b1) ahead = entry(it, b + 1);
          } else {
            row = it.src + b * kVarBlk;
          }
          ok = push(&tmK, it, hkv, b, false, row);
          if (ok && b > it.b0) ok = push(&tmV, it, hkv, b - 1, true, prev);
          prev = row;
        }
        if (ok) ok = push(&tmV, it, hkv, it.b1 - 1, true, prev);
      }
    }
    if (lane == 0) {  // drain loads still in flight
      WaitCtl dctl = ctl;
      volatile int never = 0;
      dctl.abort = &never;
      for (uint32_t i = q_issued > 2 ? q_issued - 2 : 0; i < q_issued; ++i)
        wait_bounded(ptx::smem_u32(kE4m3 ? &q_raw[i & 1] : &q_full[i & 1]), (i >> 1) & 1, dctl, 8);
      const uint32_t first = kv_issued > kRing ? kv_issued - kRing : 0;
      for (uint32_t i = first; i < kv_issued; ++i)
        wait_bounded(ptx::smem_u32(&ring_full[i % kRing]), (i / kRing) & 1, dctl, 8);
    }
    __syncwarp();
  } else if (warp == 1 || warp == 2) {
    // ------------------------------------------------------------------ MMA issuers (one thread each)
    if (lane == 0) {
      const bool s_role = warp == 1;
      uint32_t g = 0, rows = 0, seq = 0;  // blocks, items and ring positions passed
      bool ok = true;
      const uint32_t kv0 = ptx::smem_u32(sKV);
      const uint64_t qdesc0 = ptx::smem_desc(ptx::smem_u32(sQ), 16, 1024);
      const uint64_t kdesc0 = ptx::smem_desc(kv0, 16, kGroupPitch);           // K: K-major
      const uint64_t vdesc0 = ptx::smem_desc(kv0, kChunkPitch, kGroupPitch);  // V: MN-major
      VarItem it;
      int hkv;
      for (int k = 0; ok && item_at(k, it, hkv); ++k) {
        const int n = it.b1 - it.b0;
        if (n <= 0) continue;
        const uint32_t qbuf = rows & 1;
        if (s_role) {
          ok = wait_bounded(ptx::smem_u32(&q_full[qbuf]), (rows >> 1) & 1, ctl, 14);
          if (!ok) break;
        }
        for (int j = 0; j < n && ok; ++j, ++g) {
          const uint32_t b = g & 1;
          if (s_role) {
            if (g >= 2) {  // PV_{g-2} read P from this buffer
              ok = wait_bounded(ptx::smem_u32(&s_free[b]), ((g - 2) >> 1) & 1, ctl, 11);
              if (!ok) break;
            }
            const uint32_t pos = seq + attn_k_pos(j);
            const uint32_t sl = pos % kSlots;
            ok = wait_bounded(ptx::smem_u32(&kv_full[sl]), (pos / kSlots) & 1, ctl, 12);
            if (!ok) break;
            ptx::tc_fence_after();
            const uint64_t qd = qdesc0 + ((qbuf * kTile) >> 4), kd = kdesc0 + ((sl * kTile) >> 4);
#pragma unroll(kE4m3 ? 1 : kD / 16)
            for (int x = 0; x < kD / 16; ++x) {
              const uint32_t qo = ((x >> 2) * kAttnChunk + (x & 3) * 32) >> 4, ko = ((x >> 2) * kChunkPitch + (x & 3) * 32) >> 4;
              ptx::mma_f16_ss(tmem_base + 128 * b, qd + qo, kd + ko, IDESC_S, x != 0);
            }
            ptx::mma_commit(ptx::smem_u32(&kv_empty[sl]));
            ptx::mma_commit(ptx::smem_u32(&s_full[b]));
            if (j == n - 1) ptx::mma_commit(ptx::smem_u32(&q_empty[qbuf]));
          } else {
            if (j == 0 && rows > 1) {  // the first PV of an item overwrites O buffer rows % 2
              ok = wait_bounded(ptx::smem_u32(&o_free[rows & 1]), ((rows >> 1) - 1) & 1, ctl, 17);
              if (!ok) break;
            }
            ok = wait_bounded(ptx::smem_u32(&p_full[b]), (g >> 1) & 1, ctl, 13);
            if (!ok) break;
            const uint32_t pos = seq + attn_v_pos(j, n);
            const uint32_t sl = pos % kSlots;
            ok = wait_bounded(ptx::smem_u32(&kv_full[sl]), (pos / kSlots) & 1, ctl, 15);
            if (!ok) break;
            ptx::tc_fence_after();
            const uint64_t vd = vdesc0 + ((sl * kTile) >> 4);
            const uint32_t t_o = tmem_base + kAttnTmemO + 128 * (rows & 1), t_p = tmem_base + 128 * b;
#pragma unroll(kE4m3 ? 1 : 8)
            for (int x = 0; x < 8; ++x)  // K step x: keys [16x, 16x+16) in P columns 8x (+32 for the second half)
              ptx::mma_f16_ts(t_o, t_p + 8 * x + (x >= 4 ? 32 : 0), vd + ((2 * x * kGroupPitch) >> 4), IDESC_PV,
                              (j == 0 && x == 0) ? 0u : 1u);
            ptx::mma_commit(ptx::smem_u32(&kv_empty[sl]));
            ptx::mma_commit(ptx::smem_u32(&s_free[b]));
            if (j == n - 1) ptx::mma_commit(ptx::smem_u32(&o_done[rows & 1]));
          }
        }
        seq += 2 * n;
        ++rows;
      }
      const uint32_t dr = ptx::smem_u32(&drain[s_role ? 0 : 1]);
      ptx::mma_commit(dr);
      WaitCtl dctl = ctl;
      volatile int never = 0;
      dctl.abort = &never;
      wait_bounded(dr, 0, dctl, 16);
    }
    __syncwarp();
  } else if (warp == 3) {
    // ------------------------------------------------------------------ foreign V rows -> zero; e4m3: scales
    uint32_t seq = 0, phases = 0;  // ring positions passed; bit s: parity of raw_full[s]'s next completion
    bool ok = true;
    VarItem it;
    int hkv;
    if constexpr (kE4m3) {
      // Lane l has keys l, l + 32, l + 64, l + 96 of a block. Pages are looked up two blocks ahead of their scales' use and
      // scales one, so neither load is waited for; behind the sequence, and on a bad page, a scale is 0.
      uint32_t g = 0;
      for (int k = 0; ok && item_at(k, it, hkv); ++k) {
        if (it.b1 <= it.b0) continue;
        int page[4] = {-1, -1, -1, -1};
        float ks[4] = {}, vs[4] = {};
        auto look_pages = [&](int b) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int key = b * kVarBlk + 32 * x + lane;
            page[x] = b < it.b1 && key < it.kv_len ? __ldg(a.table + it.src * a.table_stride + (key >> a.page_shift)) : -1;
          }
        };
        auto look_scales = [&](int b) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int key = b * kVarBlk + 32 * x + lane;
            const bool held = page[x] >= 0 && page[x] < a.num_pages;
            const int64_t at =
                static_cast<int64_t>(held ? (page[x] << a.page_shift) + (key & ((1 << a.page_shift) - 1)) : 0) * a.kv_heads + hkv;
            ks[x] = held ? __ldg(a.k_scale + at) : 0.0f;
            vs[x] = held ? __ldg(a.v_scale + at) : 0.0f;
          }
        };
        int r_exp = kScaleLow;  // the tile's largest value scale so far: a scale divided by 2^(r_exp - 133) is below 2^7
        for (int b = it.b0 - 2; b < it.b1; ++b) {  // (two rounds of lookups before the first block)
          if (b >= it.b0) {
            const uint32_t buf = g & 1;
            if (g >= 2) {  // the softmax of block g - 2 has read this buffer
              ok = warp_wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(&p_full[buf]), ((g - 2) >> 1) & 1, ctl, 34);
              if (!ok) break;
            }
            ++g;
            int top[4], before = r_exp;  // exponents (a scale that is not finite counts as none)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int e = static_cast<int>(__float_as_uint(vs[x]) >> 23) & 255;
              top[x] = e == 255 ? kScaleLow : min(max(e, kScaleLow), kScaleHigh);
            }
            int most[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) most[x] = __reduce_max_sync(0xffffffffu, top[x]);
            if (b >= first_edge(it)) {  // some row may not see all of the block: the largest up to each key
#pragma unroll 1
              for (int o = 1; o < 32; o <<= 1)
#pragma unroll
                for (int x = 0; x < 4; ++x) top[x] = max(top[x], __shfl_up_sync(0xffffffffu, top[x], o));  // (lowest lanes: own)
              int first = r_exp;
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                v_top[128 * buf + 32 * x + lane] = max(top[x], first);
                first = max(first, most[x]);
              }
            }
            r_exp = max(r_exp, max(max(most[0], most[1]), max(most[2], most[3])));
            const float down = __int_as_float((260 - r_exp) << 23);  // 2^(133 - r_exp)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              k_sc[128 * buf + 32 * x + lane] = ks[x];
              v_sc[128 * buf + 32 * x + lane] = vs[x] * down;
            }
            if (lane == 0) {
              r_tile[buf] = r_exp;
              r_before[buf] = before;
              r_step[buf] = __int_as_float(max(127 + before - r_exp, 0) << 23);
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sc_full[buf]));
          }
          if (b + 1 >= it.b0) look_scales(b + 1);
          look_pages(b + 2);
        }
      }
    }
    for (int k = 0; !kE4m3 && ok && item_at(k, it, hkv); ++k) {
      const int n = it.b1 - it.b0;
      if (n <= 0) continue;
      const int live = tail_rows(it);
      if (live < kVarBlk) {
        const uint32_t sl = (seq + 2 * n - 1) % kSlots;  // the item's last V tile
        ok = warp_wait_bounded<false, 256>(ptx::smem_u32(&raw_full[sl]), (phases >> sl) & 1, ctl, 30);
        if (!ok) break;
        phases ^= 1u << sl;
        uint8_t* tile = sKV + sl * kTile;
        constexpr int kPer = Sh::kChunks * 8;  // 16-byte pieces per row (a row's swizzle stays within its 128 bytes)
        for (int i = lane; i < (kVarBlk - live) * kPer; i += 32) {
          const int r = live + i / kPer, c = i % kPer;
          *reinterpret_cast<uint4*>(tile + (r >> 3) * kGroupPitch + (c >> 3) * kChunkPitch + (r & 7) * 128 + (c & 7) * 16) =
              make_uint4(0, 0, 0, 0);
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&kv_full[sl]));
      }
      seq += 2 * n;
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------------ softmax (warps 4..11)
    ptx::setmaxnreg_inc<kAttnRegsHigh>();
    const int h = (warp - 4) >> 2;  // key half: S columns [64 h, 64 h + 64)
    const int q = warp & 3;         // TMEM lane quarter
    const int r = 32 * q + lane;    // row of the tile == TMEM lane
    const int tok = r / group, hd = r - tok * group;  // its token and head
    const uint32_t lane_off = static_cast<uint32_t>(32 * q) << 16;
    const uint32_t tO0 = tmem_base + kAttnTmemO + lane_off + h * kHalfD;
    float c = a.scale_log2;
    uint32_t g = 0, rows = 0, x_cnt = 0;
    bool ok = true;
    // Exchange with the warp of the other key half through the last column of each half of the S buffer.
    auto exchange = [&](uint32_t tSb, float v, float& other) -> bool {
      const uint32_t slot = x_cnt & 1;
      ptx::tmem_st_32x32b_x1(tSb + 64 * h + 63, __float_as_uint(v));
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      const uint32_t xb = ptx::smem_u32(&xbar[q * 2 + slot]);
      if (lane == 0) ptx::mbar_arrive(xb);
      if (!warp_wait_bounded(xb, (x_cnt >> 1) & 1, ctl, 23)) return false;
      ++x_cnt;
      ptx::tc_fence_after();
      other = __uint_as_float(ptx::tmem_ld_32x32b_x1(tSb + 64 * (h ^ 1) + 63));
      ptx::tmem_wait_ld();
      return true;
    };
    VarItem next;
    int next_h = 0;
    bool more = item_at(0, next, next_h);
    for (int k = 0; more && ok; ++k) {
      const VarItem it = next;
      const int hkv = next_h;
      more = item_at(k + 1, next, next_h);  // looked up one item ahead
      const int n = it.b1 - it.b0;
      if (n <= 0) {
        if (tok < it.ntok) {
          const int64_t grow = static_cast<int64_t>(it.row0 + tok) * a.heads + hkv * group + hd;
          uint4* orow = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.O) + grow * kD + h * kHalfD);
          const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int cc = 0; cc < kHalfD / 8; ++cc) orow[cc] = z;
          if (a.lse && h == 0) a.lse[grow] = -INFINITY;
        }
        continue;
      }
      // keys at or behind `limit` are masked for this row; `clear`: key blocks below it are seen by every row of the tile
      const int limit = a.causal ? it.pos0 + tok + 1 : it.kv_len;
      const int clear = (a.causal ? it.pos0 + 1 : it.kv_len) >> 7;
      float m_run = -INFINITY, l_run = 0.0f;
      const uint32_t tO = tO0 + 128 * (rows & 1);
      for (int j = 0; j < n; ++j, ++g) {
        const int kb = it.b0 + j;
        const uint32_t b = g & 1;
        const uint32_t tS = tmem_base + 128 * b + lane_off;
        if constexpr (kE4m3) {
          ok = warp_wait_bounded(ptx::smem_u32(&sc_full[b]), (g >> 1) & 1, ctl, 19);
          if (!ok) break;
          if (j == 0) {  // the rows' scales come with the converted queries
            ok = warp_wait_bounded(ptx::smem_u32(&q_full[rows & 1]), (rows >> 1) & 1, ctl, 18);
            if (!ok) break;
            c = a.scale_log2 * q_sc[(rows & 1) * 128 + r];
          }
        }
        ok = warp_wait_bounded(ptx::smem_u32(&s_full[b]), (g >> 1) & 1, ctl, 20);
        if (!ok) break;
        ptx::tc_fence_after();
        uint32_t sv[64];
        ptx::tmem_ld_32x32b_x32(tS + 64 * h, *reinterpret_cast<uint32_t(*)[32]>(&sv[0]));
        ptx::tmem_ld_32x32b_x32(tS + 64 * h + 32, *reinterpret_cast<uint32_t(*)[32]>(&sv[32]));
        ptx::tmem_wait_ld();
        float* v = reinterpret_cast<float*>(sv);
        if constexpr (kE4m3) {
          const float4* ks = reinterpret_cast<const float4*>(k_sc + 128 * b + 64 * h);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float4 x = ks[i];
            f2_unpack(f2_mul(f2_pack(v[4 * i], v[4 * i + 1]), f2_pack(x.x, x.y)), v[4 * i], v[4 * i + 1]);
            f2_unpack(f2_mul(f2_pack(v[4 * i + 2], v[4 * i + 3]), f2_pack(x.z, x.w)), v[4 * i + 2], v[4 * i + 3]);
          }
        }
        if (kb >= clear) {
          const int lim = limit - (kb * kVarBlk + 64 * h);
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i >= lim) v[i] = -INFINITY;
        }
        float pm[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) pm[x] = v[x];
#pragma unroll
        for (int i = 8; i < 64; i += 16)
#pragma unroll
          for (int x = 0; x < 8; ++x)
            pm[x] = i + 8 < 64 ? max3_nan(pm[x], v[i + x], v[(i + 8 + x) & 63]) : max_nan(pm[x], v[i + x]);
        const float mh = max3_nan(max3_nan(pm[0], pm[1], pm[2]), max3_nan(pm[3], pm[4], pm[5]), max_nan(pm[6], pm[7]));
        float mo;
        ok = exchange(tS, mh, mo);
        if (!ok) break;
        const float mbs = max_nan(mh, mo) * c;
        const bool move = !(mbs <= m_run + 8.0f);  // the reference maximum lags by at most 8: P <= 2^8; a NaN moves it
        float alpha = 1.0f;
        if (move) alpha = (m_run == -INFINITY) ? 0.0f : ex2_approx(m_run - mbs);
        if (move) m_run = max_nan(m_run, mbs);  // (a NaN stays, also through blocks that this row does not see)
        float step = 1.0f, lift = 0.0f;  // O follows the scale reference
        // The row's scale reference where it is not the tile's: a row that sees part of the block has seen all before it. How far
        // (log2) the tile's lies above the row's, and, with the row's last key in the block, the row's closing factor.
        const bool edge = kE4m3 && kb >= first_edge(it);
        auto reference = [&]() -> int {
          const int seen = limit - kb * kVarBlk;
          return seen > 0 ? max(v_top[128 * b + min(seen, kVarBlk) - 1], r_tile[b] - kScaleSpan) : r_tile[b];
        };
        if constexpr (kE4m3) {
          step = r_step[b];
          if (edge) {
            const int own = reference(), tile = r_tile[b];
            lift = static_cast<float>(tile - own);
            step = 1.0f;
            if (limit > kb * kVarBlk) {  // (a row that sees none of the block keeps its O and its closing factor)
              step = __int_as_float(max(127 + r_before[b] - own, 0) << 23);
              if (h == 0) r_end[128 * (rows & 1) + r] = __int_as_float((own - 6) << 23);  // 2^(own - 133)
            }
          }
        }
        const bool need_rescale = __any_sync(0xffffffffu, (move || step != 1.0f) && j > 0);
        const float m_sub = (m_run == -INFINITY) ? 0.0f : m_run;
        const uint64_t c2 = f2_pack(c, c), nm2 = f2_pack(lift - m_sub, lift - m_sub);
        uint64_t acc[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          float t0, t1, e0, e1;
          f2_unpack(f2_fma(f2_pack(v[i], v[i + 1]), c2, nm2), t0, t1);
          if (((i >> 1) & 7) >= 8 - kAttnPolyEighths) {
            ex2_poly2<kVarFloor>(t0, t1, e0, e1);
          } else {
            e0 = ex2_approx(t0);
            e1 = ex2_approx(t1);
          }
          acc[(i >> 1) & 3] = f2_add(acc[(i >> 1) & 3], f2_pack(e0, e1));
          if constexpr (kE4m3) {
            const float2 x = *reinterpret_cast<const float2*>(v_sc + 128 * b + 64 * h + i);
            f2_unpack(f2_mul(f2_pack(e0, e1), f2_pack(x.x, x.y)), e0, e1);
          }
          sv[i >> 1] = pack2<kOpF16>(e0, e1);
        }
        float rs;
        {
          const uint64_t a01 = f2_add(acc[0], acc[1]), a23 = f2_add(acc[2], acc[3]);
          float lo, hi;
          f2_unpack(f2_add(a01, a23), lo, hi);
          rs = lo + hi;
        }
        if constexpr (kE4m3)
          if (edge) rs *= __int_as_float((127 - (r_tile[b] - reference())) << 23);
        l_run = l_run * alpha + rs;
        if (need_rescale) {
          ok = warp_wait_bounded(ptx::smem_u32(&s_free[(g - 1) & 1]), ((g - 1) >> 1) & 1, ctl, 21);
          if (!ok) break;
          ptx::tc_fence_after();
          const float al = (move ? alpha : 1.0f) * step;
#pragma unroll 1
          for (int cc = 0; cc < kHalfD / 32; ++cc) {
            uint32_t u[32];
            ptx::tmem_ld_32x32b_x32(tO + cc * 32, u);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * al);
            ptx::tmem_st_32x32b_x32(tO + cc * 32, u);
          }
        }
        ptx::tmem_st_32x32b_x32(tS + 64 * h, *reinterpret_cast<uint32_t(*)[32]>(&sv[0]));
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&p_full[b]));
      }
      if (!ok) break;
      if (rows > 0) {  // the output warps have read the previous item's sums
        ok = warp_wait_bounded(ptx::smem_u32(&o_free[(rows - 1) & 1]), ((rows - 1) >> 1) & 1, ctl, 24);
        if (!ok) break;
      }
      l_part[h * 128 + r] = l_run;
      if (h == 0) m_row[r] = m_run;
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(l_ready));
      ++rows;
    }
  } else {
    // ------------------------------------------------------------------ output, conversion (warps 12..15)
    const int q = warp & 3;
    const int r = 32 * q + lane;
    const int tok = r / group, hd = r - tok * group;
    const uint32_t tO0 = tmem_base + kAttnTmemO + (static_cast<uint32_t>(32 * q) << 16);
    const bool o_v8 = (reinterpret_cast<uintptr_t>(a.O) & 31) == 0;
    uint32_t rows = 0;
    bool ok = true;
    // e4m3: this thread converts row r of every tile. Ring positions passed (codes and fp16 tiles alike):
    uint32_t pos = 0;
    VarItem it;
    int hkv;
    for (int k = 0; ok && item_at(k, it, hkv); ++k) {
      if (it.b1 <= it.b0) continue;  // written by the softmax warps
      if constexpr (kE4m3) {
        // queries: row r in place, bf16 -> fp16 with its largest element brought to [2^15, 2^16)
        const uint32_t qbuf = rows & 1;
        ok = warp_wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(&q_raw[qbuf]), (rows >> 1) & 1, ctl, 31);
        if (!ok) break;
        float up = 1.0f;
        if constexpr (!kF16) {
          uint8_t* row = sQ + qbuf * kTile + r * 128;
          uint32_t top = 0;
          // (loops, not unrolled: the CTA's roles share the instruction cache, which the unrolled kernel overran -- a third of
          // its time)
#pragma unroll 1
          for (int x = 0; x < kD / 8; ++x) {
            const uint4 w = *reinterpret_cast<const uint4*>(row + (x >> 3) * kAttnChunk + (x & 7) * 16);
            top = __vmaxu2(__vmaxu2(top, __vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu)),
                           __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
          }
          top = max(top >> 16, top & 0xffffu);
          const int e = max(static_cast<int>(top >> 7), 40) - 142;
          const float down = __int_as_float((127 - e) << 23);
          up = __int_as_float((127 + e) << 23);
          auto turn = [&](uint32_t u) {
            const float2 f = unpack2<false>(u);
            return pack_f16(f.x * down, f.y * down);
          };
#pragma unroll 1
          for (int x = 0; x < kD / 8; ++x) {
            uint4* at = reinterpret_cast<uint4*>(row + (x >> 3) * kAttnChunk + (x & 7) * 16);
            const uint4 w = *at;
            *at = make_uint4(turn(w.x), turn(w.y), turn(w.z), turn(w.w));
          }
          ptx::fence_proxy_async_smem();
        }
        q_sc[qbuf * 128 + r] = up;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&q_full[qbuf]));
        // One code tile -> fp16 tile: row r, 16 codes (16 bytes) at a time; both sides' 16-byte chunks are swizzled. Rows
        // behind the sequence are zero.
        const int tiles = 2 * (it.b1 - it.b0);
        for (int x = 0; x < tiles; ++x, ++pos) {  // K_0, K_1, V_0, K_2, V_1, .., V_last
          const int b = it.b0 + (x == 0 ? 0 : x == tiles - 1 ? tiles / 2 - 1 : (x & 1) ? (x + 1) / 2 : x / 2 - 1);
          const uint32_t st = pos % kStages, sl = pos % kSlots;
          ok = warp_wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(&stg_full[st]), (pos / kStages) & 1, ctl, 32);
          if (ok) ok = warp_wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(&kv_empty[sl]), ((pos / kSlots) & 1) ^ 1, ctl, 33);
          if (!ok) break;
          const uint32_t live = b * kVarBlk + r < it.kv_len ? 0xffffffffu : 0u;
          const uint8_t* src = sRaw + st * Sh::kStageBytes + r * kD;
          uint8_t* dst = sKV + sl * kTile + r * 128;
          const int sx = kD == 128 ? r & 7 : (r >> 1) & 3;
#pragma unroll 1
          for (int y = 0; y < kD / 16; y += 4) {  // a 64-column chunk: loads, then conversions
            uint4 w[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) w[z] = *reinterpret_cast<const uint4*>(src + (((y + z) ^ sx) << 4));
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const uint32_t u[4] = {w[z].x & live, w[z].y & live, w[z].z & live, w[z].w & live};
              uint8_t* d = dst + (y >> 2) * kAttnChunk;
              uint32_t f[8];
#pragma unroll
              for (int i = 0; i < 4; ++i) e4m3x4(u[i], f[2 * i], f[2 * i + 1]);
              *reinterpret_cast<uint4*>(d + (((2 * z) ^ (r & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
              *reinterpret_cast<uint4*>(d + (((2 * z + 1) ^ (r & 7)) << 4)) = make_uint4(f[4], f[5], f[6], f[7]);
            }
          }
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            ptx::mbar_arrive(ptx::smem_u32(&stg_empty[st]));
            ptx::mbar_arrive(ptx::smem_u32(&kv_full[sl]));
          }
        }
        if (!ok) break;
      }
      ok = warp_wait_bounded<false, 256>(ptx::smem_u32(l_ready), rows & 1, ctl, 25);
      if (ok) ok = warp_wait_bounded<false, 256>(ptx::smem_u32(&o_done[rows & 1]), (rows >> 1) & 1, ctl, 22);
      if (!ok) break;
      const uint32_t ob = rows & 1, tO = tO0 + 128 * ob;
      ++rows;
      ptx::tc_fence_after();
      const float m_run = m_row[r];
      const float l_tot = l_part[r] + l_part[128 + r];
      const bool live = tok < it.ntok;
      const int64_t grow = static_cast<int64_t>(it.row0 + tok) * a.heads + hkv * group + hd;
      // A row without keys has its maximum at -inf: zero. A maximum
      // of +inf (scores beyond fp32) gives NaN, as the definition does.
      const bool none = m_run == -INFINITY;
      float inv_l = m_run == INFINITY ? NAN : 1.0f / l_tot;
      if constexpr (kE4m3) inv_l *= r_end[128 * ob + r];
      if constexpr (kPaged) {
        if (it.part >= 0) {  // one of several pieces: fp32 rows and their log2 sums, for the combining kernel
          const int64_t prow = (static_cast<int64_t>(it.part) * a.kv_heads + hkv) * kVarBlk + r;
          a.part_lse[prow] = none ? -INFINITY : m_run + log2f(l_tot);
#pragma unroll 1
          for (int cc = 0; cc < kD / 32; ++cc) {
            uint32_t u[32];
            ptx::tmem_ld_32x32b_x32(tO + cc * 32, u);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] = none ? 0u : __float_as_uint(__uint_as_float(u[i]) * inv_l);
#pragma unroll
            for (int i = 0; i < 32; i += 8) st_global_v8(a.part_o + prow * kD + cc * 32 + i, u + i);
          }
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&o_free[ob]));
          continue;
        }
      }
      if (live && a.lse) a.lse[grow] = none ? -INFINITY : (m_run + log2f(l_tot)) * 0.6931471805599453f;
      uint16_t* orow = static_cast<uint16_t*>(a.O) + grow * kD;
#pragma unroll 1
      for (int cc = 0; cc < kD / 32; ++cc) {
        uint32_t u[32];
        ptx::tmem_ld_32x32b_x32(tO + cc * 32, u);
        ptx::tmem_wait_ld();
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          pk[i] = none ? 0u : pack2<kF16>(__uint_as_float(u[2 * i]) * inv_l, __uint_as_float(u[2 * i + 1]) * inv_l);
        if (live && o_v8) {
          st_global_v8(orow + cc * 32, pk);
          st_global_v8(orow + cc * 32 + 16, pk + 8);
        } else if (live) {
          uint4* dst = reinterpret_cast<uint4*>(orow + cc * 32);
#pragma unroll
          for (int gg = 0; gg < 4; ++gg) dst[gg] = make_uint4(pk[4 * gg], pk[4 * gg + 1], pk[4 * gg + 2], pk[4 * gg + 3]);
        }
        __syncwarp();
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&o_free[ob]));
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc(tmem_base, kAttnTmemCols);
}

// Pieces of split entries -> rows: with piece i's log2 sum L_i and its rows O_i,  O = sum_i 2^(L_i - max L) O_i / sum_i
// 2^(L_i - max L). Block (split entry, kv head, 16 rows), D / 4 threads per row. Reads each partial result once, from L2.
struct VarCombineArgs {
  void* O;
  const float* part_o;
  const float* part_lse;
  const VarSplit* splits;
  const int* count;  // [1]: split entries
  int heads, kv_heads, group;
};
constexpr int kCombineRows = 16;

template <bool kF16, int kD>
__global__ void __launch_bounds__(kCombineRows * kD / 4) varattn_combine_kernel(const VarCombineArgs a) {
  ptx::grid_dependency_wait();
  if (static_cast<int>(blockIdx.x) >= a.count[1]) return;
  const VarSplit sp = a.splits[blockIdx.x];
  const int hkv = blockIdx.y, r = blockIdx.z * kCombineRows + threadIdx.x / (kD / 4), c = threadIdx.x % (kD / 4);
  const int tok = r / a.group, hd = r - tok * a.group;
  if (tok >= sp.ntok) return;
  const int64_t row = (static_cast<int64_t>(sp.first) * a.kv_heads + hkv) * kVarBlk + r, step = static_cast<int64_t>(a.kv_heads) * kVarBlk;
  float top = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < sp.n; ++i) top = max_nan(top, __ldg(a.part_lse + row + i * step));
  const float sub = top == -INFINITY ? 0.0f : top;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float sum = 0.0f;
#pragma unroll 4
  for (int i = 0; i < sp.n; ++i) {
    const float w = ex2_approx(__ldg(a.part_lse + row + i * step) - sub);
    const float4 v = __ldg(reinterpret_cast<const float4*>(a.part_o + (row + i * step) * kD) + c);
    sum += w;
    acc.x += v.x * w;
    acc.y += v.y * w;
    acc.z += v.z * w;
    acc.w += v.w * w;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no piece has a key: zero
  const int64_t grow = static_cast<int64_t>(sp.row0 + tok) * a.heads + hkv * a.group + hd;
  reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.O) + grow * kD)[c] =
      make_uint2(pack2<kF16>(acc.x * inv, acc.y * inv), pack2<kF16>(acc.z * inv, acc.w * inv));
}

}  // namespace bsk
