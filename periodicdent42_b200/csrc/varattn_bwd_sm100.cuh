// Attention over packed sequences, backward, for sm_100a (tcgen05 + TMA), deterministic (no atomics).
//
// Given Q, dO [tokens, heads, D], K, V [tokens, kv_heads, D], O and the forward's log-sum-exp per query row:
//   Delta_i = sum_d dO[i,d] O[i,d]                                      (varattn_bwd_prep_kernel)
//   P = exp(scale * Q K^T - LSE), dP = dO V^T, dS = P * (dP - Delta)    (recomputed per block pair)
//   dV = P^T dO, dK = scale * dS^T Q                                    (varattn_bwd_dkdv_kernel, per key block)
//   dQ = scale * dS K                                                   (varattn_bwd_dq_kernel, per query tile)
// Query rows are the packed (token, head of the group) rows of the forward's tiles (varattn_plan.cuh), so dK and dV are
// summed over the group's heads inside the tensor core's accumulation, in fp32 and in a fixed order.
//
// The CTA's shape is that of the block-sparse backward (bsattn_bwd_sm100.cuh, where it is explained and measured): warp 0
// TMA producer, warp 1 MMA issuer, warps 4-11 two warpgroups that each take 64 columns of the 128 x 128 score tiles, P kept
// in fp32 registers between its use for dV and for dS; P^T and dS^T / dS are rounded to the inputs' type for the second
// products (half a step: 2^-8 of a weight in bf16, 2^-11 in fp16, as the results' own rounding; gradients come out
// 1.5 times as far from the 64-bit ones, normwise, as results rounded once; with windows of a few keys up to 1.8 times, since
// Delta takes the rounded O and fewer keys' dS average that out). What differs:
//   - masks go by position: keys behind a row (causal) or behind the sequence's end get P = 0;
//   - rows of a tile that are not the sequence's own (behind its end, or the 128 mod group rows that no copy fills) would
//     enter the sums as 0 x their value, so warp 2 sets them to zero in shared memory between the copy's arrival and the
//     products: Q and dO rows for dK / dV, K and V rows for dQ. Only a sequence's last tile takes this detour.
//   - row statistics lie per tile as 128 offsets -LSE log2(e) and 128 Deltas (padded rows: -inf and 0), so that one bulk copy
//     brings a tile's.
#pragma once

#include "bsattn_bwd_sm100.cuh"
#include "varattn_sm100.cuh"

namespace bsk {

constexpr uint32_t kKidVarAttnBwd = 12;

struct VarBwdArgs {
  const float* stats;    // [tile slots][kv heads][256]: -LSE * log2(e) [128], Delta [128]
  void* dQ;              // contiguous [tokens, heads, D]
  void* dK;              // contiguous [tokens, kv heads, D]
  void* dV;
  const VarItem* q_items;  // query tiles
  const VarItem* k_items;  // key blocks
  const int* q_count;
  const int* k_count;
  int heads, kv_heads, group, causal;
  float scale;           // softmax scale
  float scale_log2;      // scale * log2(e)
  int window, sinks;     // kWin: a row at position p sees keys (p - window, p] and [0, sinks)
  float* part;           // kWin: pieces of split key blocks, [pieces][kv heads][128 keys][dV | dK, unscaled]
  uint32_t* err;
  uint64_t timeout_ns;
};

// Entry and kv head of item i of a list (heads innermost); false for i < 0.
__device__ __forceinline__ bool var_item(const VarItem* items, int n_items, int kv_heads, int i, VarItem& it, int& hkv) {
  if (i < 0) return false;
  const int e = i / kv_heads;
  hkv = i - e * kv_heads;
  const int4* p = reinterpret_cast<const int4*>(items + e);
  const int4 x = __ldg(p), y = __ldg(p + 1);
  it = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  return true;
}

// Rows [first, end) of a [128 x D] tile set to zero by one warp, then made visible to the tensor core's reads.
template <int kD>
__device__ __forceinline__ void zero_rows_warp(uint8_t* tile, int first, int end) {
  constexpr int kPer = kD / 8;
  const int lane = ptx::lane_id();
  uint8_t* piece = tile + ((lane % kPer) >> 3) * kAttnChunk + (lane & 7) * 16;  // this lane's, of row 0
#pragma unroll 4
  for (int r = first + lane / kPer; r < end; r += 32 / kPer) *reinterpret_cast<uint4*>(piece + r * 128) = make_uint4(0, 0, 0, 0);
  ptx::fence_proxy_async_smem();
  __syncwarp();
}

// write_acc_half for rows that exist only (the TMEM loads are the whole warp's).
template <bool kF16, int kD>
__device__ __forceinline__ void write_acc_half_if(uint32_t t_row, int x, uint16_t* row_out, float mul, bool live) {
#pragma unroll 1
  for (int cc = 0; cc < kD / 64; ++cc) {
    const int col = x * (kD / 2) + cc * 32;
    uint32_t u[32];
    ptx::tmem_ld_32x32b_x32(t_row + col, u);
    ptx::tmem_wait_ld();
    if (live) store_row_half<kF16>(row_out + col, u, mul);
    __syncwarp();
  }
}

// The same into a piece's fp32 rows.
template <int kD>
__device__ __forceinline__ void write_acc_half_f32(uint32_t t_row, int x, float* row_out) {
#pragma unroll 1
  for (int cc = 0; cc < kD / 64; ++cc) {
    const int col = x * (kD / 2) + cc * 32;
    uint32_t u[32];
    ptx::tmem_ld_32x32b_x32(t_row + col, u);
    ptx::tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; i += 8) st_global_v8(row_out + col + i, u + i);
    __syncwarp();
  }
}

// Blocks 0 and 1 build the two work lists (query tiles, key blocks); block 2 + s * groups + i writes the statistics of tile
// slot s for kv heads i, i + groups, ..: D / 8 lanes per row, fp32 sums, the loads of all heads' rows independent of one
// another.
struct VarPrepArgs {
  PlanArgs plan[2];
  const void* dO;
  int64_t do_token_stride, do_head_stride;
  const void* O;        // contiguous
  const float* lse;     // [tokens, heads]
  float* stats;
  int heads, kv_heads, group, head_groups;
};

template <bool kF16, int kD>
__global__ void __launch_bounds__(kPlanThreads) varattn_bwd_prep_kernel(const __grid_constant__ VarPrepArgs a) {
  ptx::grid_launch_dependents();
  if (blockIdx.x < 2) {
    build_plan(a.plan[blockIdx.x]);
    return;
  }
  constexpr int kTpr = kD / 8, kRowsAtOnce = kPlanThreads / kTpr;  // 64 or 128 rows
  const int slot = (blockIdx.x - 2) / a.head_groups, first = (blockIdx.x - 2) % a.head_groups;
  VarItem it;
  if (!plan_item(a.plan[0], a.plan[0].cu, nullptr, slot, it) || it.b1 <= it.b0) return;
  const int c = threadIdx.x % kTpr;
#pragma unroll
  for (int r0 = 0; r0 < kVarBlk; r0 += kRowsAtOnce) {
    const int r = r0 + threadIdx.x / kTpr;
    const int tok = r / a.group, hd = r - tok * a.group;
    const bool live = tok < it.ntok;
    const int64_t t = it.row0 + (live ? tok : 0);
    const uint16_t* g_row = static_cast<const uint16_t*>(a.dO) + t * a.do_token_stride + hd * a.do_head_stride + 8 * c;
    const uint16_t* o_row = static_cast<const uint16_t*>(a.O) + (t * a.heads + hd) * kD + 8 * c;
    // kAtOnce heads' rows are loaded before any is used (7 sequences, 8192 tokens, 16 / 4 heads, D 64: 12.3 us where a loop
    // over single heads takes 14.6)
    constexpr int kAtOnce = 4;
    for (int h0 = first; h0 < a.kv_heads; h0 += kAtOnce * a.head_groups) {
      uint4 x[kAtOnce], y[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int hkv = h0 + i * a.head_groups;
        x[i] = y[i] = make_uint4(0, 0, 0, 0);
        if (live && hkv < a.kv_heads) {
          x[i] = __ldg(reinterpret_cast<const uint4*>(g_row + static_cast<int64_t>(hkv) * a.group * a.do_head_stride));
          y[i] = __ldg(reinterpret_cast<const uint4*>(o_row + static_cast<int64_t>(hkv) * a.group * kD));
        }
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int hkv = h0 + i * a.head_groups;
        if (hkv >= a.kv_heads) break;  // the same for the whole block
        const uint32_t wx[4] = {x[i].x, x[i].y, x[i].z, x[i].w}, wy[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
        float acc = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 fx = unpack2<kF16>(wx[k]), fy = unpack2<kF16>(wy[k]);
          acc = fmaf(fx.x, fy.x, acc);
          acc = fmaf(fx.y, fy.y, acc);
        }
#pragma unroll
        for (int o = kTpr / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
        if (c == 0) {
          float* st = a.stats + (static_cast<int64_t>(slot) * a.kv_heads + hkv) * 256 + r;
          st[0] = live ? -__ldg(a.lse + t * a.heads + hkv * a.group + hd) * 1.4426950408889634f : -INFINITY;
          st[128] = acc;
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ dQ pass
// Item = query tile and kv head; streams the K / V tiles of its key blocks through a ring. TMEM: S [0,128), dP [128,256), dQ
// accumulator [256, 256 + D), dS (packed pairs) [384, 448). Warpgroup x takes keys [64x, 64x + 64) of a block. Order per block
// j: S(j), dP(j); once S(j) sits in registers the next block's S is issued; once dS(j) is in TMEM, dQ += dS(j) K_j and the next
// block's dP.
template <bool kF16, int kD, bool kWin = false>
__global__ void __launch_bounds__(kBwdThreads, 1)
    varattn_bwd_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                         const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmdO,
                         const VarBwdArgs a) {
  using Sh = BwdDqShape<kF16, kD>;
  constexpr int kTile = Sh::kTile;
  constexpr int kSlots = Sh::kSlots;
  constexpr uint32_t kFmt = kF16 ? 0u : 1u;
  constexpr uint32_t IDESC_S = ptx::instr_desc(128, 128, kFmt, kFmt, 0, 0);  // S, dP: K = D, both K-major
  constexpr uint32_t IDESC_DQ = ptx::instr_desc(128, kD, kFmt, kFmt, 0, 1);  // dQ += dS K: K MN-major
  constexpr uint32_t T_S = 0, T_DP = 128, T_DQ = 256, T_DS = 384;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sdO = sQ + kTile;
  uint8_t* sKV = sdO + kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + kSlots * kTile);
  uint64_t* qd_full = bars + 0;
  uint64_t* qd_empty = bars + 1;
  uint64_t* kv_full = bars + 2;
  uint64_t* kv_empty = kv_full + kSlots;
  uint64_t* raw_full = kv_empty + kSlots;  // a K / V tile with foreign rows has arrived
  uint64_t* s_full = raw_full + kSlots;   // S of the current block in TMEM
  uint64_t* dp_full = s_full + 1;         // dP of the current block in TMEM
  uint64_t* s_free = dp_full + 1;         // 8 warp arrivals: S has been read into registers
  uint64_t* ds_full = s_free + 1;         // 8 warp arrivals: dS written (packed) to TMEM
  uint64_t* dq_done = ds_full + 1;
  uint64_t* dq_empty = dq_done + 1;        // 8 warp arrivals: the accumulator has been read out
  uint64_t* drain = dq_empty + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    ptx::mbar_init(ptx::smem_u32(qd_full), 1);
    ptx::mbar_init(ptx::smem_u32(qd_empty), 1);
    for (int s = 0; s < kSlots; ++s) {
      ptx::mbar_init(ptx::smem_u32(&kv_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&kv_empty[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&raw_full[s]), 1);
    }
    ptx::mbar_init(ptx::smem_u32(s_full), 1);
    ptx::mbar_init(ptx::smem_u32(dp_full), 1);
    ptx::mbar_init(ptx::smem_u32(s_free), 8);
    ptx::mbar_init(ptx::smem_u32(ds_full), 8);
    ptx::mbar_init(ptx::smem_u32(dq_done), 1);
    ptx::mbar_init(ptx::smem_u32(dq_empty), 8);
    ptx::mbar_init(ptx::smem_u32(drain), 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&tmQ);
    ptx::prefetch_tmap(&tmK);
    ptx::prefetch_tmap(&tmV);
    ptx::prefetch_tmap(&tmdO);
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_holder), kAttnTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  WaitCtl ctl{abort_flag, a.err, a.timeout_ns, kKidVarAttnBwd};
  if (warp < 4) ptx::setmaxnreg_dec<kBwdRegsLow>();

  ptx::grid_dependency_wait();
  const int n_items = *a.q_count * a.kv_heads;  // (entry, kv head), heads innermost
  const int cta = blockIdx.x, grid = gridDim.x, group = a.group, tt = kVarBlk / group;
  auto item_at = [&](int k, VarItem& it, int& hkv) -> bool {
    return var_item(a.q_items, n_items, a.kv_heads, zigzag(k, cta, grid, n_items), it, hkv);
  };
  // Key block of entry b of the item's list (see win_skip).
  const int sink_blocks = kWin ? win_sink_blocks(a.sinks) : 0;
  auto block_of = [&](const VarItem& it, int b) -> int {
    return kWin && b >= sink_blocks ? b + win_skip(it.pos0, a.window, a.sinks) : b;
  };

  // Rows [sinks_end, gap_end) of entry b's K: keys beside the sinks that the window leaves out for the whole tile. dS = 0 would not
  // stop a NaN in them (in V it would: dS of a masked key is replaced).
  const int sinks_end = kWin && a.sinks % kVarBlk ? a.sinks % kVarBlk : kVarBlk;
  auto gap_end = [&](const VarItem& it, int b) -> int {
    return kWin && b == sink_blocks - 1 ? min(it.pos0 - a.window + 1 - b * kVarBlk, kVarBlk) : 0;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (one thread)
    if (lane == 0) {
      uint32_t qd_phase = 0, slot = 0, slot_phase = 0, qd_issued = 0, kv_issued = 0;
      bool ok = true;
      const uint32_t kv0 = ptx::smem_u32(sKV);
      auto push = [&](const CUtensorMap* m, int hkv, int row, bool foreign) -> bool {
        if (!wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(&kv_empty[slot]), slot_phase ^ 1, ctl, 2)) return false;
        const uint32_t fb = ptx::smem_u32(foreign ? &raw_full[slot] : &kv_full[slot]);
        ptx::mbar_arrive_expect_tx(fb, kTile);
#pragma unroll
        for (int c = 0; c < Sh::kChunks; ++c)
          ptx::tma_load_3d(kv0 + slot * kTile + c * kAttnChunk, m, fb, 64 * c, hkv, row);
        ++kv_issued;
        if (++slot == kSlots) { slot = 0; slot_phase ^= 1; }
        return true;
      };
      VarItem it;
      int hkv;
      for (int k = 0; ok && item_at(k, it, hkv); ++k) {
        if (it.b1 <= it.b0) continue;
        ok = wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(qd_empty), qd_phase ^ 1, ctl, 1);
        if (!ok) break;
        const uint32_t qf = ptx::smem_u32(qd_full);
        ptx::mbar_arrive_expect_tx(qf, 2 * tt * group * kD * 2);
#pragma unroll
        for (int c = 0; c < Sh::kChunks; ++c) {
          ptx::tma_load_3d(ptx::smem_u32(sQ) + c * kAttnChunk, &tmQ, qf, 64 * c, hkv * group, it.row0);
          ptx::tma_load_3d(ptx::smem_u32(sdO) + c * kAttnChunk, &tmdO, qf, 64 * c, hkv * group, it.row0);
        }
        ++qd_issued;
        qd_phase ^= 1;
        for (int x = it.b0; x < it.b1 && ok; ++x) {
          const int b = block_of(it, x), row = it.src + b * kVarBlk;
          const bool foreign = it.kv_len - b * kVarBlk < kVarBlk;
          ok = push(&tmK, hkv, row, foreign || (kWin && gap_end(it, x) > sinks_end)) && push(&tmV, hkv, row, foreign);
        }
      }
      WaitCtl dctl = ctl;
      volatile int never = 0;
      dctl.abort = &never;
      if (qd_issued) wait_bounded(ptx::smem_u32(qd_full), (qd_issued - 1) & 1, dctl, 8);
      const uint32_t first = kv_issued > kSlots ? kv_issued - kSlots : 0;
      for (uint32_t i = first; i < kv_issued; ++i)
        wait_bounded(ptx::smem_u32(&kv_full[i % kSlots]), (i / kSlots) & 1, dctl, 8);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (one thread)
    if (lane == 0) {
      uint32_t qd_phase = 0, slot = 0, slot_phase = 0, items_done = 0, sf_cnt = 0, ds_cnt = 0;
      bool ok = true;
      const uint32_t kv0 = ptx::smem_u32(sKV), q0 = ptx::smem_u32(sQ), do0 = ptx::smem_u32(sdO);
      auto take = [&](uint32_t site) -> uint32_t {
        if (!wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(&kv_full[slot]), slot_phase, ctl, site)) return 0xFFFFFFFFu;
        const uint32_t s = slot;
        if (++slot == kSlots) { slot = 0; slot_phase ^= 1; }
        return s;
      };
      auto issue_s = [&](uint32_t sk) {  // S = Q K^T
        mma_kmajor<kD>(tmem_base + T_S, q0, kv0 + sk * kTile, IDESC_S);
        ptx::mma_commit(ptx::smem_u32(s_full));
      };
      auto issue_dp = [&](uint32_t sv) {  // dP = dO V^T
        mma_kmajor<kD>(tmem_base + T_DP, do0, kv0 + sv * kTile, IDESC_S);
        ptx::mma_commit(ptx::smem_u32(dp_full));
      };
      auto issue_dq = [&](uint32_t sk, bool first) {  // dQ += dS K: K step k = keys [16k, 16k + 16), dS columns 8k
        const uint32_t kA = kv0 + sk * kTile;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          ptx::mma_f16_ts(tmem_base + T_DQ, tmem_base + T_DS + 8 * k,
                          ptx::smem_desc(kA + k * 2048, kAttnChunk, 1024), IDESC_DQ, (first && k == 0) ? 0u : 1u);
      };
      // Per block j: S(j), dP(j) | S read -> S(j+1) | dS(j) written -> dQ(j), dP(j+1): the scores of the next block
      // are computed while the warps work on this one.
      VarItem it;
      int hkv;
      for (int k = 0; ok && item_at(k, it, hkv); ++k) {
        const int n = it.b1 - it.b0;
        if (n <= 0) continue;
        ok = wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(qd_full), qd_phase, ctl, 10);
        if (!ok) break;
        qd_phase ^= 1;
        uint32_t sk = take(11), sv = 0xFFFFFFFFu;
        if (sk != 0xFFFFFFFFu) sv = take(12);
        if (sv == 0xFFFFFFFFu) { ok = false; break; }
        ptx::tc_fence_after();
        issue_s(sk);
        issue_dp(sv);
        if (items_done > 0) {  // the previous item's dQ has been read out of TMEM
          ok = wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(dq_empty), (items_done - 1) & 1, ctl, 16);
          if (!ok) break;
        }
        for (int j = 0; j < n && ok; ++j) {
          ok = wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(s_free), sf_cnt & 1, ctl, 13);
          if (!ok) break;
          ++sf_cnt;
          uint32_t nk = 0xFFFFFFFFu, nv = 0xFFFFFFFFu;
          if (j + 1 < n) {
            nk = take(11);
            if (nk != 0xFFFFFFFFu) nv = take(12);
            if (nv == 0xFFFFFFFFu) { ok = false; break; }
            ptx::tc_fence_after();
            issue_s(nk);
          }
          ok = wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(ds_full), ds_cnt & 1, ctl, 14);
          if (!ok) break;
          ++ds_cnt;
          ptx::tc_fence_after();
          issue_dq(sk, j == 0);
          ptx::mma_commit(ptx::smem_u32(&kv_empty[sk]));
          ptx::mma_commit(ptx::smem_u32(&kv_empty[sv]));
          if (j + 1 < n) issue_dp(nv);
          sk = nk;
          sv = nv;
        }
        if (!ok) break;
        ptx::mma_commit(ptx::smem_u32(dq_done));
        ptx::mma_commit(ptx::smem_u32(qd_empty));
        ++items_done;
      }
      ptx::mma_commit(ptx::smem_u32(drain));
      WaitCtl dctl = ctl;
      volatile int never = 0;
      dctl.abort = &never;
      wait_bounded(ptx::smem_u32(drain), 0, dctl, 15);
    }
    __syncwarp();
  } else if (warp == 2) {
    // ------------------------------------------------------------------ foreign K and V rows -> zero
    uint32_t seq = 0, phases = 0;  // ring positions passed; bit s: parity of raw_full[s]'s next completion
    bool ok = true;
    VarItem it;
    int hkv;
    for (int k = 0; ok && item_at(k, it, hkv); ++k) {
      const int n = it.b1 - it.b0;
      if (n <= 0) continue;
      // the K tile of the last sinks' block, where some of its keys are left out, and the item's last K tile and last V tile
      for (int y = kWin ? 0 : 1; y < 2 && ok; ++y) {
        const int b = y ? it.b1 - 1 : sink_blocks - 1;
        if (kWin && !y && (b < it.b0 || b >= it.b1 - 1)) continue;
        const int live = y ? it.kv_len - block_of(it, b) * kVarBlk : kVarBlk, gap = gap_end(it, b);
        for (int w = 0; w < 2 && ok; ++w) {
          if (live >= kVarBlk && (!kWin || w || gap <= sinks_end)) continue;
          const uint32_t sl = (seq + 2 * (b - it.b0) + w) % kSlots;
          ok = warp_wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(&raw_full[sl]), (phases >> sl) & 1, ctl, 30);
          if (!ok) break;
          phases ^= 1u << sl;
          if (kWin && !w) zero_rows_warp<kD>(sKV + sl * kTile, sinks_end, gap);
          zero_rows_warp<kD>(sKV + sl * kTile, live, kVarBlk);
          if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&kv_full[sl]));
        }
      }
      seq += 2 * n;
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ dS = P (dP - Delta), dQ out
    ptx::setmaxnreg_inc<kBwdRegsHigh>();
    const int x = (warp - 4) >> 2;  // key half: positions [64x, 64x + 64)
    const int q = warp & 3;
    const int r = 32 * q + lane;    // row of the tile == TMEM lane
    const int tok = r / group, hd = r - tok * group;
    const uint32_t lane_off = static_cast<uint32_t>(32 * q) << 16;
    const uint64_t c2 = f2_pack(a.scale_log2, a.scale_log2);
    uint32_t s_cnt = 0, dp_cnt = 0, dq_cnt = 0;
    bool ok = true;
    VarItem it;
    int hkv;
    for (int k = 0; ok && item_at(k, it, hkv); ++k) {
      const bool live = tok < it.ntok;
      const int64_t grow = static_cast<int64_t>(it.row0 + tok) * a.heads + hkv * group + hd;
      uint16_t* dq_row = static_cast<uint16_t*>(a.dQ) + grow * kD;
      if (it.b1 <= it.b0) {
        if (live) zero_row_half<kD>(x, dq_row);
        continue;
      }
      const float* st = a.stats + (static_cast<int64_t>(it.part) * a.kv_heads + hkv) * 256 + r;
      const float off = __ldg(st), ndlt = -__ldg(st + 128);
      const uint64_t off2 = f2_pack(off, off), ndlt2 = f2_pack(ndlt, ndlt);
      const int limit = a.causal ? it.pos0 + tok + 1 : it.kv_len;        // keys at or behind it are masked for this row
      const int clear = (a.causal ? it.pos0 + 1 : it.kv_len) >> 7;       // key blocks below it are seen by every row
      // a window also masks keys before `lo` (the sinks apart); key blocks that start before `lo_all` have such keys for some row
      const int lo = it.pos0 + tok - a.window + 1, lo_all = it.pos0 + tt - a.window;
      for (int j = it.b0; j < it.b1; ++j) {
        const int kb = block_of(it, j);
        ok = warp_wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(s_full), s_cnt & 1, ctl, 20);
        if (!ok) break;
        ++s_cnt;
        ptx::tc_fence_after();
        uint32_t pv[64];  // S, then P (fp32) of this warp's 64 keys
        const uint32_t ts = tmem_base + lane_off + T_S + 64 * x, tp = tmem_base + lane_off + T_DP + 64 * x;
        ptx::tmem_ld_32x32b_x32(ts, *reinterpret_cast<uint32_t(*)[32]>(&pv[0]));
        ptx::tmem_ld_32x32b_x32(ts + 32, *reinterpret_cast<uint32_t(*)[32]>(&pv[32]));
        ptx::tmem_wait_ld();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(s_free));  // the next block's S may overwrite it
        const int lim = kb >= clear ? limit - (kb * kVarBlk + 64 * x) : 64;
        uint32_t seen[2] = {~0u, ~0u};
        if constexpr (kWin) {
          if (kb >= clear || (kb * kVarBlk < lo_all && (kb + 1) * kVarBlk > a.sinks)) {
            const int base = kb * kVarBlk + 64 * x;
            seen[0] = seen_bits(base, limit, lo, a.sinks);
            seen[1] = seen_bits(base + 32, limit, lo, a.sinks);
          }
        }
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          float p0, p1;
          f2_unpack(f2_ex2_split<kVarFloor>(f2_fma(f2_pack(__uint_as_float(pv[i]), __uint_as_float(pv[i + 1])), c2, off2),
                                 ((i >> 1) & 7) >= 8 - kBwdPolyEighths),
                    p0, p1);
          pv[i] = __float_as_uint(p0);
          pv[i + 1] = __float_as_uint(p1);
        }
        ok = warp_wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(dp_full), dp_cnt & 1, ctl, 21);
        if (!ok) break;
        ++dp_cnt;
        ptx::tc_fence_after();
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          uint32_t dv[32];
          ptx::tmem_ld_32x32b_x32(tp + 32 * cc, dv);
          ptx::tmem_wait_ld();
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float g0, g1;
            f2_unpack(f2_mul(f2_pack(__uint_as_float(pv[32 * cc + i]), __uint_as_float(pv[32 * cc + i + 1])),
                             f2_add(f2_pack(__uint_as_float(dv[i]), __uint_as_float(dv[i + 1])), ndlt2)),
                      g0, g1);
            // (the product, not P: dP of a masked key may be infinite)
            if (kWin ? !(seen[cc] >> i & 1) : 32 * cc + i >= lim) g0 = 0.0f;
            if (kWin ? !(seen[cc] >> (i + 1) & 1) : 32 * cc + i + 1 >= lim) g1 = 0.0f;
            pk[i >> 1] = pack2<kF16>(g0, g1);
          }
          ptx::tmem_st_32x32b_x16(tmem_base + lane_off + T_DS + 32 * x + 16 * cc, pk);
        }
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(ds_full));
      }
      if (!ok) break;
      ok = warp_wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(dq_done), dq_cnt & 1, ctl, 22);
      if (!ok) break;
      ++dq_cnt;
      ptx::tc_fence_after();
      write_acc_half_if<kF16, kD>(tmem_base + lane_off + T_DQ, x, dq_row, a.scale, live);
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(dq_empty));
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc(tmem_base, kAttnTmemCols);
}

// ------------------------------------------------------------------------------------------------ dK/dV pass
// Item = key block and kv head; streams the Q and dO tiles (and their row statistics) that see it. TMEM: S^T [0,128) -> packed
// P^T of warpgroup x's query rows [64x, 64x + 64) at [64x, 64x + 32); dP^T [128,256) -> packed dS^T likewise at [128 + 64x, ...);
// dV accumulator [256, 256 + D), dK [256 + D, 256 + 2D). Order per tile t: S^T(t), dP^T(t); P^T written -> dV(t), S^T(t+1); dS^T
// written -> dK(t), dP^T(t+1).
template <bool kF16, int kD, bool kWin = false>
__global__ void __launch_bounds__(kBwdThreads, 1)
    varattn_bwd_dkdv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                           const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmdO,
                           const VarBwdArgs a) {
  using Sh = BwdDkdvShape<kF16, kD>;
  constexpr int kTile = Sh::kTile;
  constexpr int kSlots = Sh::kSlots;
  constexpr int kSlotBytes = Sh::kSlotBytes;
  constexpr uint32_t kFmt = kF16 ? 0u : 1u;
  constexpr uint32_t IDESC_S = ptx::instr_desc(128, 128, kFmt, kFmt, 0, 0);   // S^T, dP^T: K = D, both K-major
  constexpr uint32_t IDESC_ACC = ptx::instr_desc(128, kD, kFmt, kFmt, 0, 1);  // dV, dK: B (dO, Q) MN-major
  constexpr uint32_t T_S = 0, T_DP = 128, T_DV = 256, T_DK = 256 + kD;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = sK + kTile;
  uint8_t* sQD = sV + kTile;  // [kSlots] x (Q tile, dO tile, -LSE*log2(e), Delta)
  uint64_t* bars = reinterpret_cast<uint64_t*>(sQD + kSlots * kSlotBytes);
  uint64_t* kv_full = bars + 0;
  uint64_t* kv_empty = bars + 1;
  uint64_t* qd_full = bars + 2;
  uint64_t* qd_empty = qd_full + kSlots;
  uint64_t* raw_full = qd_empty + kSlots;  // a Q / dO tile with foreign rows has arrived
  uint64_t* s_full = raw_full + kSlots;   // S^T of the current block in TMEM
  uint64_t* dp_full = s_full + 1;         // dP^T of the current block in TMEM
  uint64_t* p_full = dp_full + 1;         // 8 warp arrivals: P^T written (packed) to TMEM
  uint64_t* ds_full = p_full + 1;         // 8 warp arrivals: dS^T written (packed) to TMEM
  uint64_t* acc_done = ds_full + 1;
  uint64_t* acc_empty = acc_done + 1;      // 8 warp arrivals: dK / dV read out of TMEM
  uint64_t* drain = acc_empty + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    ptx::mbar_init(ptx::smem_u32(kv_full), 1);
    ptx::mbar_init(ptx::smem_u32(kv_empty), 1);
    for (int s = 0; s < kSlots; ++s) {
      ptx::mbar_init(ptx::smem_u32(&qd_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&qd_empty[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&raw_full[s]), 1);
    }
    ptx::mbar_init(ptx::smem_u32(s_full), 1);
    ptx::mbar_init(ptx::smem_u32(dp_full), 1);
    ptx::mbar_init(ptx::smem_u32(p_full), 8);
    ptx::mbar_init(ptx::smem_u32(ds_full), 8);
    ptx::mbar_init(ptx::smem_u32(acc_done), 1);
    ptx::mbar_init(ptx::smem_u32(acc_empty), 8);
    ptx::mbar_init(ptx::smem_u32(drain), 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (kVarBlk % a.group) {  // rows that no copy fills: they meet P = 0 and have to be finite
    for (int s = 0; s < 2 * kSlots; ++s)
      zero_tile_rows(sQD + (s >> 1) * kSlotBytes + (s & 1) * kTile, Sh::kChunks, kVarBlk / a.group * a.group);
    ptx::fence_proxy_async_smem();
  }
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&tmQ);
    ptx::prefetch_tmap(&tmK);
    ptx::prefetch_tmap(&tmV);
    ptx::prefetch_tmap(&tmdO);
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_holder), kAttnTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  WaitCtl ctl{abort_flag, a.err, a.timeout_ns, kKidVarAttnBwd};
  if (warp < 4) ptx::setmaxnreg_dec<kBwdRegsLow>();

  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int n_items = *a.k_count * a.kv_heads;  // (entry, kv head), heads innermost
  const int cta = blockIdx.x, grid = gridDim.x, group = a.group, tt = kVarBlk / group;
  auto item_at = [&](int k, VarItem& it, int& hkv) -> bool {
    return var_item(a.k_items, n_items, a.kv_heads, zigzag(k, cta, grid, n_items), it, hkv);
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (one thread)
    if (lane == 0) {
      uint32_t kv_phase = 0, slot = 0, slot_phase = 0, kv_issued = 0, qd_issued = 0;
      bool ok = true;
      const uint32_t qd0 = ptx::smem_u32(sQD);
      VarItem it;
      int hkv;
      for (int k = 0; ok && item_at(k, it, hkv); ++k) {
        if (it.b1 <= it.b0) continue;
        ok = wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(kv_empty), kv_phase ^ 1, ctl, 1);
        if (!ok) break;
        const uint32_t kf = ptx::smem_u32(kv_full);
        ptx::mbar_arrive_expect_tx(kf, 2 * kTile);
#pragma unroll
        for (int c = 0; c < Sh::kChunks; ++c) {
          ptx::tma_load_3d(ptx::smem_u32(sK) + c * kAttnChunk, &tmK, kf, 64 * c, hkv, it.row0 + it.pos0);
          ptx::tma_load_3d(ptx::smem_u32(sV) + c * kAttnChunk, &tmV, kf, 64 * c, hkv, it.row0 + it.pos0);
        }
        ++kv_issued;
        kv_phase ^= 1;
        for (int t = it.b0; t < it.b1 && ok; ++t) {
          ok = wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(&qd_empty[slot]), slot_phase ^ 1, ctl, 2);
          if (!ok) break;
          const bool foreign = it.ntok - t * tt < tt;  // the sequence's last tile, not full
          const uint32_t fb = ptx::smem_u32(foreign ? &raw_full[slot] : &qd_full[slot]);
          const uint32_t dst = qd0 + slot * kSlotBytes;
          ptx::mbar_arrive_expect_tx(fb, 2 * tt * group * kD * 2 + 1024);
          ptx::bulk_load_1d(dst + 2 * kTile, a.stats + (static_cast<int64_t>(it.src + t) * a.kv_heads + hkv) * 256, 1024, fb);
#pragma unroll
          for (int c = 0; c < Sh::kChunks; ++c) {
            ptx::tma_load_3d(dst + c * kAttnChunk, &tmQ, fb, 64 * c, hkv * group, it.row0 + t * tt);
            ptx::tma_load_3d(dst + kTile + c * kAttnChunk, &tmdO, fb, 64 * c, hkv * group, it.row0 + t * tt);
          }
          ++qd_issued;
          if (++slot == kSlots) { slot = 0; slot_phase ^= 1; }
        }
      }
      WaitCtl dctl = ctl;
      volatile int never = 0;
      dctl.abort = &never;
      if (kv_issued) wait_bounded(ptx::smem_u32(kv_full), (kv_issued - 1) & 1, dctl, 8);
      const uint32_t first = qd_issued > kSlots ? qd_issued - kSlots : 0;
      for (uint32_t i = first; i < qd_issued; ++i)
        wait_bounded(ptx::smem_u32(&qd_full[i % kSlots]), (i / kSlots) & 1, dctl, 8);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (one thread)
    if (lane == 0) {
      uint32_t kv_phase = 0, slot = 0, slot_phase = 0, items_done = 0, p_cnt = 0, ds_cnt = 0;
      bool ok = true;
      const uint32_t qd0 = ptx::smem_u32(sQD), k0 = ptx::smem_u32(sK), v0 = ptx::smem_u32(sV);
      auto take = [&](uint32_t site) -> uint32_t {
        if (!wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(&qd_full[slot]), slot_phase, ctl, site)) return 0xFFFFFFFFu;
        const uint32_t s = slot;
        if (++slot == kSlots) { slot = 0; slot_phase ^= 1; }
        return s;
      };
      auto issue_s = [&](uint32_t sl) {  // S^T = K Q^T
        mma_kmajor<kD>(tmem_base + T_S, k0, qd0 + sl * kSlotBytes, IDESC_S);
        ptx::mma_commit(ptx::smem_u32(s_full));
      };
      auto issue_dp = [&](uint32_t sl) {  // dP^T = V dO^T
        mma_kmajor<kD>(tmem_base + T_DP, v0, qd0 + sl * kSlotBytes + kTile, IDESC_S);
        ptx::mma_commit(ptx::smem_u32(dp_full));
      };
      // K step k = query rows [16k, 16k + 16): packed columns 8k of half 0, 64 + 8(k - 4) of half 1
      auto pcol = [](int k) -> uint32_t { return 8 * k + (k >= 4 ? 32 : 0); };
      auto issue_dv = [&](uint32_t sl, bool first) {  // dV += P^T dO
        const uint32_t dA = qd0 + sl * kSlotBytes + kTile;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          ptx::mma_f16_ts(tmem_base + T_DV, tmem_base + T_S + pcol(k), ptx::smem_desc(dA + k * 2048, kAttnChunk, 1024),
                          IDESC_ACC, (first && k == 0) ? 0u : 1u);
      };
      auto issue_dk = [&](uint32_t sl, bool first) {  // dK += dS^T Q
        const uint32_t qA = qd0 + sl * kSlotBytes;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          ptx::mma_f16_ts(tmem_base + T_DK, tmem_base + T_DP + pcol(k), ptx::smem_desc(qA + k * 2048, kAttnChunk, 1024),
                          IDESC_ACC, (first && k == 0) ? 0u : 1u);
      };
      // Per block t: S^T(t), dP^T(t) | P^T written -> dV(t), S^T(t+1) | dS^T written -> dK(t), dP^T(t+1): the
      // warps compute P^T while dP^T runs and dS^T while dV and the next S^T run.
      VarItem it;
      int hkv;
      for (int k = 0; ok && item_at(k, it, hkv); ++k) {
        const int n = it.b1 - it.b0;
        if (n <= 0) continue;
        ok = wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(kv_full), kv_phase, ctl, 10);
        if (!ok) break;
        kv_phase ^= 1;
        uint32_t cur = take(11);
        if (cur == 0xFFFFFFFFu) { ok = false; break; }
        ptx::tc_fence_after();
        issue_s(cur);
        issue_dp(cur);
        if (items_done > 0) {  // the previous item's dK / dV have been read out of TMEM
          ok = wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(acc_empty), (items_done - 1) & 1, ctl, 16);
          if (!ok) break;
        }
        for (int t = 0; t < n && ok; ++t) {
          // The next slot is taken in the same burst of waits as P^T (a poll after queued MMAs drains the pipe).
          ok = wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(p_full), p_cnt & 1, ctl, 12);
          if (!ok) break;
          ++p_cnt;
          uint32_t nxt = 0xFFFFFFFFu;
          if (t + 1 < n) {
            nxt = take(11);
            if (nxt == 0xFFFFFFFFu) { ok = false; break; }
          }
          ptx::tc_fence_after();
          issue_dv(cur, t == 0);
          if (t + 1 < n) issue_s(nxt);
          ok = wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(ds_full), ds_cnt & 1, ctl, 13);
          if (!ok) break;
          ++ds_cnt;
          ptx::tc_fence_after();
          issue_dk(cur, t == 0);
          ptx::mma_commit(ptx::smem_u32(&qd_empty[cur]));
          if (t + 1 < n) issue_dp(nxt);
          cur = nxt;
        }
        if (!ok) break;
        ptx::mma_commit(ptx::smem_u32(acc_done));
        ptx::mma_commit(ptx::smem_u32(kv_empty));
        ++items_done;
      }
      ptx::mma_commit(ptx::smem_u32(drain));
      WaitCtl dctl = ctl;
      volatile int never = 0;
      dctl.abort = &never;
      wait_bounded(ptx::smem_u32(drain), 0, dctl, 15);
    }
    __syncwarp();
  } else if (warp == 2) {
    // ------------------------------------------------------------------ foreign Q and dO rows -> zero
    uint32_t seq = 0, phases = 0;  // ring positions passed; bit s: parity of raw_full[s]'s next completion
    bool ok = true;
    VarItem it;
    int hkv;
    for (int k = 0; ok && item_at(k, it, hkv); ++k) {
      const int n = it.b1 - it.b0;
      if (n <= 0) continue;
      const int live = it.ntok - (it.b1 - 1) * tt;  // tokens of the last tile
      if (live < tt) {
        const uint32_t sl = (seq + n - 1) % kSlots;
        ok = warp_wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(&raw_full[sl]), (phases >> sl) & 1, ctl, 30);
        if (!ok) break;
        phases ^= 1u << sl;
        zero_rows_warp<kD>(sQD + sl * kSlotBytes, live * group, tt * group);
        zero_rows_warp<kD>(sQD + sl * kSlotBytes + kTile, live * group, tt * group);
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&qd_full[sl]));
      }
      seq += n;
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ P^T, dS^T, dK / dV out
    ptx::setmaxnreg_inc<kBwdRegsHigh>();
    const int x = (warp - 4) >> 2;  // half of the query rows ([64x, 64x + 64))
    const int q = warp & 3;
    const int r = 32 * q + lane;    // key of the block == TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>(32 * q) << 16;
    const uint64_t c2 = f2_pack(a.scale_log2, a.scale_log2);
    uint32_t s_cnt = 0, dp_cnt = 0, acc_cnt = 0, slot = 0, slot_phase = 0;
    bool ok = true;
    VarItem it;
    int hkv;
    for (int k = 0; ok && item_at(k, it, hkv); ++k) {
      const bool live = it.pos0 + r < it.kv_len;
      const int64_t grow = static_cast<int64_t>(it.row0 + it.pos0 + r) * a.kv_heads + hkv;
      uint16_t* dk_row = static_cast<uint16_t*>(a.dK) + grow * kD;
      uint16_t* dv_row = static_cast<uint16_t*>(a.dV) + grow * kD;
      if (it.b1 <= it.b0) {
        if (live) {
          zero_row_half<kD>(x, dk_row);
          zero_row_half<kD>(x, dv_row);
        }
        continue;
      }
      for (int t = it.b0; t < it.b1; ++t) {
        // Query rows c (token t * tt + c / group) before this key are masked: c < group * (key - t * tt), in this half
        // columns below `lim`.
        const int lim = a.causal ? (it.pos0 + r - t * tt) * group - 64 * x : 0;
        ok = warp_wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(&qd_full[slot]), slot_phase, ctl, 19);  // offsets
        if (ok) ok = warp_wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(s_full), s_cnt & 1, ctl, 20);
        if (!ok) break;
        ++s_cnt;
        ptx::tc_fence_after();
        const float* off_s = reinterpret_cast<const float*>(sQD + slot * kSlotBytes + 2 * kTile) + 64 * x;
        const float* dlt_s = off_s + 128;
        const uint32_t ts = tmem_base + lane_off + T_S + 64 * x, tp = tmem_base + lane_off + T_DP + 64 * x;
        bool diag = a.causal && t * tt < it.pos0 + kVarBlk - 1;
        // With a window, so are the columns from `far` on: tokens that are `window` or more behind this key (a sink has none).
        int far = 64;
        if constexpr (kWin) {
          const int key = it.pos0 + r;
          if (t * tt + tt > it.pos0 + a.window && it.pos0 + kVarBlk > a.sinks) {
            diag = true;
            if (key >= a.sinks)
              far = static_cast<int>(min(max(static_cast<int64_t>(key) + a.window - t * tt, int64_t{0}), int64_t{kVarBlk})) * group - 64 * x;
          }
        }
        float pf[64];  // P^T (fp32) of this warp's 64 query positions, kept for dS^T
        // Two chunks of 32 positions; chunk cc's packed values (16 columns) land at ts + 16cc, inside the columns
        // [0, 32) this warp has already read, never over chunk 1's unread scores.
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          uint32_t sv[32];
          ptx::tmem_ld_32x32b_x32(ts + 32 * cc, sv);
          ptx::tmem_wait_ld();
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 o = *reinterpret_cast<const float4*>(off_s + 32 * cc + i);
            float p0, p1, p2, p3;
            f2_unpack(f2_ex2_split<kVarFloor>(f2_fma(f2_pack(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1])), c2,
                                          f2_pack(o.x, o.y)),
                                   ((i >> 1) & 7) >= 8 - kBwdPolyEighths),
                      p0, p1);
            f2_unpack(f2_ex2_split<kVarFloor>(f2_fma(f2_pack(__uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3])), c2,
                                          f2_pack(o.z, o.w)),
                                   (((i >> 1) + 1) & 7) >= 8 - kBwdPolyEighths),
                      p2, p3);
            if (diag) {
              const int col = 32 * cc + i;
              if (col < lim || (kWin && col >= far)) p0 = 0.0f;
              if (col + 1 < lim || (kWin && col + 1 >= far)) p1 = 0.0f;
              if (col + 2 < lim || (kWin && col + 2 >= far)) p2 = 0.0f;
              if (col + 3 < lim || (kWin && col + 3 >= far)) p3 = 0.0f;
            }
            pf[32 * cc + i] = p0;
            pf[32 * cc + i + 1] = p1;
            pf[32 * cc + i + 2] = p2;
            pf[32 * cc + i + 3] = p3;
            pk[i >> 1] = pack2<kF16>(p0, p1);
            pk[(i >> 1) + 1] = pack2<kF16>(p2, p3);
          }
          ptx::tmem_st_32x32b_x16(ts + 16 * cc, pk);
        }
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(p_full));
        ok = warp_wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(dp_full), dp_cnt & 1, ctl, 21);
        if (!ok) break;
        ++dp_cnt;
        ptx::tc_fence_after();
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          uint32_t dv[32];
          ptx::tmem_ld_32x32b_x32(tp + 32 * cc, dv);
          ptx::tmem_wait_ld();
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 d = *reinterpret_cast<const float4*>(dlt_s + 32 * cc + i);
            float g0, g1, g2, g3;
            f2_unpack(f2_mul(f2_pack(pf[32 * cc + i], pf[32 * cc + i + 1]),
                             f2_add(f2_pack(__uint_as_float(dv[i]), __uint_as_float(dv[i + 1])), f2_pack(-d.x, -d.y))),
                      g0, g1);
            f2_unpack(f2_mul(f2_pack(pf[32 * cc + i + 2], pf[32 * cc + i + 3]),
                             f2_add(f2_pack(__uint_as_float(dv[i + 2]), __uint_as_float(dv[i + 3])),
                                    f2_pack(-d.z, -d.w))),
                      g2, g3);
            pk[i >> 1] = pack2<kF16>(g0, g1);
            pk[(i >> 1) + 1] = pack2<kF16>(g2, g3);
          }
          // P of a masked row is zero, but its dP may be infinite. (On the packed pairs, apart from the loop above: inside it,
          // every block executed the selects, 18 % more instructions and 5 % more time.)
          if (diag) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int col = 32 * cc + 2 * i;
              pk[i] &= (col < lim || (kWin && col >= far) ? 0u : 0x0000ffffu) |
                       (col + 1 < lim || (kWin && col + 1 >= far) ? 0u : 0xffff0000u);
            }
          }
          ptx::tmem_st_32x32b_x16(tp + 16 * cc, pk);
        }
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(ds_full));
        if (++slot == kSlots) { slot = 0; slot_phase ^= 1; }
      }
      if (!ok) break;
      ok = warp_wait_bounded_hint<kBwdSuspendNs>(ptx::smem_u32(acc_done), acc_cnt & 1, ctl, 22);
      if (!ok) break;
      ++acc_cnt;
      ptx::tc_fence_after();
      if (kWin && it.part >= 0) {
        float* row = a.part + ((static_cast<int64_t>(it.part) * a.kv_heads + hkv) * kVarBlk + r) * 2 * kD;
        write_acc_half_f32<kD>(tmem_base + lane_off + T_DV, x, row);
        write_acc_half_f32<kD>(tmem_base + lane_off + T_DK, x, row + kD);
      } else {
        write_acc_half_if<kF16, kD>(tmem_base + lane_off + T_DV, x, dv_row, 1.0f, live);
        write_acc_half_if<kF16, kD>(tmem_base + lane_off + T_DK, x, dk_row, a.scale, live);
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(acc_empty));
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc(tmem_base, kAttnTmemCols);
}

// Pieces of split key blocks -> dV and dK: sums in the pieces' order, one rounding. Block (split block, kv head, 16 keys); a
// thread adds up four neighbouring columns. Reads each partial result once, from L2.
struct VarJoinArgs {
  void* dK;
  void* dV;
  const float* part;
  const VarSplit* splits;
  const int* count;  // [1]: split key blocks
  int kv_heads;
  float scale;
};
constexpr int kJoinRows = 16;

template <bool kF16, int kD>
__global__ void __launch_bounds__(kJoinRows * kD / 2) varattn_bwd_join_kernel(const VarJoinArgs a) {
  ptx::grid_dependency_wait();
  if (static_cast<int>(blockIdx.x) >= a.count[1]) return;
  const VarSplit sp = a.splits[blockIdx.x];
  const int hkv = blockIdx.y, r = blockIdx.z * kJoinRows + threadIdx.x / (kD / 2), c = threadIdx.x % (kD / 2);
  if (r >= sp.ntok) return;
  const float4* p = reinterpret_cast<const float4*>(
      a.part + ((static_cast<int64_t>(sp.first) * a.kv_heads + hkv) * kVarBlk + r) * 2 * kD) + c;
  const int64_t step = static_cast<int64_t>(a.kv_heads) * kVarBlk * kD / 2;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = 0; i < sp.n; ++i) {
    const float4 v = __ldg(p + i * step);
    acc.x += v.x;
    acc.y += v.y;
    acc.z += v.z;
    acc.w += v.w;
  }
  const bool is_dk = c >= kD / 4;
  const float mul = is_dk ? a.scale : 1.0f;
  uint16_t* out = static_cast<uint16_t*>(is_dk ? a.dK : a.dV) + (static_cast<int64_t>(sp.row0 + r) * a.kv_heads + hkv) * kD;
  reinterpret_cast<uint2*>(out)[c % (kD / 4)] =
      make_uint2(pack2<kF16>(acc.x * mul, acc.y * mul), pack2<kF16>(acc.z * mul, acc.w * mul));
}

}  // namespace bsk
