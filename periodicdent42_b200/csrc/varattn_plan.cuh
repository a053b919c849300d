// Work lists of the packed / paged attention kernels, built on the device (sequence lengths stay there).
//
// The query rows of one sequence and kv head -- (token, head of the group), token-major -- are cut into tiles of
// TT = 128 / group tokens, the keys into blocks of 128. A list entry is one tile (or one key block for dK / dV); the kernels
// run every entry for each kv head. Entries are ordered by falling length (a counting sort, one CTA): the kernels hand them
// out in a fixed zigzag over the CTAs, so long and short ones even out without a counter in memory. The order inside a
// length is arbitrary and changes no result, since an entry's arithmetic depends on the entry alone.
//
// Where there are few entries for the GPU (a small chunk over a long cache), long ones are split along their keys; the
// pieces' results meet in a second kernel (varattn_combine_kernel).
//
// Tiles are numbered without a scan: tile j of sequence i is slot cu[i] / TT + i + j (sequences never overlap in it: the
// next one's first slot is at least ceil(n_i / TT) further). Slots from cu[batch] / TT + batch on cover the rows behind the
// last sequence, whose outputs are zero.
#pragma once

#include <climits>

#include "paged_decode_sm100.cuh"

namespace bsk {

constexpr uint32_t kKidVarAttn = 11;
constexpr int kPlanThreads = 1024;
constexpr int kPlanBuckets = 1024;
constexpr int kVarBlk = 128;

struct __align__(16) VarItem {
  int row0;    // first token row of the tile (of the key block's sequence, for dK / dV)
  int ntok;    // tokens of the tile (of the sequence)
  int src;     // first K / V token row, or the sequence's index for a paged cache (tile slot of the sequence, for dK / dV)
  int kv_len;  // keys of the sequence
  int pos0;    // position of the tile's first token (first key of the block, for dK / dV)
  int b0, b1;  // key blocks [b0, b1) (query tiles, for dK / dV)
  int part;    // index of a split entry's piece, -1 for a whole entry (in the backward's lists: slot of the tile)
};

// An entry that was split along its keys: pieces [first, first + n) hold its partial results.
struct __align__(16) VarSplit {
  int row0, ntok, first, n;
};

struct PlanArgs {
  const int* cu;
  const int* kv_lens;  // nullptr: packed sequences that attend to themselves
  int64_t kv_room;     // keys that a block table row has room for
  int tokens, batch, tt, causal;
  int keys;            // 1: entries are key blocks
  int tile_slots;      // 1: entries carry their slot in `part` (nothing is split)
  int split_ctas;      // > 0: entries may be split along their keys to give this many CTAs work (kv_heads items an entry)
  int kv_heads;
  VarItem* items;
  VarSplit* splits;
  int* count;          // [0] entries, [1] split entries
  uint32_t* err;
};

// Pieces that split entries can have altogether. Entries longer than a CTA's share L = work * kv_heads / CTAs become
// ceil(n / L) < 2 n / L pieces.
__host__ __device__ inline int plan_pieces(int split_ctas, int kv_heads) { return 2 * split_ctas / kv_heads + 1; }
constexpr int kPlanMinPiece = 4;  // key blocks: shorter pieces cost more in partial results than they save

// Slots that a launch reserves for `tokens` rows of `batch` sequences in tiles of tt.
__host__ __device__ inline int64_t plan_slots(int64_t tokens, int64_t batch, int64_t tt) { return tokens / tt + batch + 1; }

// Entry of `slot`, or false where the slot is empty.
__device__ __forceinline__ bool plan_item(const PlanArgs& a, int slot, VarItem& it) {
  const int step = a.keys ? kVarBlk : a.tt;
  int lo = 0, hi = a.batch + 1;  // the last i with cu[i] / step + i <= slot
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    const int base = min(max(__ldg(&a.cu[mid]), 0), a.tokens) / step + mid;
    if (base <= slot) lo = mid; else hi = mid;
  }
  if (lo == a.batch) {  // rows behind the last sequence
    const int end = min(max(__ldg(&a.cu[a.batch]), 0), a.tokens);
    const int t0 = (slot - (end / step + a.batch)) * step;
    if (t0 >= a.tokens - end) return false;
    it = {end + t0, min(step, a.tokens - end - t0), 0, 0, 0, 0, 0, slot};
    if (a.keys) it = {end + t0, min(step, a.tokens - end - t0), 0, min(step, a.tokens - end - t0), 0, 0, 0, slot};
    return true;
  }
  int r0, r1;
  bool bad;
  seq_rows(a.cu, lo, a.tokens, r0, r1, bad);
  const int t0 = (slot - (r0 / step + lo)) * step, n = r1 - r0;
  if (t0 < 0 || t0 >= n) return false;
  if (a.keys) {
    const int tiles = (n + a.tt - 1) / a.tt;
    it = {r0, n, r0 / a.tt + lo, n, t0, a.causal ? t0 / a.tt : 0, tiles, slot};
    return true;
  }
  int kv = n;
  if (a.kv_lens) {
    kv = __ldg(&a.kv_lens[lo]);
    if (kv < 0 || kv > a.kv_room) {
      atomicCAS(a.err, 0u, kErrBounds | (kKidVarAttn << 8) | (2u << 16));
      kv = kv < 0 ? 0 : static_cast<int>(a.kv_room);
    }
  }
  const int ntok = min(a.tt, n - t0), pos0 = kv - n + t0;
  const int end = a.causal ? max(pos0 + ntok, 0) : kv;
  it = {r0 + t0, ntok, a.kv_lens ? lo : r0, kv, pos0, 0, (end + kVarBlk - 1) / kVarBlk, slot};
  return true;
}

// The whole list, by one CTA of kPlanThreads threads.
__device__ __forceinline__ void build_plan(const PlanArgs& a) {
  __shared__ int hist[kPlanBuckets];
  __shared__ int warp_sum[kPlanThreads / 32];
  __shared__ unsigned long long work;             // key blocks of all entries
  __shared__ int n_live, n_split, n_part, piece;  // entries with work; ...; key blocks that an entry may have unsplit
  constexpr int kFew = 256;
  __shared__ int few[kFew];                       // lengths of the first entries with work
  static_assert(kPlanBuckets == kPlanThreads, "one bucket per thread in the scan");
  const int slots = static_cast<int>(plan_slots(a.tokens, a.batch, a.keys ? kVarBlk : a.tt));
  hist[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    work = 0;
    n_live = n_split = n_part = 0;
    piece = INT_MAX;
  }
  for (int i = threadIdx.x; i < a.batch; i += kPlanThreads) {
    int lo, hi;
    bool bad;
    seq_rows(a.cu, i, a.tokens, lo, hi, bad);
    if (bad) atomicCAS(a.err, 0u, kErrBounds | (kKidVarAttn << 8) | (1u << 16));
  }
  __syncthreads();
  if (a.split_ctas > 0) {
    for (int s = threadIdx.x; s < slots; s += kPlanThreads) {
      VarItem it;
      if (!plan_item(a, s, it) || it.b1 <= it.b0) continue;
      atomicAdd(&work, static_cast<unsigned long long>(it.b1 - it.b0));
      const int i = atomicAdd(&n_live, 1);
      if (i < kFew) few[i] = it.b1 - it.b0;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      // A CTA's even share of the work; with fewer items than CTAs, the shortest pieces that leave one per CTA (else some
      // CTAs would get two pieces, and the rest wait).
      long long l = max((static_cast<long long>(work) * a.kv_heads + a.split_ctas - 1) / a.split_ctas,
                        static_cast<long long>(kPlanMinPiece));
      const int n = n_live;
      if (n <= kFew && static_cast<int64_t>(n) * a.kv_heads < a.split_ctas)
        while (true) {
          int total = 0;
          for (int i = threadIdx.x; i < n; i += 32) total += static_cast<int>((few[i] + l - 1) / l);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
          if (static_cast<int64_t>(total) * a.kv_heads <= a.split_ctas) break;  // at the longest entry's length at the latest
          l += max(1ll, l >> 5);
        }
      if (threadIdx.x == 0) piece = static_cast<int>(min(l, static_cast<long long>(INT_MAX)));
    }
    __syncthreads();
  }
  auto pieces_of = [&](const VarItem& it) { return max((it.b1 - it.b0 - 1) / piece + 1, 1); };
  // bucket 0: the longest entries (or pieces)
  auto bucket = [](int n) { return kPlanBuckets - 1 - min(n, kPlanBuckets - 1); };
  for (int s = threadIdx.x; s < slots; s += kPlanThreads) {
    VarItem it;
    if (!plan_item(a, s, it)) continue;
    const int p = pieces_of(it);
    atomicAdd(&hist[bucket((it.b1 - it.b0) / p)], p);
  }
  __syncthreads();
  const int mine = hist[threadIdx.x];
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if ((threadIdx.x & 31) >= o) incl += v;
  }
  if ((threadIdx.x & 31) == 31) warp_sum[threadIdx.x >> 5] = incl;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < static_cast<int>(threadIdx.x >> 5); ++w) before += warp_sum[w];
  hist[threadIdx.x] = before + incl - mine;
  if (threadIdx.x == kPlanThreads - 1) a.count[0] = before + incl;
  __syncthreads();
  for (int s = threadIdx.x; s < slots; s += kPlanThreads) {
    VarItem it;
    if (!plan_item(a, s, it)) continue;
    const int n = it.b1 - it.b0, p = pieces_of(it);
    const int at = atomicAdd(&hist[bucket(n / p)], p);
    if (!a.tile_slots) it.part = -1;
    if (p == 1) {
      a.items[at] = it;
      continue;
    }
    const int first = atomicAdd(&n_part, p), b0 = it.b0;
    a.splits[atomicAdd(&n_split, 1)] = {it.row0, it.ntok, first, p};
    for (int j = 0; j < p; ++j) {
      it.b0 = b0 + static_cast<int>(static_cast<int64_t>(n) * j / p);
      it.b1 = b0 + static_cast<int>(static_cast<int64_t>(n) * (j + 1) / p);
      it.part = first + j;
      a.items[at + j] = it;
    }
  }
  if (a.split_ctas > 0) {
    __syncthreads();
    if (threadIdx.x == 0) a.count[1] = n_split;
  }
}

__global__ void __launch_bounds__(kPlanThreads) varattn_plan_kernel(const PlanArgs a) {
  ptx::grid_launch_dependents();
  build_plan(a);
}

// The k-th entry of CTA `cta` of `grid`: zigzag over the list of n entries. Returns -1 behind its end.
__device__ __forceinline__ int zigzag(int k, int cta, int grid, int n) {
  const int64_t i = static_cast<int64_t>(k) * grid + ((k & 1) ? grid - 1 - cta : cta);
  return i < n ? static_cast<int>(i) : -1;
}

}  // namespace bsk
