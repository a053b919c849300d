// A serving step's bookkeeping for a paged cache, built on the device from the requests' lengths, for sm_100a: where each new
// token goes (slot, position), which free pages the requests take (block table entries), offsets and lengths for attention.
//
// With kv[i] cached and n[i] new tokens of request i and P rows a page:
//     cu[i] = sum of n before i;   have = ceil(kv / P), need = ceil((kv + n) / P);   first[i] = sum of (need - have) before i
// and new token t of request i stands at position p = kv[i] + t in the request's page c = p / P. That page is there (c < have),
// or it is the (first[i] + c - have)-th page taken from the end of the stack of free pages. Each page taken starts with exactly
// one new token (p = c P), which writes its table entry: so the work is dealt out by tokens, and a long prompt is spread over
// the CTAs. Every CTA scans the lengths by itself, a chunk of kKvPlanThreads requests at a time, up to the last request that
// its tokens belong to; CTA 0 goes through all of them and writes what there is per request. One launch, no workspace, no
// order between CTAs.
//
// Bound: latency: lengths -> two scans -> search -> page -> slot, 12 bytes a token. 3.8 us in a graph for 64 requests of one token
// and 4.8 for 200 requests of 1 .. 499 (16658 tokens), where elementary operations take 390; the call on the host takes 7.
#pragma once

#include "ptx_sm100.cuh"

namespace bsk {

constexpr uint32_t kKidKvPlan = 13;
constexpr int kKvPlanThreads = 512;
constexpr int kKvPlanTokens = 1024;  // rows of a CTA

struct KvPlanArgs {
  const int* kv_lens;     // [batch] cached tokens
  const int* new_lens;    // [batch] new tokens
  int* table;             // [batch, width], entries of opened pages are written
  int64_t table_stride;
  const int* free_pages;  // stack, the first *free_count are free
  const int* free_count;
  int64_t* slots;         // [tokens], -1: no slot
  int* positions;         // [tokens]
  int* cu;                // [batch + 1]
  int* lens_out;          // [batch]
  int* free_out;          // [1]
  int batch, width, num_free, page, tokens;
  uint32_t* err;
};

__device__ __forceinline__ void kv_plan_flag(uint32_t* err, uint32_t site) {
  atomicCAS(err, 0u, kErrBounds | (kKidKvPlan << 8) | (site << 16));
}

// Inclusive sum over the CTA's threads; `total` is that of all.
__device__ __forceinline__ int64_t cta_scan(int64_t v, int64_t* warp_sums, int64_t& total) {
  constexpr int kWarps = kKvPlanThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();  // the sums of the scan before have been read
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const int64_t s = warp_sums[w];
    before += w < warp ? s : 0;
    total += s;
  }
  return before + v;
}

static __global__ void __launch_bounds__(kKvPlanThreads) kv_plan_kernel(const KvPlanArgs a) {
  __shared__ int64_t warp_sums[kKvPlanThreads / 32];
  __shared__ int s_cu[kKvPlanThreads + 1], s_kv[kKvPlanThreads], s_have[kKvPlanThreads];
  __shared__ int64_t s_first[kKvPlanThreads];  // pages taken by the requests before, less `have`
  const bool lead = blockIdx.x == 0;
  const int row0 = static_cast<int>(blockIdx.x) * kKvPlanTokens, row1 = static_cast<int>(min(static_cast<int64_t>(row0) + kKvPlanTokens, static_cast<int64_t>(a.tokens)));
  const int64_t room = min(static_cast<int64_t>(a.width) * a.page, static_cast<int64_t>(INT32_MAX));
  const int stated = __ldg(a.free_count);
  const int n_free = min(max(stated, 0), a.num_free);
  if (lead && threadIdx.x == 0) {
    if (stated != n_free) kv_plan_flag(a.err, 1);
    a.cu[0] = 0;
  }
  int64_t tokens_before = 0, pages_before = 0;
  int done = row0;  // rows of this CTA up to here are written
  for (int c0 = 0; c0 < a.batch && (lead || done < row1); c0 += kKvPlanThreads) {
    const int i = c0 + threadIdx.x, count = min(kKvPlanThreads, a.batch - c0);
    int kv = 0, n = 0;
    if (i < a.batch) {
      kv = __ldg(a.kv_lens + i);
      n = __ldg(a.new_lens + i);
      if (lead && (kv < 0 || n < 0 || static_cast<int64_t>(max(kv, 0)) + n > room)) kv_plan_flag(a.err, 2);
      kv = static_cast<int>(min(static_cast<int64_t>(max(kv, 0)), room));
      n = max(n, 0);
    }
    int64_t total, pages;
    const int64_t sum = tokens_before + cta_scan(n, warp_sums, total);
    // rows behind the last one are left out
    const int end = static_cast<int>(min(sum, static_cast<int64_t>(a.tokens)));
    const int begin = static_cast<int>(min(sum - n, static_cast<int64_t>(a.tokens)));
    const int after = static_cast<int>(min(static_cast<int64_t>(kv) + (end - begin), room));
    const int have = kv / a.page + (kv % a.page != 0), need = after / a.page + (after % a.page != 0);
    const int64_t taken = pages_before + cta_scan(need - have, warp_sums, pages);
    if (i < a.batch) {
      s_cu[threadIdx.x] = begin;
      s_kv[threadIdx.x] = kv;
      s_have[threadIdx.x] = have;
      s_first[threadIdx.x] = taken - (need - have) - have;
      if (lead) {
        a.cu[i + 1] = end;
        a.lens_out[i] = after;
      }
    }
    tokens_before += total;
    pages_before += pages;
    const int chunk_end = static_cast<int>(min(tokens_before, static_cast<int64_t>(a.tokens)));
    __syncthreads();
    const int stop = min(row1, chunk_end);
    for (uint32_t x = done + threadIdx.x; x < static_cast<uint32_t>(stop); x += kKvPlanThreads) {  // (passes 2^31 near the last row)
      const int row = static_cast<int>(x);
      int lo = 0, hi = count;  // the last request that begins at or before the row (those without tokens begin where the next does)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= row) lo = mid; else hi = mid;
      }
      const int64_t at = static_cast<int64_t>(s_kv[lo]) + (row - s_cu[lo]);
      int page = -1;
      if (at < room) {
        const int place = static_cast<int>(at), cell = place / a.page;
        int* entry = a.table + (static_cast<int64_t>(c0) + lo) * a.table_stride + cell;
        if (cell < s_have[lo]) {
          page = *entry;
        } else {
          const int64_t k = s_first[lo] + cell;
          if (k < n_free) page = __ldg(a.free_pages + (n_free - 1 - k));
          if (place % a.page == 0) *entry = page;
        }
        if (page < 0) kv_plan_flag(a.err, 3);  // no page is left, or the request's own was given back
        a.slots[row] = page < 0 ? -1 : static_cast<int64_t>(page) * a.page + place % a.page;
      } else {
        a.slots[row] = -1;  // (reported above)
      }
      a.positions[row] = static_cast<int>(min(at, static_cast<int64_t>(INT32_MAX)));
    }
    done = max(done, stop);
    __syncthreads();
  }
  for (uint32_t x = done + threadIdx.x; x < static_cast<uint32_t>(row1); x += kKvPlanThreads) {  // padding
    a.slots[x] = -1;
    a.positions[x] = 0;
  }
  if (lead && threadIdx.x == 0) {
    if (tokens_before > a.tokens) kv_plan_flag(a.err, 4);
    a.free_out[0] = static_cast<int>(max(n_free - pages_before, int64_t{0}));
  }
}

}  // namespace bsk
