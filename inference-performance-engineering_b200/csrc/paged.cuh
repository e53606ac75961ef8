// The paged K/V cache as the kernels see it, and the lookups they share.
//
// Pages are bf16 [num_pages][kv_heads][page_size][128], keys and values apart; position p of
// sequence s is row p % page_size of page page_table[s][p / page_size]. page_size is 16, 32, 64 or
// 128, so a page's rows of one head are one contiguous run. New tokens are ragged: sequence s brings
// rows cu_tokens[s] .. cu_tokens[s + 1] - 1, the last ones of its lengths[s] positions. All of these
// integers live on the device, so a captured launch replays with other lengths; what the host cannot
// check, the kernels do: no value of theirs is used as an address before it was compared with its
// bound.
#pragma once

#include "common.cuh"

namespace ipe {

constexpr int kErrPage = 5;  // a page ID outside the cache

struct PagedCache {
  const int* page_table;    // [sequences][max_pages]
  const int* lengths;       // [sequences], the new tokens included
  const int* cu_tokens;     // [sequences + 1], or null: one token per sequence
  const int* prefix_pages;  // pages of the positions every sequence shares, or null
  int prefix_count;         // pages in prefix_pages; page_table is not read for those positions
  int sequences;
  int max_pages;
  int page_shift;  // log2(page_size)
  int kv_heads;
  int num_pages;
  int* err;

  __device__ __forceinline__ int page_size() const { return 1 << page_shift; }
  // a sequence's length, 0 (and device error 2) where it does not fit its row of the page table
  __device__ __forceinline__ int length(int s) const { return checked_length(__ldg(lengths + s)); }
  __device__ __forceinline__ int checked_length(int n) const {
    if (n >= 0 && n <= (static_cast<int64_t>(max_pages) << page_shift)) return n;
    report(err, kErrPositionRange);
    return 0;
  }
  // what the tables say of a position below length(s), not looked at
  __device__ __forceinline__ int page_id(int s, int position) const {
    const int j = position >> page_shift;
    return j < prefix_count ? __ldg(prefix_pages + j) : __ldg(page_table + static_cast<int64_t>(s) * max_pages + j);
  }
  // a page outside the cache sets device error 5 and reads as page 0, so nothing outside the cache is touched
  __device__ __forceinline__ int checked(int id) const {
    if (static_cast<unsigned>(id) < static_cast<unsigned>(num_pages)) return id;
    report(err, kErrPage);
    return 0;
  }
  __device__ __forceinline__ int page(int s, int position) const { return checked(page_id(s, position)); }
  // first row (of 128 elements) of a page's head
  __device__ __forceinline__ int64_t page_row(int page_id, int kv_head) const {
    return (static_cast<int64_t>(page_id) * kv_heads + kv_head) << page_shift;
  }
};

// Pairs of fp32 in one 64-bit register: two operations per instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float* lo, float* hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(*lo), "=f"(*hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// The sequence that brings token `t`: the last s with cu_tokens[s] <= t, if t < cu_tokens[s + 1]; -1
// for a row behind the last sequence. Called by a whole warp: each round probes 31 places between the
// bounds and leaves at most ceil(range / 32) of them, so it ends whatever the array holds.
__device__ __forceinline__ int find_sequence(const int* __restrict__ cu_tokens, int sequences, int t) {
  const int lane = threadIdx.x & 31;
  int low = 0, high = sequences + 1;  // cu_tokens[low] <= t as far as known, cu_tokens[high] > t
  while (high - low > 1) {
    const int step = (high - low + 31) >> 5;
    const int probe = low + lane * step;
    const bool below = lane > 0 && probe < high && __ldg(cu_tokens + probe) <= t;
    const int passed = __popc(__ballot_sync(0xffffffffu, below));
    const int next = low + passed * step;
    high = min(high, passed == 31 ? high : next + step);
    low = next;
  }
  if (low >= sequences) return -1;
  return __ldg(cu_tokens + low) <= t && t < __ldg(cu_tokens + low + 1) ? low : -1;
}

}  // namespace ipe
