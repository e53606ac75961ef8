// Parts of softmax rows, and how they come together.
//
// The attention kernels over a paged cache deal their units of work (a number of keys of one item: a
// sequence's KV head, or a block of query rows) to CTAs in equal contiguous runs. A run that begins or
// ends inside an item writes its part of each of the item's rows as a record: o = sum p v, the maximum m
// the weights p = 2^((s - m) c) refer to, and their sum. Parts with (o, m, l) join as
// o = sum_i 2^((m_i - M) c) o_i, likewise l, M the largest m: in order of the keys, so a call's bits do
// not depend on which part came first.
#pragma once

#include "paged.cuh"

namespace ipe {

constexpr int kRecord = 132;  // floats: o[128], maximum, sum, 2 unused
constexpr float kScaleLog2 = 0.08838834764831845f * 1.4426950408889634f;  // c: 128^-0.5 * log2(e)

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The units are dealt to `runs` CTAs, none of them without one; run r begins with unit run_start(r).
__device__ __forceinline__ int runs_of(int64_t units, int ctas) { return units < ctas ? static_cast<int>(units) : ctas; }
__device__ __forceinline__ int64_t run_start(int64_t units, int run, int runs) { return units * run / max(runs, 1); }

// The records of one row: those of runs lo..hi at base[run][slot][rows][kRecord]. A run has two slots: 0
// for the piece it begins with, 1 for another that it ends with.
struct Parts {
  const float* base;
  int64_t row;
  int rows, lo, hi, slot_lo;

  // the parts of a row of the item that owns units first .. first + n - 1
  __device__ __forceinline__ void find(int64_t first, int64_t n, int64_t units, int ctas) {
    const int runs = runs_of(units, ctas);
    lo = static_cast<int>(((first + 1) * runs - 1) / units);
    hi = static_cast<int>(((first + n) * runs - 1) / units);
    slot_lo = run_start(units, lo, runs) == first ? 0 : 1;
  }
  __device__ __forceinline__ void single(const float* record) { *this = Parts{record, 0, 0, 0, 0, 0}; }
  __device__ __forceinline__ void none() { *this = Parts{nullptr, 0, 0, 0, -1, 0}; }
  __device__ __forceinline__ const float* at(int run) const {
    return base + ((static_cast<int64_t>(run) * 2 + (run == lo ? slot_lo : 0)) * rows + row) * kRecord;
  }
};

// Joins the parts in order, by a whole warp; lane l writes elements 4l..4l+3 of the bf16 row `out`.
template <int N>
__device__ __forceinline__ void join_parts(const Parts (&parts)[N], bf16* out) {
  const int lane = threadIdx.x & 31;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i)
    for (int run = parts[i].lo + lane; run <= parts[i].hi; run += 32) top = fmaxf(top, __ldcg(parts[i].at(run) + 128));
  top = warp_max(top);
  const float base = top == -INFINITY ? 0.f : top * kScaleLog2;
  float sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll 4
    for (int run = parts[i].lo; run <= parts[i].hi; ++run) {
      const float* rec = parts[i].at(run);
      const float4 x = __ldcg(reinterpret_cast<const float4*>(rec) + lane);
      const float e = exp2_approx(__ldcg(rec + 128) * kScaleLog2 - base);
      sum += e * __ldcg(rec + 129);
      o.x += e * x.x;
      o.y += e * x.y;
      o.z += e * x.z;
      o.w += e * x.w;
    }
  }
  const float inv = 1.f / sum;
  *reinterpret_cast<uint2*>(out + lane * 4) =
      make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
}

// How the kernel of the shared keys cuts its work: blocks of 2 * per_tile sequences' query rows (two tiles of 128
// rows), each with `tiles` units per KV head.
struct SharedKeys {
  float* records;  // [ctas][2][256][kRecord]
  float* whole;    // [sequences][q_heads][kRecord]
  int64_t units;
  int per_tile, tiles, ctas;
};

}  // namespace ipe
