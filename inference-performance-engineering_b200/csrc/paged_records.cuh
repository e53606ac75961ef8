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

constexpr float kTiny = 1.17549435e-38f;  // 2^-126, the least normal number, of bf16 too

// What a part with maximum m counts beside `base` (of the largest one), at least kTiny: infinite values stay infinite.
// A part without a key (m = -infinity) holds zeros.
__device__ __forceinline__ float part_weight(float m, float base) { return fmaxf(exp2_approx(m * kScaleLog2 - base), kTiny); }

// Units dealt to CTAs in contiguous runs, none of them without a unit and none with over one more than another.
struct Deal {
  int runs, each, more;  // the first `more` runs have each + 1 units

  __device__ __forceinline__ Deal(int units, int ctas) : runs(min(units, ctas)), each(units / max(runs, 1)), more(units - each * runs) {}
  // first unit of a run; a CTA without one begins where the units end
  __device__ __forceinline__ int start(int run) const { return min(run, runs) * each + min(run, more); }
  __device__ __forceinline__ int run_of(int unit) const {
    const int longer = more * (each + 1);
    return unit < longer ? unit / (each + 1) : more + (unit - longer) / max(each, 1);
  }
};

// Which runs hold the parts of an item: first run * 2 + its slot (a run has two: 0 for the piece that it
// begins with, 1 for another that it ends with; every later run begins inside the item) and last run.
// Written by the CTA that has the item's first unit; an item that one run has whole says so.
constexpr int kWhole = -1;
__device__ __forceinline__ int2 item_parts(const Deal& deal, int first_unit, int n, int run) {
  const int last = deal.run_of(first_unit + n - 1);
  if (last == run) return make_int2(kWhole, 0);
  return make_int2(run * 2 + (deal.start(run) == first_unit ? 0 : 1), last);
}

// The records of one row of an item. The decode kernel writes a row's 132 floats together. The kernels with a
// row per thread write blocks of 256 rows, 32 bytes of each row side by side (whole sectors for the reads
// here, few lines for a store there): float o[16][256][8], m[256], sum[256].
constexpr int kBlockRows = 256;
constexpr int kBlockRecord = kBlockRows * 130;  // floats
__device__ __forceinline__ int block_vector(int v) { return (v >> 1) * (kBlockRows * 8) + (v & 1) * 4; }  // of a row's 32
struct Parts {
  const float* base;  // of the row in record slot 0
  int first, last;    // first run * 2 + slot, last run
  int slot_stride, vector, m, sum;  // `vector`: of this lane's four elements

  __device__ __forceinline__ int count() const { return last - (first >> 1) + 1; }
  __device__ __forceinline__ const float* at(int i) const {
    return base + static_cast<int64_t>(i == 0 ? first : ((first >> 1) + i) * 2) * slot_stride;
  }
  __device__ __forceinline__ void rows(const float* records, int row, int rows_per_slot, int2 item) {
    const int lane = threadIdx.x & 31;
    *this = Parts{records + static_cast<int64_t>(row) * kRecord, item.x, item.y, rows_per_slot * kRecord, lane * 4, 128, 129};
  }
  __device__ __forceinline__ void blocks(const float* records, int row, int2 item) {
    const int lane = threadIdx.x & 31;
    *this = Parts{records + row * 8, item.x, item.y, kBlockRecord, block_vector(lane), kBlockRows * 128 - row * 7,
                  kBlockRows * 129 - row * 7};
  }
  __device__ __forceinline__ void single(const float* record) { rows(record, 0, 0, make_int2(0, 0)); }
  __device__ __forceinline__ void none() { rows(nullptr, 0, 0, make_int2(0, -1)); }
};

// Joins the parts in order, by a whole warp; lane l writes elements 4l..4l+3 of the bf16 row `out`. Up to
// kTogether records are loaded at once; a later group's maximum rescales what the groups before gave.
template <int kTogether, int N>
__device__ __forceinline__ void join_parts(const Parts (&parts)[N], bf16* out) {
  float top = -INFINITY, sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int n = parts[i].count();
    for (int k0 = 0; k0 < n; k0 += kTogether) {
      float4 x[kTogether];
      float m[kTogether], l[kTogether], most = top;
#pragma unroll
      for (int k = 0; k < kTogether; ++k) {
        m[k] = -INFINITY;
        l[k] = 0.f;
        x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k0 + k < n) {
          const float* rec = parts[i].at(k0 + k);
          x[k] = __ldcg(reinterpret_cast<const float4*>(rec + parts[i].vector));
          m[k] = __ldcg(rec + parts[i].m);
          l[k] = __ldcg(rec + parts[i].sum);
        }
      }
#pragma unroll
      for (int k = 0; k < kTogether; ++k) most = fmaxf(most, m[k]);
      const float base = most == -INFINITY ? 0.f : most * kScaleLog2;
      const float keep = part_weight(top, base);
      top = most;
      sum *= keep;
      o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
#pragma unroll
      for (int k = 0; k < kTogether; ++k) {
        const float e = part_weight(m[k], base);
        sum += e * l[k];
        o.x += e * x[k].x;
        o.y += e * x[k].y;
        o.z += e * x[k].z;
        o.w += e * x[k].w;
      }
    }
  }
  const float inv = 1.f / sum;
  *reinterpret_cast<uint2*>(out + (threadIdx.x & 31) * 4) =
      make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
}

// How the kernel of the shared keys cuts its work: blocks of 2 * per_tile sequences' query rows (two tiles of 128
// rows), each with `tiles` units per KV head.
struct SharedKeys {
  float* records;  // [ctas][2][kBlockRecord]
  float* whole;    // [sequences][q_heads][kRecord]
  int2* items;     // [blocks][kv_heads]
  int64_t units;
  int64_t items_count;
  int per_tile, tiles, ctas;
};

}  // namespace ipe
