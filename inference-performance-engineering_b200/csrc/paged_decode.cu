// Decode attention over a paged cache: one query token per sequence, G = 1..8 query heads per KV head.
//
// Bound by memory: every key and value byte is read once for the G heads that share it. The batch's
// keys are cut into units of 64 keys of one (sequence, KV head), in that order, and the units are dealt
// to the CTAs in equal contiguous runs, so a batch with one long sequence keeps every SM as busy as an
// even one. A run's first and last piece may be part of an item; parts go to the workspace as records
// (unnormalised o, maximum, sum) that a second kernel merges in order of the keys.
//
// In a unit each of the 4 warps has 16 keys and a running softmax of its own; the warps meet once per
// piece. S = K q^T and O^T = V^T P^T as m16n8k16 products with the keys (then the head's dimensions) as
// the 16 rows and the query heads as the 8 columns, so a thread's scores and its output accumulators
// belong to the same two heads. P enters as two bf16 terms (the value cut off and the remainder), so the
// weights keep 16 bits: the products are idle anyway. Neither term of a key with a finite score is ever
// 0 or negative, nor a factor that rescales what came before 0 (kTiny is the least of them): an infinite
// value that a row sees stays infinite, with its sign, however small its weight. What a warp waits for (its
// loads, the chain from scores to weights) the other warps of the SM fill: 3 CTAs with 2 units in flight each
// against 2 with 3 measured 101.5 and 110.8 us for 160 rows behind a shared prefix, 111.0 and 114.8 for 64 rows
// of 700 to 12289 keys, in captured graphs. Measured, called alone behind a flush of L2, and as a share of a
// captured graph of 12 calls: those 64 rows 115.6 and 112.1 us (5.8 and 6.0 TB/s); 16 rows of 90 to 30001 keys
// 59.9 and 57.8 us (5.1 and 5.2 TB/s), of which the start and the merge take 8; one row of 640 keys 8.2 and
// 5.9 us, two launches and their chains of loads.
// K and V come through per-warp rings of cp.async copies, which fill keys past the sequence's end with zeros
// without reading them: what an unused row holds (NaN, say) never meets a weight of zero.
#include <algorithm>

#include "launch.h"
#include "paged_records.cuh"
#include "tensor_map.h"

namespace ipe {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kUnit = 16 * kWarps;       // keys
constexpr int kStages = 2;               // units in flight per CTA
constexpr int kStageBytes = 2 * 16 * 256;  // one warp's keys and values of a unit
constexpr int kCtasPerSm = 3;  // by registers
constexpr int kHeads = 8;                // columns of the products
constexpr int kNothing = -2;             // an item without keys
constexpr int kMergeStride = 132;        // floats; spreads a warp's 4 head pairs over the banks
constexpr size_t smem_bytes(int group) {
  return static_cast<size_t>(kStages) * kWarps * kStageBytes + static_cast<size_t>(kWarps) * group * kMergeStride * sizeof(float);
}

struct DecodeArgs {
  PagedCache c;
  const bf16* q;
  const bf16* k;
  const bf16* v;
  bf16* out;
  float* records;    // [grid][2][G][kRecord]
  int2* items;       // [sequences][kv_heads]: item_parts
  float* whole;      // null, or where rows that are not in parts go: [sequences][q_heads][kRecord], not to out
  int first;         // keys before this one are left out
  int q_heads;
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// 2^(score - base): 0 for a score of -infinity, else at least kTiny; NaN if the score is
__device__ __forceinline__ float key_weight(float score, float base) {
  float p;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(p) : "f"(exp2_approx(score * kScaleLog2 - base)), "f"(kTiny));
  return score == -INFINITY ? 0.f : p;
}
// weights cut off to bf16, and what that leaves of one, above 0 where the weight is
__device__ __forceinline__ uint32_t cut_bf16x2(float lo, float hi) {
  return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}
__device__ __forceinline__ float remainder_of(float p) {
  return p > 0.f ? fmaxf(p - __uint_as_float(__float_as_uint(p) & 0xffff0000u), kTiny) : 0.f;
}

// a sequence's keys behind the shared ones
__device__ __forceinline__ int keys_of(const DecodeArgs& a, int s) { return max(0, a.c.length(s) - a.first); }
__device__ __forceinline__ int units_of(int keys) { return (keys + kUnit - 1) / kUnit; }

// A place in the batch's sequence of units.
struct Cursor {
  int s, h, unit, units, keys;
  __device__ __forceinline__ void advance(const DecodeArgs& a) {
    if (++unit < units) return;
    unit = 0;
    if (++h < a.c.kv_heads) return;
    h = 0;
    do {
      ++s;
      keys = s < a.c.sequences ? keys_of(a, s) : kUnit;
      units = units_of(keys);
    } while (units == 0);
  }
};

__global__ void __launch_bounds__(kThreads, kCtasPerSm) paged_decode_kernel(const DecodeArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int warp_units[kWarps];
  __shared__ Cursor start;
  __shared__ float stats[kWarps][kHeads][2];
  float* merge = reinterpret_cast<float*>(smem + static_cast<size_t>(kStages) * kWarps * kStageBytes);
  const PagedCache& c = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.q_heads / c.kv_heads;
  // Behind the kernel of the shared keys, which starts when the kernels before it have finished, this one starts
  // early and has nothing to wait for.
  pdl_trigger();

  // ------------------------------------------------------------------ this CTA's run of units
  const int per = (c.sequences + kThreads - 1) / kThreads;
  const int s_lo = min(c.sequences, static_cast<int>(threadIdx.x) * per), s_hi = min(c.sequences, s_lo + per);
  int mine = 0;
  for (int s = s_lo; s < s_hi; ++s) mine += units_of(keys_of(a, s));
  int scan = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += up;
  }
  if (lane == 31) warp_units[warp] = scan;
  __syncthreads();
  int before = scan - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_units[w];
    total += warp_units[w];
  }
  const Deal deal(total * c.kv_heads, gridDim.x);
  const int u0 = deal.start(blockIdx.x), count = deal.start(blockIdx.x + 1) - u0;
  for (int s = s_lo; s < s_hi; ++s) {
    const int keys = keys_of(a, s), n = units_of(keys);
    if (n > 0 && u0 >= before * c.kv_heads && u0 < (before + n) * c.kv_heads) {
      const int r = u0 - before * c.kv_heads;
      start = Cursor{s, r / n, r % n, n, keys};
    }
    before += n;
  }
  for (int s = blockIdx.x; s < c.sequences; s += gridDim.x) {  // no keys: zeros
    if (keys_of(a, s) > 0) continue;
    for (int h = threadIdx.x; h < c.kv_heads; h += kThreads) a.items[static_cast<int64_t>(s) * c.kv_heads + h] = make_int2(kNothing, 0);
    if (a.whole) continue;
    uint4* row = reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(s) * a.q_heads * 128);
    for (int i = threadIdx.x; i < a.q_heads * 16; i += kThreads) row[i] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  if (static_cast<int>(blockIdx.x) >= deal.runs) {
    if (a.whole) pdl_wait();
    return;
  }

  // ------------------------------------------------------------------ loads
  const uint32_t ring = smem_addr(smem) + warp * kStageBytes;  // stage i at + i * kWarps * kStageBytes
  Cursor ahead = start;
  int issued = 0;
  int page = 0;  // of `ahead`
  auto look_up = [&] {
    const int key0 = ahead.unit * kUnit + warp * 16;
    page = key0 < ahead.keys ? c.page(ahead.s, a.first + key0) : 0;
  };
  auto issue = [&](int stage) {
    if (issued < count) {
      const int key0 = ahead.unit * kUnit + warp * 16;
      const int valid = ahead.keys - key0;  // keys of these 16 that exist
      const int64_t row0 = c.page_row(page, ahead.h) + (key0 & (c.page_size() - 1));
      const int chunk = lane & 15;
      const uint32_t dst = ring + stage * (kWarps * kStageBytes);
      // The 16 rows lie in one page, so every address is inside the cache; rows past the end are not read.
      const bf16* ks = a.k + (row0 + (lane >> 4)) * 128 + chunk * 8;
      const bf16* vs = a.v + (row0 + (lane >> 4)) * 128 + chunk * 8;
      const uint32_t at = (lane >> 4) * 256 + ((chunk ^ (lane >> 4)) << 4);  // row r's chunk c: r * 256 + (c ^ r % 8) * 16
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t to = dst + i * 512 + (at ^ ((2 * i & 7) << 4));
        const uint32_t bytes = (lane >> 4) + 2 * i < valid ? 16 : 0;
        cp_async16(to, ks + i * 256, bytes);
        cp_async16(to + 4096, vs + i * 256, bytes);
      }
      if (++issued < count) {
        ahead.advance(a);
        look_up();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  look_up();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue(i);

  // ------------------------------------------------------------------ products
  Cursor at = start;
  uint32_t qb[8][2];  // q^T of this piece: k = 16 kk + 2 (lane % 4) (+ 8), n = lane / 4
  float acc[8][4];    // O^T: rows 16 t + lane / 4 (+ 8), heads 2 (lane % 4) (+ 1)
  float m[2], l[2];
  bool fresh = true, first_piece = true, whole_start = true;
  const int frow = (lane & 7) + ((lane >> 3) & 1) * 8, fcol = lane >> 4;  // K fragments
  const int trow = (lane & 7) + (lane >> 4) * 8, tcol = (lane >> 3) & 1;  // V fragments, transposed
  int stage = 0;
  for (int u = 0; u < count; ++u) {
    issue(stage == 0 ? kStages - 1 : stage - 1);
    if (fresh) {
      fresh = false;
      whole_start = at.unit == 0;
      const bf16* qr = a.q + (static_cast<int64_t>(at.s) * a.q_heads + at.h * group + (lane >> 2)) * 128 + 2 * (lane & 3);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const bool real = (lane >> 2) < group;
        qb[kk][0] = real ? *reinterpret_cast<const uint32_t*>(qr + 16 * kk) : 0u;
        qb[kk][1] = real ? *reinterpret_cast<const uint32_t*>(qr + 16 * kk + 8) : 0u;
      }
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    const uint32_t ks = ring + stage * (kWarps * kStageBytes), vs = ks + 4096;
    float sc[2][4] = {};
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      uint32_t f0, f1, f2, f3;
      ldmatrix_x4(f0, f1, f2, f3, ks + frow * 256 + (((2 * kk + fcol) ^ (frow & 7)) << 4));
      mma16816(sc[kk & 1], f0, f1, f2, f3, qb[kk][0], qb[kk][1]);
    }
    const int key = at.unit * kUnit + warp * 16 + (lane >> 2);
    float s4[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s4[i] = key + (i >> 1) * 8 < at.keys ? sc[0][i] + sc[1][i] : -INFINITY;
    float keep[2], p[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float top = fmaxf(s4[e], s4[2 + e]);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      top = fmaxf(top, m[e]);
      const float base = top == -INFINITY ? 0.f : top * kScaleLog2;
      keep[e] = part_weight(m[e], base);
      m[e] = top;
      p[e] = key_weight(s4[e], base);
      p[2 + e] = key_weight(s4[2 + e], base);
      l[e] = l[e] * keep[e] + p[e] + p[2 + e];
    }
    const uint32_t b0 = transpose8x8(cut_bf16x2(p[0], p[1])), b1 = transpose8x8(cut_bf16x2(p[2], p[3]));
    const uint32_t r0 = transpose8x8(pack_bf16x2(remainder_of(p[0]), remainder_of(p[1])));
    const uint32_t r1 = transpose8x8(pack_bf16x2(remainder_of(p[2]), remainder_of(p[3])));
    if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] *= keep[i & 1];
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      uint32_t f0, f1, f2, f3;
      ldmatrix_x4_trans(f0, f1, f2, f3, vs + trow * 256 + (((2 * t + tcol) ^ (trow & 7)) << 4));
      mma16816(acc[t], f0, f1, f2, f3, b0, b1);
      mma16816(acc[t], f0, f1, f2, f3, r0, r1);
    }
    __syncwarp();
    if (++stage == kStages) stage = 0;

    if (at.unit + 1 == at.units || u + 1 == count) {  // the piece ends: the warps meet
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], o);
        const int g = 2 * (lane & 3) + e;
        if (lane < 4) {
          stats[warp][g][0] = m[e];
          stats[warp][g][1] = l[e];
        }
        float* o = merge + (warp * group + g) * kMergeStride + (lane >> 2);
        if (g < group) {
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            o[16 * t] = acc[t][e];
            o[16 * t + 8] = acc[t][2 + e];
          }
        }
      }
      __syncthreads();
      const bool whole = whole_start && at.unit + 1 == at.units;
      const int slot = first_piece ? 0 : 1;
      first_piece = false;
      if (whole_start && threadIdx.x == 0)
        a.items[static_cast<int64_t>(at.s) * c.kv_heads + at.h] =
            item_parts(deal, u0 + u - at.unit, at.units, blockIdx.x);
      for (int g = 0; g < group; ++g) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stats[w][g][0]);
        const float base = top == -INFINITY ? 0.f : top * kScaleLog2;
        float sum = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float e = part_weight(stats[w][g][0], base);
          sum += e * stats[w][g][1];
          o += e * merge[(w * group + g) * kMergeStride + threadIdx.x];
        }
        const int64_t row = static_cast<int64_t>(at.s) * a.q_heads + at.h * group + g;
        if (whole && !a.whole) {
          a.out[row * 128 + threadIdx.x] = __float2bfloat16_rn(o / sum);
        } else {
          float* rec = whole ? a.whole + row * kRecord
                             : a.records + ((static_cast<int64_t>(blockIdx.x) * 2 + slot) * group + g) * kRecord;
          rec[threadIdx.x] = o;
          if (threadIdx.x == 0) {
            rec[128] = top;
            rec[129] = sum;
          }
        }
      }
      __syncthreads();
      fresh = true;
    }
    if (u + 1 < count) at.advance(a);
  }
  // beside the kernel of the shared keys: whoever waits for this grid then waits for that one too
  if (a.whole) pdl_wait();
}

// The parts of a row, none where the sequence has no keys or the row is whole.
__device__ __forceinline__ Parts decode_parts(const DecodeArgs& a, int s, int head) {
  const int group = a.q_heads / a.c.kv_heads;
  const int2 item = __ldcg(a.items + static_cast<int64_t>(s) * a.c.kv_heads + head / group);
  Parts p;
  p.rows(a.records, head % group, group, item);
  if (item.x < 0) p.none();
  if (item.x == kWhole && a.whole) p.single(a.whole + (static_cast<int64_t>(s) * a.q_heads + head) * kRecord);
  return p;
}

// Records of a row that a merge loads at once. Few rows wait for their chain of loads, so the more the better (12
// instead of 8 or 4: one sequence of 640 keys 6.1, 6.5, 6.7 us, 16 of 90 to 30001 keys 57.7, 58.2, 59.7); where there
// are more rows than warps at a time, the registers that they take cost more than the wait (160 sequences behind a
// shared prefix, 5120 rows: 102.4 us with 12, 101.3 with 8, 98.9 with 4).
constexpr int kFewRows = 12, kManyRows = 4;
constexpr int kManyFrom = 16;  // rows per SM

// One warp per (sequence, query head) in parts.
__global__ void __launch_bounds__(kThreads) paged_decode_merge_kernel(const DecodeArgs a) {
  const int row = static_cast<int>(blockIdx.x * kWarps + (threadIdx.x >> 5));
  if (row >= a.c.sequences * a.q_heads) return;
  const int s = row / a.q_heads, head = row - s * a.q_heads;
  pdl_wait();
  const Parts parts[1] = {decode_parts(a, s, head)};
  if (parts[0].count() > 0) join_parts<kFewRows>(parts, a.out + static_cast<int64_t>(row) * 128);
}

// One warp per (sequence, query head): the parts of the shared keys and those of the sequence's own.
template <int kTogether>
__global__ void __launch_bounds__(kThreads) shared_prefix_merge_kernel(const DecodeArgs a, const SharedKeys shared) {
  const int row = static_cast<int>(blockIdx.x * kWarps + (threadIdx.x >> 5)), lane = threadIdx.x & 31;
  if (row >= a.c.sequences * a.q_heads) return;
  const int s = row / a.q_heads, head = row - s * a.q_heads;
  const int group = a.q_heads / a.c.kv_heads, per_block = 2 * shared.per_tile;
  const int block = s / per_block, in_block = s % per_block, tile = in_block / shared.per_tile;
  bf16* out = a.out + static_cast<int64_t>(row) * 128;
  const bool empty = a.c.length(s) == 0;
  pdl_wait();
  if (empty) {
    *reinterpret_cast<uint2*>(out + lane * 4) = make_uint2(0u, 0u);
    return;
  }
  const int2 item = __ldcg(shared.items + static_cast<int64_t>(block) * a.c.kv_heads + head / group);
  Parts parts[2];
  parts[0].blocks(shared.records, tile * 128 + (in_block - tile * shared.per_tile) * group + head % group, item);
  // whole (or what a kernel that gave up on a wait left)
  if (item.x < 0 || item.y >= shared.ctas || item.y < item.x >> 1) parts[0].single(shared.whole + static_cast<int64_t>(row) * kRecord);
  parts[1] = decode_parts(a, s, head);
  join_parts<kTogether>(parts, out);
}

std::atomic<uint64_t> shared_memory_allowed{0};  // of paged_decode_kernel, by device

// CTAs per SM: the third fits beside the others' shared memory up to 5 query heads per KV head
int ctas_per_sm(int group) { return group <= 5 ? kCtasPerSm : 2; }

size_t items_bytes(int64_t items) { return (static_cast<size_t>(items) * sizeof(int2) + 255) / 256 * 256; }

DecodeArgs decode_args(const PagedCache& c, const void* q, const void* k_pages, const void* v_pages, void* out, int q_heads,
                       void* workspace) {
  DecodeArgs a{};
  a.c = c;
  a.q = static_cast<const bf16*>(q);
  a.k = static_cast<const bf16*>(k_pages);
  a.v = static_cast<const bf16*>(v_pages);
  a.out = static_cast<bf16*>(out);
  a.items = static_cast<int2*>(workspace);
  a.records = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) +
                                       items_bytes(static_cast<int64_t>(c.sequences) * c.kv_heads));
  a.q_heads = q_heads;
  return a;
}

int decode_grid(const PagedCache& c, int q_heads) {
  const int64_t capacity = static_cast<int64_t>(c.max_pages - c.prefix_count) << c.page_shift;
  const int64_t most = static_cast<int64_t>(c.sequences) * c.kv_heads * ((capacity + kUnit - 1) / kUnit);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ctas_per_sm(q_heads / c.kv_heads) * sm_count(), most)));
}

dim3 merge_grid(const PagedCache& c, int q_heads) {
  return dim3(static_cast<unsigned>((static_cast<int64_t>(c.sequences) * q_heads + kWarps - 1) / kWarps));
}

}  // namespace

size_t paged_decode_workspace_bytes(int sequences, int q_heads, int kv_heads) {
  return items_bytes(static_cast<int64_t>(sequences) * kv_heads) + static_cast<size_t>(ctas_per_sm(q_heads / kv_heads) * sm_count()) * 2 * (q_heads / kv_heads) * kRecord * sizeof(float);
}

cudaError_t launch_paged_decode(const PagedCache& c, const void* q, const void* k_pages, const void* v_pages, void* out,
                                int q_heads, void* workspace, cudaStream_t stream) {
  cudaError_t e = allow_shared_memory(paged_decode_kernel, smem_bytes(kHeads), &shared_memory_allowed);
  if (e != cudaSuccess) return e;
  const DecodeArgs a = decode_args(c, q, k_pages, v_pages, out, q_heads, workspace);
  const int grid = decode_grid(c, q_heads);
  paged_decode_kernel<<<grid, kThreads, smem_bytes(q_heads / c.kv_heads), stream>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess || (c.max_pages << c.page_shift) <= kUnit) return e;  // one unit per item: nothing to merge
  return launch_pdl(paged_decode_merge_kernel, merge_grid(c, q_heads), dim3(kThreads), 0, stream, a);
}

size_t shared_prefix_workspace_bytes(const PagedCache& c, int q_heads) {
  const size_t rows = static_cast<size_t>(c.sequences) * q_heads * kRecord * sizeof(float);
  const SharedKeys plan = shared_keys_plan(c, q_heads);
  return paged_decode_workspace_bytes(c.sequences, q_heads, c.kv_heads) + items_bytes(plan.items_count) + 2 * rows +
         static_cast<size_t>(plan.ctas) * 2 * kBlockRecord * sizeof(float);
}

cudaError_t launch_shared_prefix(const PagedCache& c, const void* q, const void* k_pages, const void* v_pages, void* out,
                                 int q_heads, void* workspace, cudaStream_t stream) {
  if (c.prefix_count == 0) return launch_paged_decode(c, q, k_pages, v_pages, out, q_heads, workspace, stream);
  cudaError_t e = allow_shared_memory(paged_decode_kernel, smem_bytes(kHeads), &shared_memory_allowed);
  if (e != cudaSuccess) return e;
  const size_t rows = static_cast<size_t>(c.sequences) * q_heads * kRecord;
  SharedKeys shared = shared_keys_plan(c, q_heads);
  DecodeArgs a = decode_args(c, q, k_pages, v_pages, out, q_heads, workspace);
  unsigned char* behind = static_cast<unsigned char*>(workspace) + paged_decode_workspace_bytes(c.sequences, q_heads, c.kv_heads);
  shared.items = reinterpret_cast<int2*>(behind);
  shared.whole = reinterpret_cast<float*>(behind + items_bytes(shared.items_count));
  a.whole = shared.whole + rows;
  shared.records = a.whole + rows;
  a.first = c.prefix_count << c.page_shift;
  e = launch_shared_keys(c, q, k_pages, v_pages, q_heads, shared, stream);
  if (e != cudaSuccess) return e;
  // the sequences' own keys: nothing of it waits for the kernel before, so its CTAs start as that one's end
  const int grid = decode_grid(c, q_heads);
  e = launch_pdl(paged_decode_kernel, dim3(grid), dim3(kThreads), smem_bytes(q_heads / c.kv_heads), stream, a);
  if (e != cudaSuccess) return e;
  const bool many = static_cast<int64_t>(c.sequences) * q_heads > kManyFrom * sm_count();
  return launch_pdl(many ? shared_prefix_merge_kernel<kManyRows> : shared_prefix_merge_kernel<kFewRows>, merge_grid(c, q_heads),
                    dim3(kThreads), 0, stream, a, shared);
}

}  // namespace ipe
