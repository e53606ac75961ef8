// q/k RMSNorm per head, split-half rotation at each token's own position, and the append of keys and
// values to a paged cache, for a ragged batch of new tokens.
//
// y = w * x * rsqrt(mean(x^2) + eps); o_d = y_d cos_d + r_d sin_d with r_d = -y_{d+64} for d < 64 and
// y_{d-64} above, all in fp32 and rounded to bf16 once (the contiguous append rounds at the reference's
// own points instead: it has to match the reference's bits, this one the formula).
//
// Bound by memory: 256 bytes in and out per head slot. A warp has a few consecutive tokens, or a share of one
// token's slots where there are few: enough warps to fill the GPU once, so the chain of lookups that a place
// takes (sequence, length, page; a lane per token) is paid once per warp and behind the first rows' loads.
// 16 lanes per row, each with elements 4j..4j+3 and 64+4j..64+4j+3, so the rotation stays in the lane; a token's
// cosines and sines stay in registers over its rows.
#include <algorithm>

#include "launch.h"
#include "paged.cuh"
#include "tensor_map.h"

namespace ipe {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kAhead = 2;       // pairs of rows in flight
constexpr int kMostSplit = 8;   // warps that share a token's slots
constexpr int kMostTokens = 32;  // of a warp

__device__ __forceinline__ void unpack4(const uint2& v, float* f) {
  f[0] = __uint_as_float(v.x << 16);
  f[1] = __uint_as_float(v.x & 0xffff0000u);
  f[2] = __uint_as_float(v.y << 16);
  f[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void load4(const bf16* p, float* f) { unpack4(__ldg(reinterpret_cast<const uint2*>(p)), f); }
__device__ __forceinline__ void load4(const float* p, float* f) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  f[0] = a.x;
  f[1] = a.y;
  f[2] = a.z;
  f[3] = a.w;
}

// The sequence that brings token `t`, or -1: each lane for its own token.
__device__ __forceinline__ int sequence_of(const PagedCache& c, int t) {
  int low = 0, high = c.sequences;  // the last s in [low, high) with cu_tokens[s] <= t
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (__ldg(c.cu_tokens + mid) <= t) low = mid;
    else high = mid;
  }
  return __ldg(c.cu_tokens + low) <= t && t < __ldg(c.cu_tokens + low + 1) ? low : -1;
}

// What a lane finds out of its token: -1 where nothing of it is written.
struct Place {
  int position;
  int stored;   // whether its page is one
  int64_t row;  // cache row of KV head 0
};

__device__ __forceinline__ Place place_of(const PagedCache& c, int s, int t, int64_t table_rows) {
  Place p{-1, 0, 0};
  if (s < 0) return p;  // a row behind the last sequence: left as it is
  const int position = c.length(s) - (__ldg(c.cu_tokens + s + 1) - t);
  if (position < 0 || position >= table_rows) {  // more new tokens than positions, or past the rotation tables
    report(c.err, kErrPositionRange);
    return p;
  }
  const int id = __ldg(c.page_table + static_cast<int64_t>(s) * c.max_pages + (position >> c.page_shift));
  p.position = position;
  p.stored = static_cast<unsigned>(id) < static_cast<unsigned>(c.num_pages);
  if (!p.stored) report(c.err, kErrPage);
  p.row = c.page_row(p.stored ? id : 0, 0) + (position & (c.page_size() - 1));
  return p;
}

struct Row {
  uint2 lo, hi;  // a lane's elements of a row: 4j.., 64 + 4j..
};

template <typename Table>
__global__ void __launch_bounds__(kThreads, 4) paged_append_kernel(const PagedCache c, const bf16* __restrict__ qkv,
                                                                   int tokens, int per_warp, int split, int q_heads,
                                                                   const bf16* __restrict__ q_norm,
                                                                   const bf16* __restrict__ k_norm,
                                                                   const Table* __restrict__ cos_t,
                                                                   const Table* __restrict__ sin_t, int64_t table_rows,
                                                                   bf16* __restrict__ q_out, bf16* __restrict__ k_pages,
                                                                   bf16* __restrict__ v_pages, float eps) {
  const int warp = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int t0 = warp / split * per_warp, mine = min(per_warp, tokens - t0);
  if (mine <= 0) return;
  const int slots = q_heads + 2 * c.kv_heads, share = (slots + split - 1) / split;
  const int slot0 = warp % split * share, slot1 = min(slots, slot0 + share);
  const int team = lane >> 4, d0 = (lane & 15) * 4;
  const bf16* src = qkv + static_cast<int64_t>(t0) * slots * 128 + d0;
  Row raw[kAhead];
  auto load = [&](int token, int slot) {  // this lane's part of row `slot + team`
    Row x{make_uint2(0, 0), make_uint2(0, 0)};
    if (token < mine && slot + team < slot1) {
      const bf16* p = src + (token * slots + slot + team) * 128;
      x.lo = __ldcs(reinterpret_cast<const uint2*>(p));
      x.hi = __ldcs(reinterpret_cast<const uint2*>(p + 64));
    }
    return x;
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) raw[u] = load(0, slot0 + 2 * u);
  Place own{-1, 0, 0};
  if (per_warp == 1)
    own = place_of(c, find_sequence(c.cu_tokens, c.sequences, t0), t0, table_rows);
  else if (lane < mine)
    own = place_of(c, sequence_of(c, t0 + lane), t0 + lane, table_rows);
  const uint2 wq_lo = __ldg(reinterpret_cast<const uint2*>(q_norm + d0)), wq_hi = __ldg(reinterpret_cast<const uint2*>(q_norm + 64 + d0));
  const uint2 wk_lo = __ldg(reinterpret_cast<const uint2*>(k_norm + d0)), wk_hi = __ldg(reinterpret_cast<const uint2*>(k_norm + 64 + d0));

  for (int token = 0; token < mine; ++token) {
    const int position = __shfl_sync(0xffffffffu, own.position, token);
    const bool stored = __shfl_sync(0xffffffffu, own.stored, token);
    const int64_t row0 = __shfl_sync(0xffffffffu, own.row, token);
    float cos_lo[4], cos_hi[4], sin_lo[4], sin_hi[4];
    const int64_t at = static_cast<int64_t>(max(position, 0)) * 128 + d0;
    load4(cos_t + at, cos_lo);
    load4(cos_t + at + 64, cos_hi);
    load4(sin_t + at, sin_lo);
    load4(sin_t + at + 64, sin_hi);
    for (int base = slot0; base < slot1; base += 2 * kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const Row row = raw[u];
        // the row that takes this place next: of this token, or of the next
        raw[u] = base + 2 * kAhead < slot1 ? load(token, base + 2 * (kAhead + u)) : load(token + 1, slot0 + 2 * u);
        const int first = base + 2 * u, slot = first + team;  // slots first, first + 1
        if (first >= slot1) continue;
        const bool is_q = slot < q_heads, is_v = slot >= q_heads + c.kv_heads;
        Row out = row;
        if (first < q_heads + c.kv_heads) {  // not two value heads
          float lo[4], hi[4], wl[4], wh[4];
          unpack4(row.lo, lo);
          unpack4(row.hi, hi);
          unpack4(is_q ? wq_lo : wk_lo, wl);
          unpack4(is_q ? wq_hi : wk_hi, wh);
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) ss += lo[i] * lo[i] + hi[i] * hi[i];
#pragma unroll
          for (int k = 8; k > 0; k >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, k);
          const float r = rsqrtf(ss * (1.f / 128.f) + eps);
          float a[4], b[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float l = lo[i] * r * wl[i], h = hi[i] * r * wh[i];
            a[i] = l * cos_lo[i] - h * sin_lo[i];
            b[i] = h * cos_hi[i] + l * sin_hi[i];
          }
          if (!is_v) {
            out.lo = make_uint2(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]));
            out.hi = make_uint2(pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3]));
          }
        }
        if (position < 0 || slot >= slot1 || (!is_q && !stored)) continue;
        const int h = slot - q_heads - (is_v ? c.kv_heads : 0);
        bf16* dst = is_q ? q_out + (static_cast<int64_t>(t0 + token) * q_heads + slot) * 128
                         : (is_v ? v_pages : k_pages) + (row0 + (static_cast<int64_t>(h) << c.page_shift)) * 128;
        *reinterpret_cast<uint2*>(dst + d0) = out.lo;
        *reinterpret_cast<uint2*>(dst + 64 + d0) = out.hi;
      }
    }
  }
}

}  // namespace

cudaError_t launch_paged_append(const PagedCache& c, const void* qkv, int64_t tokens, int q_heads, const void* q_norm,
                                const void* k_norm, const void* cos_t, const void* sin_t, bool fp32_tables,
                                int64_t table_rows, void* q_out, void* k_pages, void* v_pages, float eps,
                                cudaStream_t stream) {
  const auto x = static_cast<const bf16*>(qkv), qn = static_cast<const bf16*>(q_norm), kn = static_cast<const bf16*>(k_norm);
  const auto q = static_cast<bf16*>(q_out), k = static_cast<bf16*>(k_pages), v = static_cast<bf16*>(v_pages);
  // warps that fill the GPU once (32 per SM): shares of a token where there are few tokens, several tokens where many
  const int64_t fill = 32 * static_cast<int64_t>(sm_count());
  int split = 1;
  while (split < kMostSplit && 2 * split * tokens <= fill) split *= 2;
  const int per_warp = static_cast<int>(std::min<int64_t>(kMostTokens, (tokens + fill - 1) / fill));
  const int64_t warps = (tokens + per_warp - 1) / per_warp * split;
  const unsigned grid = static_cast<unsigned>((warps + kWarps - 1) / kWarps);
  const int n = static_cast<int>(tokens);
  if (fp32_tables)
    paged_append_kernel<float><<<grid, kThreads, 0, stream>>>(c, x, n, per_warp, split, q_heads, qn, kn, static_cast<const float*>(cos_t),
                                                              static_cast<const float*>(sin_t), table_rows, q, k, v, eps);
  else
    paged_append_kernel<bf16><<<grid, kThreads, 0, stream>>>(c, x, n, per_warp, split, q_heads, qn, kn, static_cast<const bf16*>(cos_t),
                                                             static_cast<const bf16*>(sin_t), table_rows, q, k, v, eps);
  return cudaGetLastError();
}

}  // namespace ipe
