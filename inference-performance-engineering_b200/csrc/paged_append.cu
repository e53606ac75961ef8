// q/k RMSNorm per head, split-half rotation at each token's own position, and the append of keys and
// values to a paged cache, for a ragged batch of new tokens.
//
// y = w * x * rsqrt(mean(x^2) + eps); o_d = y_d cos_d + r_d sin_d with r_d = -y_{d+64} for d < 64 and
// y_{d-64} above, all in fp32 and rounded to bf16 once (the contiguous append rounds at the reference's
// own points instead: it has to match the reference's bits, this one the formula).
//
// Bound by memory: 256 bytes in and out per head slot. A warp has a few consecutive tokens, or a share of one
// token's slots where there are few: enough warps to fill the GPU once, so the chain of lookups that a place
// takes (sequence, length, page; a lane per token, so once per warp) is paid once and behind the first rows'
// loads. 16 lanes per row with 16 bytes each, so the rotation's partner element sits 8 lanes away; a token's
// cosines and sines stay in registers over its rows.
#include <algorithm>

#include "launch.h"
#include "paged.cuh"
#include "tensor_map.h"

namespace ipe {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kAhead = 4;       // rows of 16 lanes in flight
constexpr int kMostSplit = 8;   // warps that share a token's slots
constexpr int kMostTokens = 32;  // of a warp

__device__ __forceinline__ void load_table(const bf16* p, float* f) { unpack8(ldg16(p), f); }
__device__ __forceinline__ void load_table(const float* p, float* f) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
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

__device__ __forceinline__ Place place_of(const PagedCache& c, int t, int64_t table_rows) {
  Place p{-1, 0, 0};
  const int s = sequence_of(c, t);
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
  const int team = lane >> 4, d0 = (lane & 15) * 8;
  uint4 raw[kAhead];
  auto load = [&](int token, int slot) {  // this lane's part of row `slot + team`
    const bool real = token < mine && slot + team < slot1;
    return real ? __ldcs(reinterpret_cast<const uint4*>(qkv + (static_cast<int64_t>(t0 + token) * slots + slot + team) * 128 + d0))
                : make_uint4(0, 0, 0, 0);
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) raw[u] = load(0, slot0 + 2 * u);
  Place own{-1, 0, 0};
  if (lane < mine) own = place_of(c, t0 + lane, table_rows);
  const uint4 wq = ldg16(q_norm + d0), wk = ldg16(k_norm + d0);

  for (int token = 0; token < mine; ++token) {
    const int position = __shfl_sync(0xffffffffu, own.position, token);
    const bool stored = __shfl_sync(0xffffffffu, own.stored, token);
    const int64_t row0 = __shfl_sync(0xffffffffu, own.row, token);
    float cs[8], sn[8];
    load_table(cos_t + static_cast<int64_t>(max(position, 0)) * 128 + d0, cs);
    load_table(sin_t + static_cast<int64_t>(max(position, 0)) * 128 + d0, sn);
#pragma unroll
    for (int i = 0; i < 8; ++i) sn[i] = d0 < 64 ? -sn[i] : sn[i];
    for (int base = slot0; base < slot1; base += 2 * kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const uint4 row = raw[u];
        // the row that takes this place next: of this token, or of the next
        const int after = base + 2 * (kAhead + u);
        raw[u] = base + 2 * kAhead < slot1 ? load(token, after) : load(token + 1, slot0 + 2 * u);
        if (base + 2 * u >= slot1) continue;
        const int slot = base + 2 * u + team;
        const bool is_q = slot < q_heads, is_v = slot >= q_heads + c.kv_heads;
        float x[8], w[8], o[8];
        unpack8(row, x);
        unpack8(is_q ? wq : wk, w);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, k);
        const float r = rsqrtf(ss * (1.f / 128.f) + eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = w[i] * (x[i] * r);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = x[i] * cs[i] + __shfl_xor_sync(0xffffffffu, x[i], 8) * sn[i];
        if (position < 0 || slot >= slot1) continue;
        if (is_q) {
          *reinterpret_cast<uint4*>(q_out + (static_cast<int64_t>(t0 + token) * q_heads + slot) * 128 + d0) = pack8(o);
        } else if (stored) {
          const int h = slot - q_heads - (is_v ? c.kv_heads : 0);
          bf16* dst = (is_v ? v_pages : k_pages) + (row0 + (static_cast<int64_t>(h) << c.page_shift)) * 128 + d0;
          *reinterpret_cast<uint4*>(dst) = is_v ? row : pack8(o);
        }
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
