// q/k RMSNorm per head, split-half rotation at each token's own position, and the append of keys and
// values to a paged cache, for a ragged batch of new tokens.
//
// y = w * x * rsqrt(mean(x^2) + eps); o_d = y_d cos_d + r_d sin_d with r_d = -y_{d+64} for d < 64 and
// y_{d-64} above, all in fp32 and rounded to bf16 once (the contiguous append rounds at the reference's
// own points instead: it has to match the reference's bits, this one the formula).
//
// Bound by memory: 256 bytes in and out per head slot. One block per token, 16 lanes per slot with 16
// bytes each, so the rotation's partner element sits 8 lanes away. All of a token's rows are loaded
// before the chain of lookups (sequence, length, page) that its stores wait for.
#include "launch.h"
#include "paged.cuh"

namespace ipe {
namespace {

constexpr int kThreads = 256;
constexpr int kTeams = kThreads / 16;
constexpr int kUnroll = 2;  // slots of one team in flight

__device__ __forceinline__ void load_table(const bf16* p, float* f) { unpack8(ldg16(p), f); }
__device__ __forceinline__ void load_table(const float* p, float* f) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

template <typename Table>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const PagedCache c, const bf16* __restrict__ qkv,
                                                                int q_heads, const bf16* __restrict__ q_norm,
                                                                const bf16* __restrict__ k_norm,
                                                                const Table* __restrict__ cos_t,
                                                                const Table* __restrict__ sin_t, int64_t table_rows,
                                                                bf16* __restrict__ q_out, bf16* __restrict__ k_pages,
                                                                bf16* __restrict__ v_pages, float eps) {
  const int t = blockIdx.x;
  const int team = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * 8;
  const int slots = q_heads + 2 * c.kv_heads;
  const bf16* src = qkv + static_cast<int64_t>(t) * slots * 128 + d0;
  uint4 raw[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int slot = team + u * kTeams;
    raw[u] = slot < slots ? *reinterpret_cast<const uint4*>(src + slot * 128) : make_uint4(0, 0, 0, 0);
  }
  const int s = find_sequence(c.cu_tokens, c.sequences, t);
  if (s < 0) return;  // a row behind the last sequence: left as it is
  const int length = c.length(s);
  const int pos = length - (__ldg(c.cu_tokens + s + 1) - t);
  if (pos < 0 || pos >= table_rows) {  // more new tokens than positions, or past the rotation tables
    if (threadIdx.x == 0) report(c.err, kErrPositionRange);
    return;
  }
  const int id = __ldg(c.page_table + static_cast<int64_t>(s) * c.max_pages + (pos >> c.page_shift));
  const bool stored = static_cast<unsigned>(id) < static_cast<unsigned>(c.num_pages);
  if (!stored && threadIdx.x == 0) report(c.err, kErrPage);
  const int64_t row0 = c.page_row(stored ? id : 0, 0) + (pos & (c.page_size() - 1));

  float cs[8], sn[8], wq[8], wk[8];
  load_table(cos_t + static_cast<int64_t>(pos) * 128 + d0, cs);
  load_table(sin_t + static_cast<int64_t>(pos) * 128 + d0, sn);
  unpack8(ldg16(q_norm + d0), wq);
  unpack8(ldg16(k_norm + d0), wk);
#pragma unroll
  for (int i = 0; i < 8; ++i) sn[i] = d0 < 64 ? -sn[i] : sn[i];

  for (int base = 0; base < slots; base += kUnroll * kTeams) {
    uint4 next[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int slot = base + team + (kUnroll + u) * kTeams;
      next[u] = slot < slots ? *reinterpret_cast<const uint4*>(src + slot * 128) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int slot = base + team + u * kTeams;
      const bool is_q = slot < q_heads, is_v = slot >= q_heads + c.kv_heads;
      float x[8], o[8];
      unpack8(raw[u], x);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
      for (int k = 8; k > 0; k >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, k);
      const float r = rsqrtf(ss * (1.f / 128.f) + eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (is_q ? wq[i] : wk[i]) * (x[i] * r);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = x[i] * cs[i] + __shfl_xor_sync(0xffffffffu, x[i], 8) * sn[i];
      if (slot < slots) {
        if (is_q) {
          *reinterpret_cast<uint4*>(q_out + (static_cast<int64_t>(t) * q_heads + slot) * 128 + d0) = pack8(o);
        } else if (stored) {
          const int h = slot - q_heads - (is_v ? c.kv_heads : 0);
          bf16* dst = (is_v ? v_pages : k_pages) + (row0 + (static_cast<int64_t>(h) << c.page_shift)) * 128 + d0;
          *reinterpret_cast<uint4*>(dst) = is_v ? raw[u] : pack8(o);
        }
      }
      raw[u] = next[u];
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
  const unsigned grid = static_cast<unsigned>(tokens);
  if (fp32_tables)
    paged_append_kernel<float><<<grid, kThreads, 0, stream>>>(c, x, q_heads, qn, kn, static_cast<const float*>(cos_t),
                                                              static_cast<const float*>(sin_t), table_rows, q, k, v, eps);
  else
    paged_append_kernel<bf16><<<grid, kThreads, 0, stream>>>(c, x, q_heads, qn, kn, static_cast<const bf16*>(cos_t),
                                                             static_cast<const bf16*>(sin_t), table_rows, q, k, v, eps);
  return cudaGetLastError();
}

}  // namespace ipe
