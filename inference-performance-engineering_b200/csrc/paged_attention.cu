// Attention over a paged cache, one warp per (token, query head): the plain kernel behind the paged
// decode, the paged prefill and the shared-prefix attention.
//
// Lane l holds elements 4l..4l+3 of the query and of the output; keys are taken one at a time with an
// fp32 running maximum m and sum l: m' = max(m, s), o' = o e^(m-m') + v e^(s-m'). Rows without a key
// are zero.
#include "launch.h"
#include "paged.cuh"

namespace ipe {
namespace {

constexpr int kThreads = 256;
constexpr float kScaleLog2 = 0.08838834764831845f * 1.4426950408889634f;  // 128^-0.5 * log2(e)

__global__ void __launch_bounds__(kThreads) paged_attention_kernel(const PagedCache c, const bf16* __restrict__ q,
                                                                   const bf16* __restrict__ k_pages,
                                                                   const bf16* __restrict__ v_pages,
                                                                   bf16* __restrict__ out, int64_t tokens, int q_heads) {
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  if (warp >= tokens * q_heads) return;
  const int lane = threadIdx.x & 31;
  const int t = static_cast<int>(warp / q_heads), head = static_cast<int>(warp % q_heads);
  const int kv_head = head / (q_heads / c.kv_heads);
  int s = t, behind = 0;  // new tokens of the sequence after this one
  if (c.cu_tokens) {
    s = find_sequence(c.cu_tokens, c.sequences, t);
    if (s < 0) return;
    behind = __ldg(c.cu_tokens + s + 1) - t - 1;
  }
  const int keys = c.length(s) - behind;
  if (keys < 0) report(c.err, kErrPositionRange);
  const uint2 raw = *reinterpret_cast<const uint2*>(q + warp * 128 + lane * 4);
  float x[4] = {__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u), __uint_as_float(raw.y << 16),
                __uint_as_float(raw.y & 0xffff0000u)};
  float o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  for (int key = 0; key < keys; ++key) {
    const int64_t at = (c.page_row(c.page(s, key), kv_head) + (key & (c.page_size() - 1))) * 128 + lane * 4;
    const uint2 kr = *reinterpret_cast<const uint2*>(k_pages + at), vr = *reinterpret_cast<const uint2*>(v_pages + at);
    float dot = x[0] * __uint_as_float(kr.x << 16) + x[1] * __uint_as_float(kr.x & 0xffff0000u) +
                x[2] * __uint_as_float(kr.y << 16) + x[3] * __uint_as_float(kr.y & 0xffff0000u);
    dot = warp_sum(dot) * kScaleLog2;
    const float top = fmaxf(m, dot);
    const float keep = exp2f(m - top), p = exp2f(dot - top);
    m = top;
    l = l * keep + p;
    o[0] = o[0] * keep + p * __uint_as_float(vr.x << 16);
    o[1] = o[1] * keep + p * __uint_as_float(vr.x & 0xffff0000u);
    o[2] = o[2] * keep + p * __uint_as_float(vr.y << 16);
    o[3] = o[3] * keep + p * __uint_as_float(vr.y & 0xffff0000u);
  }
  const float inv = keys > 0 ? 1.f / l : 0.f;
  *reinterpret_cast<uint2*>(out + warp * 128 + lane * 4) =
      make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
}

}  // namespace

cudaError_t launch_paged_attention(const PagedCache& c, const void* q, const void* k_pages, const void* v_pages,
                                   void* out, int64_t tokens, int q_heads, cudaStream_t stream) {
  const int64_t blocks = (tokens * q_heads * 32 + kThreads - 1) / kThreads;
  paged_attention_kernel<<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(
      c, static_cast<const bf16*>(q), static_cast<const bf16*>(k_pages), static_cast<const bf16*>(v_pages),
      static_cast<bf16*>(out), tokens, q_heads);
  return cudaGetLastError();
}

}  // namespace ipe
