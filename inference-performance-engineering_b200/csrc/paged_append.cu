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
// Its rows are one contiguous run of qkv, which bulk copies bring into a ring of 4 KB pieces, so loads cost no
// instructions and never wait for arithmetic. 16 lanes per row, each with elements 4j..4j+3 and
// 64+4j..64+4j+3, so the rotation stays in the lane: o_lo = r (x_lo a_lo - x_hi b_lo), o_hi = r (x_hi a_hi +
// x_lo b_hi) with a = w cos, b = w sin formed once per token and kind of head.
// Measured: 22150 tokens of 16 + 2 * 8 heads 75 us (4.9 TB/s in and out), 24 sequences of 1 to 509 tokens of
// 32 + 2 * 8 heads 15.6 us (3.9 TB/s), 16 single tokens 3.0 us (a launch and the lookups).
#include <algorithm>

#include "launch.h"
#include "paged.cuh"
#include "tensor_map.h"

namespace ipe {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPiece = 16;       // rows of a bulk copy
constexpr int kStages = 2;       // pieces of a warp in flight
constexpr int kBlocksPerSm = 3;  // by shared memory and registers
constexpr int kMostSplit = 8;    // warps that share a token's slots
constexpr int kMostTokens = 32;  // of a warp
constexpr size_t kSmem = static_cast<size_t>(kWarps) * kStages * kPiece * 256;

// Four elements as two pairs.
__device__ __forceinline__ void unpack4(const uint2& v, uint64_t* f) {
  f[0] = pair(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u));
  f[1] = pair(__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}
__device__ __forceinline__ void load4(const bf16* p, uint64_t* f) { unpack4(__ldg(reinterpret_cast<const uint2*>(p)), f); }
__device__ __forceinline__ void load4(const float* p, uint64_t* f) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  f[0] = pair(a.x, a.y);
  f[1] = pair(a.z, a.w);
}
__device__ __forceinline__ uint32_t pack2(uint64_t v) {
  float lo, hi;
  unpair(v, &lo, &hi);
  return pack_bf16x2(lo, hi);
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

template <typename Table>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    paged_append_kernel(const PagedCache c, const bf16* __restrict__ qkv, int tokens, int per_warp, int split, int q_heads,
                        const bf16* __restrict__ q_norm, const bf16* __restrict__ k_norm, const Table* __restrict__ cos_t,
                        const Table* __restrict__ sin_t, int64_t table_rows, bf16* __restrict__ q_out,
                        bf16* __restrict__ k_pages, bf16* __restrict__ v_pages, float eps) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint64_t bars[kWarps][kStages];
  const int local = threadIdx.x >> 5, lane = threadIdx.x & 31, warp = blockIdx.x * kWarps + local;
  const int t0 = warp / split * per_warp, mine = min(per_warp, tokens - t0);
  const int slots = q_heads + 2 * c.kv_heads, share = (slots + split - 1) / split;
  const int slot0 = warp % split * share, width = min(slots, slot0 + share) - slot0;  // of the slots
  const int rows = mine > 0 && width > 0 ? mine * width : 0;  // one run: several tokens only with all their slots
  if (rows == 0) return;
  pdl_wait();  // for the kernels that wrote qkv, or still read what is written here
  pdl_trigger();
  unsigned char* ring = smem + local * (kStages * kPiece * 256);
  const bf16* src = qkv + (static_cast<int64_t>(t0) * slots + slot0) * 128;
  auto fetch = [&](int piece) {
    const int n = min(kPiece, rows - piece * kPiece) * 256;
    uint64_t* bar = &bars[local][piece % kStages];
    mbar_expect_tx(bar, n);
    bulk_copy(smem_addr(ring) + piece % kStages * (kPiece * 256), src + static_cast<int64_t>(piece) * (kPiece * 128), n, bar);
  };
  const int pieces = (rows + kPiece - 1) / kPiece;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bars[local][i], 1);
    fence_barrier_init();
    for (int i = 0; i < min(kStages, pieces); ++i) fetch(i);
  }
  Place own{-1, 0, 0};
  if (per_warp == 1)
    own = place_of(c, find_sequence(c.cu_tokens, c.sequences, t0), t0, table_rows);
  else if (lane < mine)
    own = place_of(c, sequence_of(c, t0 + lane), t0 + lane, table_rows);
  __syncwarp();

  const int team = lane >> 4, d0 = (lane & 15) * 4;
  // This half warp's row, its slot counted from slot0, and what it shares with the rows after it until `left`, the
  // slots of its token and kind of head from it on, runs out.
  int token = 0, slot = team, left = 0;
  bool normed = false, writes = false;
  uint64_t a_lo[2], a_hi[2], b_lo[2], b_hi[2];
  bf16* dst = nullptr;  // this lane's part of the row
  int64_t stride = 0;   // elements from a head's row to the next
  for (int piece = 0; piece < pieces; ++piece) {
    if (!mbar_wait(&bars[local][piece % kStages], (piece / kStages) & 1, c.err)) {
      for (int i = piece + 1; i < min(piece + kStages, pieces); ++i) mbar_wait(&bars[local][i % kStages], (i / kStages) & 1, c.err);
      return;  // the copies in flight have had their time too
    }
    const unsigned char* in = ring + piece % kStages * (kPiece * 256) + team * 256 + d0 * 2;
    const int n = min(kPiece, rows - piece * kPiece);
#pragma unroll 4
    for (int k = 0; k < kPiece / 2; ++k) {
      if (2 * k >= n) break;
      uint2 lo = *reinterpret_cast<const uint2*>(in + k * 512), hi = *reinterpret_cast<const uint2*>(in + k * 512 + 128);
      if (__any_sync(0xffffffffu, left <= 0)) {  // another token, or another kind of head
        while (slot >= width) {
          slot -= width;
          ++token;
        }
        const int head = slot0 + slot, kind = (head >= q_heads) + (head >= q_heads + c.kv_heads);
        const int from = min(token, 31), first = kind == 0 ? 0 : q_heads + (kind - 1) * c.kv_heads;
        const int position = __shfl_sync(0xffffffffu, own.position, from);
        const bool stored = __shfl_sync(0xffffffffu, own.stored, from);
        const int64_t row0 = __shfl_sync(0xffffffffu, own.row, from);
        left = min(width - slot, first + (kind == 0 ? q_heads : c.kv_heads) - head);
        normed = kind < 2;
        writes = position >= 0 && (kind == 0 || stored);
        stride = kind == 0 ? 128 : static_cast<int64_t>(128) << c.page_shift;
        dst = (kind == 0 ? q_out + static_cast<int64_t>(t0 + token) * q_heads * 128 : (kind == 1 ? k_pages : v_pages) + row0 * 128) +
              (head - first) * stride + d0;
        const int64_t angle = static_cast<int64_t>(max(position, 0)) * 128 + d0;
        const bf16* w = kind == 0 ? q_norm : k_norm;
        uint64_t w_lo[2], w_hi[2];
        load4(w + d0, w_lo);
        load4(w + 64 + d0, w_hi);
        load4(cos_t + angle, a_lo);
        load4(cos_t + angle + 64, a_hi);
        load4(sin_t + angle, b_lo);
        load4(sin_t + angle + 64, b_hi);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          a_lo[i] = mul2(a_lo[i], w_lo[i]);
          a_hi[i] = mul2(a_hi[i], w_hi[i]);
          b_lo[i] = mul2(mul2(b_lo[i], w_hi[i]), pair(-1.f, -1.f));
          b_hi[i] = mul2(b_hi[i], w_lo[i]);
        }
      }
      if (__any_sync(0xffffffffu, normed)) {
        uint64_t x[2], y[2];
        unpack4(lo, x);
        unpack4(hi, y);
        const uint64_t ss2 = fma2(y[1], y[1], fma2(y[0], y[0], fma2(x[1], x[1], mul2(x[0], x[0]))));
        float ss, more, r;
        unpair(ss2, &ss, &more);
        ss += more;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(ss * (1.f / 128.f) + eps));
        if (normed) {
          const uint64_t r2 = pair(r, r);
          lo = make_uint2(pack2(mul2(r2, fma2(y[0], b_lo[0], mul2(x[0], a_lo[0])))), pack2(mul2(r2, fma2(y[1], b_lo[1], mul2(x[1], a_lo[1])))));
          hi = make_uint2(pack2(mul2(r2, fma2(x[0], b_hi[0], mul2(y[0], a_hi[0])))), pack2(mul2(r2, fma2(x[1], b_hi[1], mul2(y[1], a_hi[1])))));
        }
      }
      if (writes && 2 * k + team < n) {
        *reinterpret_cast<uint2*>(dst) = lo;
        *reinterpret_cast<uint2*>(dst + 64) = hi;
      }
      slot += 2;
      left -= 2;
      dst += 2 * stride;
    }
    __syncwarp();
    if (lane == 0 && piece + kStages < pieces) fetch(piece + kStages);
  }
}

}  // namespace

cudaError_t launch_paged_append(const PagedCache& c, const void* qkv, int64_t tokens, int q_heads, const void* q_norm,
                                const void* k_norm, const void* cos_t, const void* sin_t, bool fp32_tables,
                                int64_t table_rows, void* q_out, void* k_pages, void* v_pages, float eps,
                                cudaStream_t stream) {
  const auto x = static_cast<const bf16*>(qkv), qn = static_cast<const bf16*>(q_norm), kn = static_cast<const bf16*>(k_norm);
  const auto q = static_cast<bf16*>(q_out), k = static_cast<bf16*>(k_pages), v = static_cast<bf16*>(v_pages);
  // warps that fill the GPU once: shares of a token where there are few tokens, several tokens where many
  const int64_t fill = static_cast<int64_t>(kBlocksPerSm) * kWarps * sm_count();
  int split = 1;
  while (split < kMostSplit && 2 * split * tokens <= fill) split *= 2;
  const int per_warp = static_cast<int>(std::min<int64_t>(kMostTokens, (tokens + fill - 1) / fill));
  const int64_t warps = (tokens + per_warp - 1) / per_warp * split;
  const unsigned grid = static_cast<unsigned>((warps + kWarps - 1) / kWarps);
  const int n = static_cast<int>(tokens);
  static std::atomic<uint64_t> allowed[2] = {{0}, {0}};
  cudaError_t e = fp32_tables ? allow_shared_memory(paged_append_kernel<float>, kSmem, &allowed[1])
                              : allow_shared_memory(paged_append_kernel<bf16>, kSmem, &allowed[0]);
  if (e != cudaSuccess) return e;
  if (fp32_tables)
    return launch_pdl(paged_append_kernel<float>, dim3(grid), dim3(kThreads), kSmem, stream, c, x, n, per_warp, split, q_heads,
                      qn, kn, static_cast<const float*>(cos_t), static_cast<const float*>(sin_t), table_rows, q, k, v, eps);
  return launch_pdl(paged_append_kernel<bf16>, dim3(grid), dim3(kThreads), kSmem, stream, c, x, n, per_warp, split, q_heads,
                    qn, kn, static_cast<const bf16*>(cos_t), static_cast<const bf16*>(sin_t), table_rows, q, k, v, eps);
}

}  // namespace ipe
