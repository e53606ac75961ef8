// Causal attention of ragged new tokens over a paged cache, on the 5th-generation tensor cores.
//
// A block of work is up to 256 query rows of one (sequence, KV head): two tiles of 128 rows, a row being
// one of the G query heads of one token (128 / G whole tokens to a tile), so the G heads share every key
// that is read. Per key tile of 128 keys and query tile: S = Q K^T (tcgen05.mma into tensor memory), a row
// per thread reads its scores, keeps an fp32 running maximum and sum in base 2, writes P over the scores
// as bf16, and O += P V takes P from tensor memory. The two query tiles take turns: while one's scores
// are in the softmax warps the tensor cores work on the other's products.
//
// P is the one rounding before the output's: weights of 8 bits, whose errors average out over the keys;
// the sum they are divided by is of the unrounded weights. The running maximum moves only when a row's
// scores pass it by 2^8 (weights up to 256 are as exact in bf16 and fp32 as weights up to 1), so the
// accumulator in tensor memory is rescaled a few times per row instead of at every tile.
//
// Bound, on long prompts, by the chain of a tile: a step (128 keys of both query tiles) is 2070 cycles of
// products and takes about 2950, with the scores' way through the softmax warps (1400 cycles per tile, the
// special function unit half busy) and back between two products of the same tile. Measured, called alone behind a
// flush of L2, and as a share of a captured graph of 12 calls: 8192 new tokens, 16 query heads over 8, 253 and 225 us,
// 1090 and 1220 TFLOP/s of the products below the diagonal (0.66 and 0.74 of the measured peak). Nine prompts of
// 17 to 2500 tokens, 32 heads over 8, 136 and 115 us, 830 and 980 TFLOP/s; there the change from one piece to the
// next counts, 6000 cycles beside a step's. Much of them is instruction fetch, so what runs once per piece stands
// in rolled loops (in the graph 119 us with them unrolled). Pieces of two prompts on 9000 to 20000 cached tokens: 62
// and 57 to 68 us, about 2 TB/s. 512 tokens: 16.4 and 15.5 us, a chain of lookups and four steps.
//
// Warps 0-3 and 4-7: softmax of query tile 0 and 1, one row per thread; warp 8: work list and TMA loads;
// warp 9: tensor memory and MMA issue. Persistent, one CTA per SM; the blocks go to the CTAs heaviest
// first, back and forth. Where there are fewer blocks than that can balance (two per SM), every block's key
// tiles are dealt to the CTAs in equal contiguous runs instead; parts of a block go to the workspace as
// records (unnormalised o, maximum, sum), merged by a second kernel in order of the keys. The host decides
// between the two by the sizes it sees, rows behind the last sequence among them, not by the lengths: many
// sequences, or a buffer much larger than its tokens, leave a long context to one CTA per block. (One new token
// each of 36 and of 40 sequences, one of them on 30000 keys, 16 heads over 8: 106 and 446 us. Two pieces on 9000
// and 20000 keys, no, 4000 and 4800 rows behind them: 79, 87 and 311 us.)
//
// Values past a block's last key are zeroed in shared memory before they meet their zero weights. A row
// whose accumulator is not finite all the same (a value that is infinite or NaN, its own or one of a
// later token in the tile) is computed again from the keys it sees, when the CTA is done with its list of
// work: no other row, and no wait, is behind it. A row that sees a score of infinity or NaN is NaN.
// Every mbarrier wait is bounded; a timeout sets the device error word and the CTA winds down.
#include <algorithm>

#include "launch.h"
#include "paged_records.cuh"
#include "tensor_map.h"

namespace ipe {
namespace {

constexpr int kThreads = 384;      // three warpgroups: softmax of query tile 0, of tile 1, and the rest
constexpr int kLoadWarp = 8, kMmaWarp = 9;  // warps 0-7: softmax; 10, 11 idle
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;  // 2 * 208 + 88 = 3 * 168, what the launch holds
constexpr int kBM = 128, kBN = 128, kD = 128;
constexpr int kHalf = 128 * 64 * 2;  // a 128-row x 64-column bf16 block, 128-byte swizzle
constexpr int kTile = 2 * kHalf;
constexpr int kStages = 2;           // pairs of tiles in the ring: the values of a step and the keys of the next
constexpr int kTmemCols = 512;       // all there are, so they begin at column
constexpr uint32_t kTmem = 0;        // S0 [0, 128), S1 [128, 256), O0 [256, 384), O1 [384, 512)
constexpr int kMaxListed = 1024;     // sequences (and, in runs, blocks) listed in shared memory
constexpr int kMergeTiles = 5;       // what records and their merge cost, in key tiles' time (9 us)
constexpr int kByCubic = 1;          // of every 4 pairs of weights, those whose 2^x is a cubic
constexpr float kSlack = 8.f / kScaleLog2;  // how far scores may pass the maximum in use

struct Work {       // one piece: key tiles of a block
  int token0;       // first query row's token (row of q)
  int tokens;       // of the block
  int position0;    // of token0 in its sequence
  int sequence;
  int kv_head;
  int keys;         // the block's keys: tiles end here
  int tile0;        // first key tile of the piece
  int count[2];     // key tiles of each query tile in this piece
  int record;       // the record slot of a part, -1 for a whole block
};

struct Shared {
  uint64_t q_full, q_empty;
  uint64_t pair_full[kStages], pair_empty[kStages];
  uint64_t s_full[2], p_full[2][2], o_full[2], o_empty[2];
  uint32_t tmem;
  int abort;
  int again[8];  // by softmax warp: the list of rows that are attended again
  Work work[2];
  alignas(16) uint4 stage[8][32 * 4];  // by softmax warp
  int low[kMaxListed + 1], high[kMaxListed + 1];
};
constexpr size_t kSmem = 1024 + static_cast<size_t>(2 + 2 * kStages) * kTile + sizeof(Shared);

struct PrefillArgs {
  PagedCache c;
  const bf16* q;
  const bf16* k;
  const bf16* v;
  bf16* out;
  float* records;  // [grid][2][kBlockRecord] where the key tiles are dealt in runs, else null
  int2* items;     // in runs: [blocks][kv_heads], item_parts
  int4* blocks;    // in runs: of each block token0, tokens, position0; before them, how many there are
  float* whole;    // shared keys: where rows that are not in parts go, [tokens][q_heads][kRecord]
  int tokens;
  int q_heads;
  int shared_keys;
  int most_blocks;  // in runs: room for so many
};

// Shared-memory operands with the 128-byte swizzle, 8-row groups 1024 bytes apart. The upper words of
// their descriptors are alike; the lower ones hold the address, and for an MN-major operand (V: the
// head's dimensions contiguous) the distance of its 64-column halves.
constexpr uint32_t kDescUpper = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_kmajor(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mnmajor(uint32_t addr) { return (addr >> 4) | (static_cast<uint32_t>(kHalf >> 4) << 16); }
// kind::f16: fp32 D, bf16 A and B, M = N = 128; B transposed (MN-major) when transpose_b.
__device__ __forceinline__ constexpr uint32_t instr_desc(bool transpose_b) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (transpose_b ? (1u << 16) : 0u) | (static_cast<uint32_t>(kBN >> 3) << 17) |
         (static_cast<uint32_t>(kBM >> 4) << 24);
}
__device__ __forceinline__ void mma_smem(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescUpper));
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescUpper));
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes != 0;
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// 32 consecutive 32-bit columns of this warp's 32 TMEM lanes (one row per lane); no wait.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// The wait for this thread's loads; the loaded registers pass through it, so no use of them moves ahead.
__device__ __forceinline__ void tmem_ld_wait(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// Bounded waits of a whole converged warp, the same answer in every lane. The first try is all that is
// inline: a warp that finds the phase complete, as the MMA warp mostly does, goes through few instructions.
__device__ __forceinline__ bool wait_longer(uint64_t* bar, uint32_t parity, int* err) {
  uint64_t start = 0;
  for (uint32_t i = 1;; ++i) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((i & 63u) == 0) {
      const uint64_t now = __shfl_sync(0xffffffffu, globaltimer_ns(), 0);
      if (start == 0) start = now;
      if (now - start > kWaitLimitNs) {
        report(err, kErrWaitTimeout);
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || wait_longer(bar, parity, err);
}

// whether a phase is complete, at once
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t yes;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(yes)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return yes != 0;
}

// the largest of three; NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x for a pair, without the special function unit, which is the busiest: x = n + f, n the nearest
// integer, 2^f on [-1/2, 1/2] by the cubic through 1 of least largest relative error (1.02e-4, fitted by
// iteratively reweighted least squares; a bf16 weight is off by up to 3.9e-3), n added to the exponent.
// x below -127 counts as -127, where the exponent field and the cubic's fraction reach zero together: a
// hidden key's weight is exactly 0, as it has to be beside a value of the type's largest.
__device__ __forceinline__ void exp2_pair(uint64_t x, float* p0, float* p1) {
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it leaves the nearest integer in the low bits
  float lo, hi;
  unpair(x, &lo, &hi);
  x = pair(fmaxf(lo, -127.f), fmaxf(hi, -127.f));
  const uint64_t n = add2(x, pair(kRound, kRound));
  const uint64_t f = fma2(add2(n, pair(-kRound, -kRound)), pair(-1.f, -1.f), x);
  uint64_t y = fma2(pair(0.0550089329f, 0.0550089329f), f, pair(0.242210969f, 0.242210969f));
  y = fma2(y, f, pair(0.693282902f, 0.693282902f));
  y = fma2(y, f, pair(1.f, 1.f));
  float n0, n1, y0, y1;
  unpair(n, &n0, &n1);
  unpair(y, &y0, &y1);
  *p0 = __int_as_float((__float_as_int(n0) << 23) + __float_as_int(y0));
  *p1 = __int_as_float((__float_as_int(n1) << 23) + __float_as_int(y1));
}

// Which halves of two bf16 hold what, as 1 each.
constexpr uint32_t kOnes = 0x3f803f80u, kInfinities = 0x7f807f80u;
__device__ __forceinline__ uint32_t ones_where_infinite(uint32_t x, uint32_t sign) { return __vcmpeq2(x, kInfinities | sign) & kOnes; }
__device__ __forceinline__ uint32_t ones_where_nan(uint32_t x) { return __vcmpgtu2(x & 0x7fff7fffu, kInfinities) & kOnes; }
__device__ __forceinline__ uint32_t not_finite(uint32_t x) { return __vcmpgeu2(x & 0x7fff7fffu, kInfinities); }

// --------------------------------------------------------------------------- the list of work

// A sequence's new tokens [begin, end) of q's rows, and its length, -1 where the offsets are none. The list ends before
// the first such sequence: the offsets of those before it ascend, so no row belongs to two of them.
struct Span {
  int begin, tokens, length;
};
__device__ __forceinline__ Span span_from(const PagedCache& c, int rows, int b, int e, int n) {
  if (b < 0 || e < b || e > rows) {
    report(c.err, kErrPositionRange);
    return Span{0, 0, -1};
  }
  const int length = c.checked_length(n);
  if (e - b > length) report(c.err, kErrPositionRange);
  return Span{b, e - b, length};
}
__device__ __forceinline__ Span span_of(const PagedCache& c, int s, int rows) {
  return span_from(c, rows, __ldg(c.cu_tokens + s), __ldg(c.cu_tokens + s + 1), __ldg(c.lengths + s));
}

// The piece of block `b` of sequence `s`: key tiles [tile0, tile1) (tile1 < 0: all of them).
__device__ __forceinline__ int block_keys(const Span& x, int b, int per_block) {
  return max(0, x.length - x.tokens + min((b + 1) * per_block, x.tokens));
}
__device__ __forceinline__ int tiles_of(int keys) { return max(1, (keys + kBN - 1) / kBN); }

__device__ __forceinline__ Work make_work(const Span& x, int s, int b, int kv_head, int per_tile, int tile0, int tile1) {
  Work w;
  w.token0 = x.begin + b * 2 * per_tile;
  w.tokens = min(2 * per_tile, x.tokens - b * 2 * per_tile);
  w.position0 = x.length - x.tokens + b * 2 * per_tile;
  w.sequence = s;
  w.kv_head = kv_head;
  w.keys = max(0, w.position0 + w.tokens);
  w.tile0 = tile0;
  w.record = -1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int mine = min(per_tile, w.tokens - i * per_tile);  // tokens of this query tile
    const int tiles = mine > 0 ? tiles_of(w.position0 + i * per_tile + mine) : 0;
    w.count[i] = max(0, min(tiles, tile1 < 0 ? tiles : tile1) - tile0);
  }
  return w;
}

// exclusive prefix sums of x over the warp
__device__ __forceinline__ int warp_scan(int x) {
  int scan = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, scan, o);
    if ((threadIdx.x & 31) >= o) scan += up;
  }
  return scan - x;
}

// the last index below n whose value is at most x, of an ascending list that starts with 0
__device__ __forceinline__ int last_at_most(const int* list, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (list[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Where a row goes unless to the output: `row` of a block's 256 in its record slot, or its own record.
struct RecordPlace {
  float* rec;  // null: to the output
  bool part;
  int m, sum;
  __device__ __forceinline__ int vector(int v) const { return part ? block_vector(v) : v * 4; }
};
template <bool kShared>
__device__ __forceinline__ RecordPlace record_place(const PrefillArgs& a, int record, int row, int64_t out_row) {
  RecordPlace p;
  p.part = record >= 0;
  p.rec = p.part    ? a.records + static_cast<int64_t>(record) * kBlockRecord + row * 8
          : kShared ? a.whole + out_row * kRecord
                    : nullptr;
  p.m = p.part ? kBlockRows * 128 - row * 7 : 128;
  p.sum = p.part ? p.m + kBlockRows : 129;
  return p;
}

// Rows of a softmax warp whose scores are finite and whose accumulators are not wait until the CTA's list of work has
// ended, so that nothing waits for them. They make a list: what is known of a piece's rows stands in the place of the
// first of them (no row is another piece's), which is named by its row of out or, where that is a part's, by
// ~(record slot * 256 + row).
struct Again {
  int token0, position0, sequence, kv_head, tile0, count;
  unsigned rows;  // of the warp's 32
  int next;
};
constexpr int kNoRow = INT32_MAX;
template <bool kShared>
__device__ __forceinline__ uint4* place_of_row(const PrefillArgs& a, int name) {
  if (name < 0) return reinterpret_cast<uint4*>(a.records + static_cast<int64_t>(~name / kBlockRows) * kBlockRecord + ~name % kBlockRows * 8);
  if (kShared) return reinterpret_cast<uint4*>(a.whole + static_cast<int64_t>(name) * kRecord);
  return reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(name) * 128);
}

// The rows of one entry of that list, from the keys of their piece that each sees; gives the next entry's name. 16 rows
// at a time, 16 keys a step, m16n8k16 products straight from the cache: 3 us a step, a chain of loads. (8192 tokens that
// all see a NaN value: 4.7 ms instead of 0.25; a row of theirs alone would take as long key by key.) A value that is not
// finite enters the products as 0; the rows that see it are found by products of 0 and 1 with where it is, and get
// infinity, or NaN. The products' inner index is any order of the dimensions, and so are the values' columns: they are
// such that a lane loads and stores 16 bytes at a time.
template <bool kShared>
__device__ __noinline__ int attend_again(const PrefillArgs& a, int name) {
  const PagedCache& c = a.c;
  const int lane = threadIdx.x & 31, g = lane >> 2, col = lane & 3, tile = threadIdx.x >> 7;
  const int group = a.q_heads / c.kv_heads, per_tile = kBM / group;
  const uint4* entry = place_of_row<kShared>(a, name);
  const uint4 e0 = ldcg16(entry), e1 = ldcg16(entry + 1);
  const Again w{static_cast<int>(e0.x), static_cast<int>(e0.y), static_cast<int>(e0.z), static_cast<int>(e0.w),
                static_cast<int>(e1.x), static_cast<int>(e1.y), e1.z, static_cast<int>(e1.w)};
  const int from = w.tile0 * kBN, to = from + w.count * kBN;
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    const unsigned rows = w.rows >> (16 * half) & 0xffffu;
    if (rows == 0) continue;
    int number[2], lim[2];  // this lane's rows, g and g + 8 of the 16: as in the tile, and the keys they see
    int64_t row[2];         // of q and out
    uint4 q[2][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      number[r] = (threadIdx.x & 96) + half * 16 + g + 8 * r;
      const int place = number[r] / group, token = tile * per_tile + place;
      row[r] = static_cast<int64_t>(w.token0 + token) * a.q_heads + w.kv_head * group + number[r] - place * group;
      lim[r] = 0;
      if (rows >> (g + 8 * r) & 1) lim[r] = min(to, kShared ? c.length(w.token0 + token) : w.position0 + token + 1);
      if (kShared) lim[r] = min(lim[r], a.shared_keys);
#pragma unroll
      for (int i = 0; i < 4; ++i) q[r][i] = lim[r] > from ? ldcg16(a.q + row[r] * 128 + i * 32 + col * 8) : make_uint4(0, 0, 0, 0);
    }
    const int end = __reduce_max_sync(0xffffffffu, max(lim[0], lim[1]));
    float o[16][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll 1
    for (int key0 = from; key0 < end; key0 += 16) {
      const int64_t at = c.page_row(c.page(w.sequence, key0), w.kv_head) + (key0 & (c.page_size() - 1));  // 16 keys lie in a page
      float s[2][4] = {};
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        uint4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = ldcg16(a.k + (at + 8 * t + g) * 128 + i * 32 + col * 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          mma16816(s[t], q[0][i].x, q[1][i].x, q[0][i].y, q[1][i].y, x[i].x, x[i].y);
          mma16816(s[t], q[0][i].z, q[1][i].z, q[0][i].w, q[1][i].w, x[i].z, x[i].w);
        }
      }
      uint4 v[4][2];  // keys 2 col, 2 col + 1, and 8 on from these: dimensions 16 g .. 16 g + 15
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = 2 * col + (j & 1) + (j >> 1) * 8;
        const bf16* vr = a.v + (at + key) * 128 + g * 16;
        const bool seen = key0 + key < end;
        v[j][0] = seen ? ldcg16(vr) : make_uint4(0, 0, 0, 0);
        v[j][1] = seen ? ldcg16(vr + 8) : make_uint4(0, 0, 0, 0);
      }
      uint32_t p[4], counted[4], nothing[4];  // as fragments: weights, whether they are above 0, whether a seen key's is 0
      float keep[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float x[4], top = m[r];
        bool seen[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          seen[e] = key0 + 8 * (e >> 1) + 2 * col + (e & 1) < lim[r];
          x[e] = seen[e] ? s[e >> 1][2 * r + (e & 1)] : -INFINITY;
          top = fmaxf(top, x[e]);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float base = top == -INFINITY ? 0.f : top * kScaleLog2;
        keep[r] = part_weight(m[r], base);
        m[r] = top;
        l[r] *= keep[r];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float p0 = exp2_approx(x[2 * t] * kScaleLog2 - base), p1 = exp2_approx(x[2 * t + 1] * kScaleLog2 - base);
          l[r] += p0 + p1;
          p[2 * t + r] = pack_bf16x2(p0, p1);
          const uint32_t lo = seen[2 * t] ? 0x3f80u : 0u, hi = seen[2 * t + 1] ? 0x3f800000u : 0u;
          const uint32_t lost = (x[2 * t] == -INFINITY ? 0xffffu : 0u) | (x[2 * t + 1] == -INFINITY ? 0xffff0000u : 0u);
          counted[2 * t + r] = (lo | hi) & ~lost;
          nothing[2 * t + r] = (lo | hi) & lost;
        }
      }
      if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
        for (int t = 0; t < 16; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[t][e] *= keep[e >> 1];
      }
      uint32_t odd = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) odd |= not_finite(v[j][i].x) | not_finite(v[j][i].y) | not_finite(v[j][i].z) | not_finite(v[j][i].w);
      const bool any_odd = __any_sync(0xffffffffu, odd != 0);
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        uint32_t b[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint4 &x = v[2 * j][t >> 3], &y = v[2 * j + 1][t >> 3];
          const int word = t >> 1 & 3;
          b[j] = __byte_perm(word == 0 ? x.x : word == 1 ? x.y : word == 2 ? x.z : x.w,
                             word == 0 ? y.x : word == 1 ? y.y : word == 2 ? y.z : y.w, t & 1 ? 0x7632 : 0x5410);
        }
        if (any_odd) {
          float up[4] = {}, down[4] = {}, none[4] = {};
          mma16816(up, counted[0], counted[1], counted[2], counted[3], ones_where_infinite(b[0], 0u), ones_where_infinite(b[1], 0u));
          mma16816(down, counted[0], counted[1], counted[2], counted[3], ones_where_infinite(b[0], 0x80008000u), ones_where_infinite(b[1], 0x80008000u));
          mma16816(none, counted[0], counted[1], counted[2], counted[3], ones_where_nan(b[0]), ones_where_nan(b[1]));
          mma16816(none, nothing[0], nothing[1], nothing[2], nothing[3], not_finite(b[0]) & kOnes, not_finite(b[1]) & kOnes);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (up[e] > 0.f) o[t][e] += INFINITY;
            if (down[e] > 0.f) o[t][e] -= INFINITY;
            if (none[e] > 0.f) o[t][e] = NAN;
          }
          b[0] &= ~not_finite(b[0]);
          b[1] &= ~not_finite(b[1]);
        }
        mma16816(o[t], p[0], p[1], p[2], p[3], b[0], b[1]);
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (!(rows >> (g + 8 * r) & 1)) continue;
      const RecordPlace at = record_place<kShared>(a, name < 0 ? ~name / kBlockRows : -1, tile * kBM + number[r], row[r]);
      const float inv = lim[r] <= from ? 0.f : at.rec ? 1.f : 1.f / l[r];
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // dimensions 32 col + 8 e on: of column 2 col, then of 2 col + 1
        float f[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) f[d] = o[(e & 1) * 8 + d][2 * r + (e >> 1)] * inv;
        if (at.rec) {
#pragma unroll
          for (int d = 0; d < 2; ++d)
            *reinterpret_cast<float4*>(at.rec + at.vector(col * 8 + 2 * e + d)) = make_float4(f[4 * d], f[4 * d + 1], f[4 * d + 2], f[4 * d + 3]);
        } else {
          *reinterpret_cast<uint4*>(a.out + row[r] * 128 + col * 32 + e * 8) = pack8(f);
        }
      }
      if (at.rec && col == 0) {
        at.rec[at.m] = m[r];
        at.rec[at.sum] = l[r];
      }
    }
  }
  __syncwarp();
  return w.next;
}

// kShared: the "new tokens" are one query token of each sequence, all on the pages of c.prefix_pages (a
// row sees those of them that its sequence's length covers), key tiles dealt in runs, and all rows go to
// records that the decode kernel's merge joins with the rest of each sequence.
template <bool kShared>
__global__ void __launch_bounds__(kThreads, 1)
    paged_prefill_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PrefillArgs a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* s_q = smem;
  unsigned char* ring = smem + 2 * kTile;
  Shared& sh = *reinterpret_cast<Shared*>(ring + kStages * 2 * kTile);
  volatile int* abort_flag = &sh.abort;
  const PagedCache& c = a.c;
  int* err = c.err;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.q_heads / c.kv_heads;
  const int per_tile = kBM / group, per_block = 2 * per_tile;  // tokens
  const bool in_runs = kShared || a.records != nullptr;
  pdl_trigger();

  if (threadIdx.x == 0) {
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_empty, 1 + 8);  // the last S of the piece, and every softmax warp's look at the list
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sh.pair_full[s], 1);
      mbar_init(&sh.pair_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i][0], 128);  // the first and the second 64 keys
      mbar_init(&sh.p_full[i][1], 128);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.o_empty[i], 128);
    }
    sh.abort = 0;
    for (int i = 0; i < 8; ++i) sh.again[i] = kNoRow;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }

  int first[3] = {0, 0, 0};  // what the list of work begins with, on its way while the CTA is set up
  if (!kShared && warp == kLoadWarp && lane < c.sequences) {
    first[0] = __ldg(c.cu_tokens + lane);
    first[1] = __ldg(c.cu_tokens + lane + 1);
    first[2] = __ldg(c.lengths + lane);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0 && sh.tmem != kTmem) report(err, kErrShape);
  if (warp >= kLoadWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kLoadWarp) {
      // ------------------------------------------------------------------ work list and loads
      if (lane < 3)
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane == 0 ? &map_q : lane == 1 ? &map_k : &map_v))
                     : "memory");
      const int ps = c.page_size(), subs = kBN >> c.page_shift;
      // In runs: sh.low = blocks before each sequence, sh.high = key tiles before each block. Otherwise
      // sh.low .. sh.high: the sequence's blocks as numbers that grow with their keys (block 0 of a sequence
      // on a context starts at the context's length in blocks), `most` past the largest.
      const int shared_tiles = (a.shared_keys + kBN - 1) / kBN;
      int blocks = 0, tiles = 0, most = 0;
      bool whole = false;
      int sound = c.sequences;         // sequences before the first whose offsets are none
      Span mine{0, 0, 0};            // of sequence `lane`
      int mine_first = 0, mine_n = 0;  // its blocks among all
      auto span_at = [&](int s) {  // of any, for a whole warp
        if (c.sequences > 32) return span_of(c, s, a.tokens);
        return Span{__shfl_sync(0xffffffffu, mine.begin, s), __shfl_sync(0xffffffffu, mine.tokens, s),
                    __shfl_sync(0xffffffffu, mine.length, s)};
      };
      if (kShared) {
        blocks = (a.tokens + per_block - 1) / per_block;
        tiles = blocks * shared_tiles;
      } else {
        for (int base = 0; base < c.sequences; base += 32) {
          const int s = base + lane;
          Span x{0, 0, 0};
          if (s < sound) x = base == 0 ? span_from(c, a.tokens, first[0], first[1], first[2]) : span_of(c, s, a.tokens);
          const unsigned none = __ballot_sync(0xffffffffu, x.length < 0);
          if (none != 0) sound = base + __ffs(none) - 1;
          if (s >= sound) x = Span{0, 0, 0};
          const int n = (x.tokens + per_block - 1) / per_block, low = max(0, x.length - x.tokens) / per_block;
          const int before = blocks + warp_scan(n);
          if (base == 0) {
            mine = x;
            mine_first = before;
            mine_n = n;
          }
          if (s < kMaxListed) {
            sh.low[s] = in_runs ? min(before, a.most_blocks) : low;
            sh.high[s] = low + n;
          }
          if (n > 0) most = max(most, low + n);
          blocks = __shfl_sync(0xffffffffu, before + n, 31);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        __syncwarp();
      }
      if (!kShared && in_runs) {
        blocks = min(blocks, a.most_blocks);
        if (blockIdx.x == 0 && lane == 0) a.blocks[-1].x = blocks;
        int longest = 0;
        for (int base = 0; base < blocks; base += 32) {
          const int i = base + lane;
          const int s = last_at_most(sh.low, c.sequences, min(i, blocks - 1));
          const Span x = span_at(s);
          const int n = i < blocks ? tiles_of(block_keys(x, i - sh.low[s], per_block)) : 0;
          const int before = tiles + warp_scan(n);
          if (i < blocks) sh.high[i] = before;
          longest = max(longest, n);
          tiles = __shfl_sync(0xffffffffu, before + n, 31);
        }
        // Whole blocks after all where the runs would save less than the records and their merge cost.
        longest = __reduce_max_sync(0xffffffffu, longest);
        const int ctas = gridDim.x;
        whole = longest * ((blocks * c.kv_heads + ctas - 1) / ctas) <= (tiles * c.kv_heads + ctas - 1) / ctas + kMergeTiles;
        if (whole) {
          for (int i = lane; i < blocks; i += 32) sh.high[i] = i;  // a block is one unit
          tiles = blocks;
        }
        if (lane == 0) sh.high[blocks] = tiles;
        __syncwarp();
      }
      const int works = blocks * c.kv_heads;
      const Deal deal(in_runs ? tiles * c.kv_heads : 0, gridDim.x);
      int unit = deal.start(blockIdx.x);  // in runs
      const int unit_end = deal.start(blockIdx.x + 1);
      const bool listed = c.sequences <= kMaxListed;
      auto range_of = [&](int s, int* low, int* high) {
        *low = *high = 0;
        if (s >= sound) return;
        if (listed) {
          *low = sh.low[s];
          *high = sh.high[s];
        } else {
          const Span x = span_of(c, s, a.tokens);
          *low = max(0, x.length - x.tokens) / per_block;
          *high = *low + (x.tokens + per_block - 1) / per_block;
        }
      };
      // the `rank`-th block in descending order of its number; the whole warp takes part
      int low0 = 0, high0 = 0;  // of sequence `lane`
      if (!in_runs) range_of(lane, &low0, &high0);
      auto select = [&](int rank, int* seq, int* block) {
        auto at_least = [&](int x) {
          int n = max(0, high0 - max(low0, x));
          for (int s = lane + 32; s < c.sequences; s += 32) {
            int low, high;
            range_of(s, &low, &high);
            n += max(0, high - max(low, x));
          }
          return static_cast<int>(__reduce_add_sync(0xffffffffu, n));
        };
        int lo = 0, hi = most, above = 0;  // at_least(lo) > rank >= at_least(hi) = above
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1, n = at_least(mid);
          if (n > rank) {
            lo = mid;
          } else {
            hi = mid;
            above = n;
          }
        }
        int left = rank - above;  // so many sequences with a block `lo` come before
        *seq = *block = 0;
        for (int base = 0; base < c.sequences; base += 32) {
          int low = low0, high = high0;
          if (base > 0) range_of(base + lane, &low, &high);
          const bool has = low <= lo && lo < high;
          const unsigned all = __ballot_sync(0xffffffffu, has);
          const unsigned it = __ballot_sync(0xffffffffu, has && __popc(all & ((1u << lane) - 1)) == left);
          if (it != 0) {
            const int at = __ffs(it) - 1;
            *seq = base + at;
            *block = lo - __shfl_sync(0xffffffffu, low, at);
            return;
          }
          left -= __popc(all);
        }
      };
      // The next piece of this CTA's list, if there is one.
      int round = 0;
      auto take = [&](Work* out) {
        Work w;
        if (in_runs) {
          if (unit >= unit_end) return false;
          const int block = kShared ? unit / (shared_tiles * c.kv_heads) : last_at_most(sh.high, blocks, unit / c.kv_heads);
          const int before = kShared ? block * shared_tiles : sh.high[block];
          const int n = kShared ? shared_tiles : sh.high[block + 1] - before;
          const int r = unit - before * c.kv_heads, kv_head = r / n;
          const int tile0 = r - kv_head * n, tile1 = min(n, tile0 + unit_end - unit);
          if (tile0 == 0 && lane == 0)
            a.items[static_cast<int64_t>(block) * c.kv_heads + kv_head] = item_parts(deal, unit, n, blockIdx.x);
          if (kShared) {
            // every row sees up to all shared keys: as if the tokens stood behind them
            w = make_work(Span{0, a.tokens, a.shared_keys + a.tokens}, 0, block, kv_head, per_tile, tile0, tile1);
            w.keys = a.shared_keys;
#pragma unroll
            for (int i = 0; i < 2; ++i) w.count[i] = w.tokens > i * per_tile ? tile1 - tile0 : 0;
          } else {
            const int s = last_at_most(sh.low, c.sequences, block);
            w = make_work(span_at(s), s, block - sh.low[s], kv_head, per_tile, tile0, whole ? -1 : tile1);
            if (tile0 == 0 && kv_head == 0 && lane == 0) a.blocks[block] = make_int4(w.token0, w.tokens, w.position0, 0);
          }
          if (tile0 > 0 || tile1 < n) w.record = static_cast<int>(blockIdx.x) * 2 + (round == 0 ? 0 : 1);
          unit += tile1 - tile0;
          ++round;
        } else {
          const int ctas = gridDim.x;
          int rank;
          do {  // a round that ends before this CTA's place is the last one but for an empty one
            if (round * ctas >= works) return false;
            rank = round * ctas + ((round & 1) ? ctas - 1 - blockIdx.x : blockIdx.x);
            ++round;
          } while (rank >= works);
          int s, b = rank / c.kv_heads;
          if (works <= ctas && c.sequences <= 32) {  // a block per CTA at most: in any order
            s = __ffs(__ballot_sync(0xffffffffu, b >= mine_first && b < mine_first + mine_n)) - 1;
            b -= __shfl_sync(0xffffffffu, mine_first, s);
          } else {
            select(b, &s, &b);
          }
          w = make_work(span_at(s), s, b, rank % c.kv_heads, per_tile, 0, -1);
        }
        *out = w;
        return true;
      };

      // One pair of tiles at a time. The next piece is looked up while the one at hand has its first pairs on
      // their way: that takes about two steps' time (7000 cycles with its loads), which nobody then waits for.
      int slot = 0, piece = 0, step = 0, steps = -1;
      uint32_t phase = 0, armed = 0;  // bit s: parity armed on pair_full[s]; bit 16 + s: armed at all
      bool ok = true, known = false, more = false;
      Work w, next;
      // This lane's page of a step's tile: its ID is loaded a step ahead and looked at when it is used.
      auto key_of = [&](const Work& x, int step) { return (x.tile0 + step) * kBN + lane * ps; };
      auto has_page = [&](const Work& x, int step) {
        return lane < subs && step < max(x.count[0], x.count[1]) && key_of(x, step) < x.keys;
      };
      auto load_id = [&](const Work& x, int step) { return has_page(x, step) ? c.page_id(x.sequence, key_of(x, step)) : 0; };
      int id = 0, id_next = 0, row = 0, row_v = 0;  // cache rows of the keys to load, and of the step before
      bool has = false, has_v = false;
      while (!*abort_flag) {
        if (!known && (step > steps || step == 3)) {
          known = true;
          more = take(&next);
          if (more) id_next = load_id(next, 0);
        }
        if (step > steps) {
          if (!more) break;
          w = next;
          id = id_next;
          known = false;
          step = 0;
          steps = max(w.count[0], w.count[1]);
          has = has_page(w, 0);
          has_v = false;
        }
        // The block's queries, once the piece before is done with its own: at once if it is, else after the keys.
        auto send_queries = [&] {
          if (lane == 0) {
            sh.work[piece & 1] = w;
            const int rows = group * per_tile * 128;  // bytes of a query tile's half
            const int n = w.tokens > per_tile ? 2 : 1;
            mbar_expect_tx(&sh.q_full, 2 * rows * n);
            for (int i = 0; i < n; ++i) {
              const uint32_t dst_q = smem_addr(s_q) + i * kTile;
              tma_load_3d(dst_q, &map_q, &sh.q_full, 0, w.kv_head * group, w.token0 + i * per_tile);
              tma_load_3d(dst_q + kHalf, &map_q, &sh.q_full, 64, w.kv_head * group, w.token0 + i * per_tile);
            }
          }
          __syncwarp();
          ++piece;
        };
        const bool early = step == 0 && __all_sync(0xffffffffu, mbar_test(&sh.q_empty, (piece & 1) ^ 1));
        if (early) send_queries();
        // keys of `step`, values of the step before
        if (has) row = static_cast<int>(c.page_row(c.checked(id), w.kv_head));
        id = load_id(w, step + 1);
        const int parts = __popc(__ballot_sync(0xffffffffu, has)) + __popc(__ballot_sync(0xffffffffu, has_v));
        if (!wait_warp(&sh.pair_empty[slot], phase ^ 1, err)) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_expect_tx(&sh.pair_full[slot], parts * ps * 256);
        __syncwarp();
        const uint32_t dst = smem_addr(ring) + slot * 2 * kTile + lane * ps * 128;
        if (has_v) {
          tma_load_2d(dst, &map_v, &sh.pair_full[slot], 0, row_v);
          tma_load_2d(dst + kHalf, &map_v, &sh.pair_full[slot], 64, row_v);
        }
        if (has) {
          tma_load_2d(dst + kTile, &map_k, &sh.pair_full[slot], 0, row);
          tma_load_2d(dst + kTile + kHalf, &map_k, &sh.pair_full[slot], 64, row);
        }
        armed = (armed & ~(1u << slot)) | (phase << slot) | (1u << (16 + slot));
        if (step == 0 && !early) {
          if (!wait_warp(&sh.q_empty, (piece & 1) ^ 1, err)) {
            ok = false;
            break;
          }
          send_queries();
        }
        if (++slot == kStages) {
          slot = 0;
          phase ^= 1;
        }
        row_v = row;
        has_v = has;
        has = has_page(w, ++step);
      }
      if (!ok) *abort_flag = 1;
      // tell the others that the list has ended
      if (ok && !*abort_flag && wait_warp(&sh.q_empty, (piece & 1) ^ 1, err)) {
        if (lane == 0) {
          sh.work[piece & 1].token0 = -1;
          mbar_arrive(&sh.q_full);
        }
      } else {
        *abort_flag = 1;
        if (piece > 0) mbar_wait(&sh.q_full, (piece - 1) & 1, err);
      }
      // copies and arrivals in flight land before the CTA's shared memory goes away
      for (int s = 0; s < kStages; ++s) {
        if (!(armed & (1u << (16 + s)))) continue;
        mbar_wait(&sh.pair_full[s], (armed >> s) & 1u, err);
        if (!*abort_flag) mbar_wait(&sh.pair_empty[s], (armed >> s) & 1u, err);
      }
    } else if (warp == kMmaWarp) {
      // ------------------------------------------------------------------ MMA issue
      // Everything an MMA is given is the same in all lanes and looks so to the compiler (constants, loop
      // counters, warp reductions): operands that may differ cost it about 100 cycles per MMA.
      constexpr uint32_t idesc_s = instr_desc(false), idesc_o = instr_desc(true);
      const uint32_t q_desc = desc_kmajor(smem_addr(s_q)), k_desc = desc_kmajor(smem_addr(ring) + kTile),
                     v_desc = desc_mnmajor(smem_addr(ring));
      uint32_t it = 0;  // pairs taken so far
      uint32_t p_seen[2] = {0, 0}, o_seen[2] = {0, 0};
      auto wait_pair = [&] { return wait_warp(&sh.pair_full[it % kStages], (it / kStages) & 1, err); };
      auto issue_s = [&](int i) {  // S_i = Q_i K^T
        tc_fence_after();
        if (elect_one()) {
          const uint32_t qd = q_desc + i * (kTile >> 4), kd = k_desc + (it % kStages) * (2 * kTile >> 4);
#pragma unroll
          for (uint32_t kk = 0; kk < kD / 16; ++kk) {
            const uint32_t off = (kk >> 2) * (kHalf >> 4) + 2 * (kk & 3);  // 64-column half, 32 bytes per 16 columns
            mma_smem(kTmem + i * kBN, qd + off, kd + off, idesc_s, kk > 0 ? 1u : 0u);
          }
          mma_commit(&sh.s_full[i]);
        }
        __syncwarp();
      };
      auto issue_o = [&](int i, bool first, int half) {  // O_i (+)= P_i V over 64 keys
        tc_fence_after();
        if (elect_one()) {
          const uint32_t vd = v_desc + (it % kStages) * (2 * kTile >> 4);
#pragma unroll
          for (uint32_t kk = half * 4; kk < half * 4 + 4; ++kk)
            mma_tmem(kTmem + 256 + i * kBN, kTmem + i * kBN + kk * 8, vd + kk * (16 * 128 >> 4), idesc_o,
                     (!first || kk > 0) ? 1u : 0u);
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) mma_commit(bar);
        __syncwarp();
      };
      bool ok = true;
      for (int piece = 0; ok && !*abort_flag; ++piece) {
        if (!wait_warp(&sh.q_full, piece & 1, err)) {
          ok = false;
          break;
        }
        const int token0 = sh.work[piece & 1].token0, count0 = sh.work[piece & 1].count[0],
                  count1 = sh.work[piece & 1].count[1], left = sh.work[piece & 1].keys - sh.work[piece & 1].tile0 * kBN;
        if (token0 < 0) break;
        const int count[2] = {static_cast<int>(__reduce_max_sync(0xffffffffu, count0)),
                              static_cast<int>(__reduce_max_sync(0xffffffffu, count1))};
        const int steps = max(count[0], count[1]);
        if (!wait_pair()) {
          ok = false;
          break;
        }
#pragma unroll 1
        for (int i = 0; i < 2; ++i)
          if ((i ? count[1] : count[0]) > 0) issue_s(i);
        commit(&sh.pair_empty[it % kStages]);
        if (steps == 1) commit(&sh.q_empty);
        ++it;
        for (int step = 0; step < steps; ++step, ++it) {
          if (!wait_pair()) {
            ok = false;
            break;
          }
          const int valid = left - step * kBN;
          if (valid < kBN) {  // values past the block's keys: zeros, whatever is there
            const uint32_t va = smem_addr(ring) + (it % kStages) * 2 * kTile;
            for (int r = max(valid, 0) + (lane >> 3); r < kBN; r += 4)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(va + h * kHalf + r * 128 + (lane & 7) * 16), "r"(0)
                             : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (step >= count[i]) continue;
            if (step == 0) ok = wait_warp(&sh.o_empty[i], (o_seen[i]++ & 1) ^ 1, err);
            ok = ok && wait_warp(&sh.p_full[i][0], p_seen[i] & 1, err);
            if (!ok) break;
            issue_o(i, step == 0, 0);
            ok = wait_warp(&sh.p_full[i][1], p_seen[i]++ & 1, err);
            if (!ok) break;
            issue_o(i, step == 0, 1);
            // The next scores overwrite this tile's P: one thread's MMAs run in the order of their issue.
            if (step + 1 < count[i]) issue_s(i);
            else commit(&sh.o_full[i]);
          }
          if (!ok) break;
          commit(&sh.pair_empty[it % kStages]);
          if (step + 2 == steps) commit(&sh.q_empty);
        }
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ------------------------------------------------------------------ softmax, one row per thread
    const int i = warp >> 2;                                  // query tile
    const int r = (warp & 3) * 32 + lane;                     // row of it
    const int place = r / group, head = r - place * group;    // token and query head of the row
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = kTmem + lanes + i * kBN, t_o = kTmem + lanes + 256 + i * kBN;
    uint32_t s_seen = 0, o_seen = 0;
    bool ok = true;
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return wait_warp(bar, parity, err); };
    for (int piece = 0; ok && !*abort_flag; ++piece) {
      if (!wait_all(&sh.q_full, piece & 1)) {
        ok = false;
        break;
      }
      const Work w = sh.work[piece & 1];
      if (w.token0 < 0) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_empty);
      const int count = w.count[i];
      const int token = i * per_tile + place;
      const bool real = place < per_tile && token < w.tokens;
      int limit = 0;  // keys the row sees
      if (real) limit = kShared ? min(c.length(w.token0 + token), a.shared_keys) : max(0, w.position0 + token + 1);
      float m = -INFINITY, l = 0.f;
      bool odd = false;  // scores that are infinite or not a number: there is no softmax
      for (int step = 0; step < count && ok; ++step) {
        if (!wait_all(&sh.s_full[i], s_seen & 1)) {
          ok = false;
          break;
        }
        ++s_seen;
        tc_fence_after();
        uint32_t x[kBN];
#pragma unroll
        for (int b = 0; b < kBN / 32; ++b) tmem_ld32(t_s + b * 32, x + b * 32);
#pragma unroll
        for (int b = 0; b < kBN / 32; ++b) tmem_ld_wait(x + b * 32);
        const int seen = limit - (w.tile0 + step) * kBN;  // of this tile's keys
        if (__any_sync(0xffffffffu, seen < kBN)) {
#pragma unroll
          for (int e = 0; e < kBN; ++e)
            if (e >= seen) x[e] = __float_as_uint(-INFINITY);
        }
        float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < kBN / 2; ++e)
          t4[e & 3] = max3(t4[e & 3], __uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
        const float top = max3(max3(t4[0], t4[1], t4[2]), t4[3], t4[3]);
        odd = odd || !(top < INFINITY);
        const bool moves = top > m + kSlack || (m == -INFINITY && top > m);
        const float next = moves ? top : m;
        const float base = next == -INFINITY ? 0.f : next * kScaleLog2;
        if (step > 0 && __any_sync(0xffffffffu, moves)) {  // the products of the tile before have finished: S came after
          const float keep = exp2_approx(m * kScaleLog2 - base);
          l *= moves ? keep : 1.f;
#pragma unroll 1
          for (int b = 0; b < kD / 32; ++b) {
            uint32_t o[32];
            tmem_ld32(t_o + b * 32, o);
            tmem_ld_wait(o);
            if (moves) {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
            }
            tmem_st32(t_o + b * 32, o);
          }
        }
        m = next;
        const uint64_t scale2 = pair(kScaleLog2, kScaleLog2), base2 = pair(-base, -base);
        uint64_t sum2[2] = {0, 0};
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          uint32_t packed[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const uint64_t y = fma2(pair(__uint_as_float(x[b * 64 + 2 * e]), __uint_as_float(x[b * 64 + 2 * e + 1])), scale2, base2);
            float p0, p1;
            if ((e & 3) < kByCubic) {
              exp2_pair(y, &p0, &p1);
            } else {
              unpair(y, &p0, &p1);
              p0 = exp2_approx(p0);
              p1 = exp2_approx(p1);
            }
            sum2[e & 1] = add2(sum2[e & 1], pair(p0, p1));
            packed[e] = pack_bf16x2(p0, p1);
          }
          tmem_st32(t_s + b * 32, packed);
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          tc_fence_before();
          mbar_arrive(&sh.p_full[i][b]);
        }
        float s0, s1;
        unpair(add2(sum2[0], sum2[1]), &s0, &s1);
        l += s0 + s1;
      }
      if (!ok) break;
      if (count > 0 && !wait_all(&sh.o_full[i], o_seen & 1)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int64_t out_row = static_cast<int64_t>(w.token0 + token) * a.q_heads + w.kv_head * group + head;
      const RecordPlace at = record_place<kShared>(a, w.record, i * kBM + r, out_row);
      float* rec = at.rec;
      const bool sees = limit > w.tile0 * kBN;  // a key of this piece; else its weights are none
      const float inv = odd ? NAN : !sees ? 0.f : rec ? 1.f : 1.f / l;
      float largest = 0.f;  // NaN if something is
      if (count > 0) {
        // Rows go out through shared memory, 64 bytes of 8 rows per store: 16 bytes of 32 rows each would
        // take the L1 a cycle per row and store, 4000 for the two tiles.
        const int mine = real ? static_cast<int>(out_row) : -1;
        int rows[4];  // whose pieces this lane stores
#pragma unroll
        for (int q = 0; q < 4; ++q) rows[q] = __shfl_sync(0xffffffffu, mine, q * 8 + (lane >> 2));
        uint4* stage = sh.stage[warp];
        float large[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int b = 0; b < kD / 32; ++b) {
          uint32_t ob[32];
          tmem_ld32(t_o + b * 32, ob);
          tmem_ld_wait(ob);
          float f[32];
#pragma unroll
          for (int e = 0; e < 16; ++e)
            unpair(mul2(pair(__uint_as_float(ob[2 * e]), __uint_as_float(ob[2 * e + 1])), pair(inv, inv)), &f[2 * e],
                   &f[2 * e + 1]);
#pragma unroll
          for (int e = 0; e < 16; ++e) large[e & 3] = max3(large[e & 3], fabsf(f[2 * e]), fabsf(f[2 * e + 1]));
          if (rec) {
            if (real) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<float4*>(rec + at.vector(b * 8 + e)) =
                    make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) stage[lane * 4 + (e ^ (lane >> 1 & 3))] = pack8(f + 8 * e);
            __syncwarp();
            uint4 y[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int from = q * 8 + (lane >> 2);
              y[q] = stage[from * 4 + ((lane & 3) ^ (from >> 1 & 3))];
            }
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (rows[q] >= 0)
                *reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(rows[q]) * 128 + b * 32 + (lane & 3) * 8) = y[q];
          }
        }
        largest = max3(max3(large[0], large[1], large[2]), large[3], large[3]);
        tc_fence_before();
        mbar_arrive(&sh.o_empty[i]);
        ++o_seen;
      } else if (rec && real) {
        for (int e = 0; e < kD / 4; ++e) *reinterpret_cast<float4*>(rec + block_vector(e)) = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      if (rec && real) {
        rec[at.m] = m;
        rec[at.sum] = odd ? NAN : sees ? l : 0.f;
      }
      // rows with finite scores and something not finite
      const unsigned again = __ballot_sync(0xffffffffu, real && count > 0 && !odd && !(largest <= 3.4e38f));
      if (__builtin_expect(again != 0, 0)) {
        __syncwarp();
        if (lane == __ffs(again) - 1) {
          const int name = at.part ? ~(w.record * kBlockRows + i * kBM + r) : static_cast<int>(out_row);
          uint4* entry = place_of_row<kShared>(a, name);
          entry[0] = make_uint4(w.token0, w.position0, w.sequence, w.kv_head);
          entry[1] = make_uint4(w.tile0, count, again, sh.again[warp]);
          sh.again[warp] = name;
        }
      }
    }
    __syncwarp();
    for (int name = sh.again[warp]; name != kNoRow;) name = attend_again<kShared>(a, name);
    if (!ok) *abort_flag = 1;
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(kTmem), "r"(kTmemCols));
  }
}

// The blocks whose key tiles lie in more than one run: a CTA per (block, KV head, 4 rows), a warp per row.
constexpr int kMergeRows = 4;
__global__ void __launch_bounds__(kMergeRows * 32) paged_prefill_merge_kernel(const PrefillArgs a, int ctas) {
  const int block = blockIdx.x / a.c.kv_heads, kv_head = blockIdx.x - block * a.c.kv_heads;
  const int group = a.q_heads / a.c.kv_heads, per_tile = kBM / group;
  pdl_wait();
  const int blocks = min(__ldcg(&a.blocks[-1].x), a.most_blocks);  // loaded together; of a block that is none, nothing is used
  const int2 item = __ldcg(a.items + blockIdx.x);
  const int4 b = __ldcg(a.blocks + block);
  // whole, already written; or what a kernel that gave up on a wait left
  if (block >= blocks || item.x < 0 || item.y >= ctas || item.y < item.x >> 1) return;
  const int r = blockIdx.y * kMergeRows + (threadIdx.x >> 5), tile = r / kBM, in_tile = r - tile * kBM;
  const int place = in_tile / group, token = tile * per_tile + place;
  if (place >= per_tile || token >= b.y || b.x < 0 || b.x + token >= a.tokens) return;
  bf16* row = a.out + (static_cast<int64_t>(b.x + token) * a.q_heads + kv_head * group + in_tile - place * group) * 128;
  Parts parts[1];
  parts[0].blocks(a.records, r, item);
  if (b.z + token < 0)  // no position: no keys
    *reinterpret_cast<uint2*>(row + (threadIdx.x & 31) * 4) = make_uint2(0u, 0u);
  else
    join_parts<8>(parts, row);
}

// most blocks that `tokens` new tokens of `sequences` sequences make
int64_t most_blocks(int64_t tokens, int sequences, int group) {
  const int64_t per_block = 2 * (kBM / group);
  return std::min<int64_t>((tokens + sequences * (per_block - 1)) / per_block, tokens);
}

// Whether the key tiles are dealt in runs: where whole blocks may leave SMs idle for long, as far as the sizes say.
// (The kernel looks at the lengths too. A call that it would not cut up in any case needs no merge: 512 tokens on a
// table of no more 20.0 and 15.8 us.)
bool deal_in_runs(int64_t tokens, int sequences, int q_heads, int kv_heads, int64_t most_tiles) {
  const int64_t blocks = most_blocks(tokens, sequences, q_heads / kv_heads), sms = sm_count();
  return blocks <= kMaxListed && sequences <= kMaxListed && blocks * kv_heads < 2 * sms &&
         most_tiles * ((blocks * kv_heads + sms - 1) / sms) > kMergeTiles;
}

size_t list_bytes(size_t blocks, int kv_heads) {
  return (sizeof(int4) + blocks * (sizeof(int4) + kv_heads * sizeof(int2)) + 255) / 256 * 256;
}

}  // namespace

size_t paged_prefill_workspace_bytes(int64_t tokens, int sequences, int q_heads, int kv_heads) {
  if (!deal_in_runs(tokens, sequences, q_heads, kv_heads, INT32_MAX)) return 0;
  const size_t blocks = static_cast<size_t>(most_blocks(tokens, sequences, q_heads / kv_heads));
  return list_bytes(blocks, kv_heads) + static_cast<size_t>(sm_count()) * 2 * kBlockRecord * sizeof(float);
}

namespace {

struct Maps {
  CUtensorMap q, k, v;
};

// The tensor maps and arguments that both launches share.
cudaError_t prepare(const PagedCache& c, const void* q, const void* k_pages, const void* v_pages, int64_t tokens,
                    int q_heads, Maps* maps, PrefillArgs* a) {
  const int group = q_heads / c.kv_heads, page_size = 1 << c.page_shift;
  const int rows = static_cast<int>(static_cast<int64_t>(c.num_pages) * c.kv_heads * page_size);
  if (!make_map_3d(&maps->q, q, kD, q_heads, static_cast<int>(tokens), q_heads, group, 64, kBM / group) ||
      !make_map_2d(&maps->k, k_pages, rows, kD, page_size, 64) || !make_map_2d(&maps->v, v_pages, rows, kD, page_size, 64))
    return cudaErrorInvalidValue;
  *a = PrefillArgs{};
  a->c = c;
  a->q = static_cast<const bf16*>(q);
  a->k = static_cast<const bf16*>(k_pages);
  a->v = static_cast<const bf16*>(v_pages);
  a->tokens = static_cast<int>(tokens);
  a->q_heads = q_heads;
  return cudaSuccess;
}

template <bool kShared>
cudaError_t launch(int64_t grid, const Maps& maps, const PrefillArgs& a, cudaStream_t stream) {
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_shared_memory(paged_prefill_kernel<kShared>, kSmem, &allowed);
  if (e != cudaSuccess) return e;
  paged_prefill_kernel<kShared><<<static_cast<unsigned>(grid), kThreads, kSmem, stream>>>(maps.q, maps.k, maps.v, a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_prefill(const PagedCache& c, const void* q, const void* k_pages, const void* v_pages, void* out,
                                 int64_t tokens, int q_heads, void* workspace, cudaStream_t stream) {
  Maps maps;
  PrefillArgs a;
  cudaError_t e = prepare(c, q, k_pages, v_pages, tokens, q_heads, &maps, &a);
  if (e != cudaSuccess) return e;
  a.out = static_cast<bf16*>(out);
  const int64_t most_tiles = ((static_cast<int64_t>(c.max_pages) << c.page_shift) + kBN - 1) / kBN;
  const bool in_runs = deal_in_runs(tokens, c.sequences, q_heads, c.kv_heads, most_tiles);
  const int64_t blocks = most_blocks(tokens, c.sequences, q_heads / c.kv_heads);
  int64_t grid = blocks * c.kv_heads;
  if (in_runs) {
    a.blocks = static_cast<int4*>(workspace) + 1;
    a.most_blocks = static_cast<int>(blocks);
    a.items = reinterpret_cast<int2*>(a.blocks + blocks);
    a.records = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + list_bytes(blocks, c.kv_heads));
    grid *= most_tiles;
  }
  grid = std::min<int64_t>(grid, sm_count());
  e = launch<false>(grid, maps, a, stream);
  if (e != cudaSuccess || !in_runs) return e;
  return launch_pdl(paged_prefill_merge_kernel, dim3(static_cast<unsigned>(blocks * c.kv_heads), 2 * kBM / kMergeRows),
                    dim3(kMergeRows * 32), 0, stream, a, static_cast<int>(grid));
}

SharedKeys shared_keys_plan(const PagedCache& c, int q_heads) {
  SharedKeys p{};
  p.per_tile = kBM / (q_heads / c.kv_heads);
  p.tiles = ((c.prefix_count << c.page_shift) + kBN - 1) / kBN;
  const int64_t blocks = (c.sequences + 2 * p.per_tile - 1) / (2 * p.per_tile);
  p.items_count = blocks * c.kv_heads;
  p.units = p.items_count * p.tiles;
  p.ctas = static_cast<int>(std::min<int64_t>(p.units, sm_count()));
  return p;
}

cudaError_t launch_shared_keys(const PagedCache& c, const void* q, const void* k_pages, const void* v_pages, int q_heads,
                               const SharedKeys& plan, cudaStream_t stream) {
  Maps maps;
  PrefillArgs a;
  cudaError_t e = prepare(c, q, k_pages, v_pages, c.sequences, q_heads, &maps, &a);
  if (e != cudaSuccess) return e;
  a.records = plan.records;
  a.whole = plan.whole;
  a.items = plan.items;
  a.shared_keys = c.prefix_count << c.page_shift;
  return launch<true>(plan.ctas, maps, a, stream);
}

}  // namespace ipe
