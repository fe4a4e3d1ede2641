// Attention of many query rows over caches on tcgen05: prompts with a sliding window and first tokens that stay visible, and
// the rows of all sequences over a prefix that they share.
//
// A block has two halves, each with a query tile of 128 stacked rows (row x query head of one KV head), and walks its tokens in
// tiles of 64. Per tile and half: S = Q K^T into tensor memory, a thread per row takes its 64 scores out, makes the weights
// relative to its running maximum and puts them back as BF16 over the scores, from where they are the A operand of O += P V (V
// as it stands in the cache is that product's N-major B operand). Scores have two places, so that a tile's are computed while
// the last one's weights are made: 2 x (64 + 64 + 128) columns are all of the tensor memory.
//
// A running maximum may lag the true one by 2^8 (weights up to 256 are as exact in BF16 as those up to 1), as is published for
// attention on tensor memory, so that the outputs are hardly ever taken out to be rescaled; the sum is of the rounded weights, so
// that those used add up to one exactly and a row that one token dominates is that token's values. (Outputs are 0.0021 of their
// size off 64 bits, 0.0019 with the true maximum, whose weight is exactly 1, and 0.0017 rounded from 32-bit arithmetic; the true
// maximum costs 20 %. The prompts of uniform decoders, whose sum is of unrounded weights, follow the true one.)
//
// Tokens are a list of boxes of 32, first those of the sinks, then those of the window of the block's rows; two make a tile, so
// that a few sinks cost no tile of their own. What a box holds beyond its stretch is masked in the scores and cleared in V.
// An odd last query tile has both halves of its block, which then take every other tile of tokens. Where the blocks are
// fewer than the SMs, those of a cluster share the tokens of the same rows and join their sums through distributed shared
// memory; a prefix is also cut into stretches that leave partial results (span_choice.hpp).
//
// What bounds it: the softmax warps' own chain. A tile takes a pair of halves some 2200 cycles, of which the exponentials are
// 1024 (16 a cycle), the products 1280; by leaving parts out in copies, everything but the softmax takes 1200. Two warps a
// scheduler share the exponentials: alone a warp needs 820 cycles for its 64, beside the other 1200. Sixteen softmax warps, two a
// row by columns or by turns, came out the same; so did tiles of 128 tokens with one place for the scores, whose halves fall
// into step and then wait for their products together. 2048 rows of 32 / 8 heads behind 6144 tokens, window 2048: 97 to 100 us = 690
// to 709 TFLOP/s (289 us by the few-row kernel); 256 blocks are 1.73 waves, which costs 13 %, and a block some 9 us to start and to leave.
//
// Roles of the twelve warps: 0-3 and 4-7 the weights of one half each, 8 the copies, 9 and 10 the MMAs of one half each, 11 the
// tensor memory. A stage of the ring of four holds a tile's V and the K of the half's next scores. Every wait is bounded: a role
// whose wait runs out raises `abort`, which every other wait polls; when all roles have left, the copies and MMAs in flight are
// waited for (bounded), the block's rows come out as NaN and the tensor memory is freed. The host can ask how often that happened.
#include "span_attention.cuh"

#include "cluster.cuh"
#include "per_device.hpp"
#include "prompt_attention.cuh"

#include <algorithm>

namespace ei {
namespace {

constexpr int kDim = 128;
constexpr int kThreads = 384;
constexpr int kHalfBytes = kSpanTile * 128;  // 64 values of a tile's tokens
constexpr int kBufferBytes = 2 * kHalfBytes;
constexpr int kBoxBytes = kSpanBox * 128;
constexpr int kBoxes = kSpanTile / kSpanBox;
constexpr int kStages = 4;  // each a tile's V and the K that the half's next scores are made of
constexpr int kStageBytes = 2 * kBufferBytes;
constexpr int kQueryBytes = 2 * kSpanRows * 128;
constexpr float kSlack = 8.0f;  // powers of two
// A weight is 2^(s scale - m scale) by one multiplication and addition, with m scale rounded. That rounding is the same for a
// row's equal scores, but from 2^31 on it soon reaches the exponents' range: the row's largest weight, 1, would be 0 or infinite.
// Scores of that size are multiples of 128, so that any but those equal to the maximum weigh nothing at a power of two of about
// the scale as well, and with that the products are exact.
constexpr float kFarScore = 2147483648.0f, kFarScale = 0.125f;  // rsqrt(128) log2(e) = 0.1275
constexpr size_t kStateBytes = 512;
// Queries, first K of each half, ring, state.
constexpr size_t kSpanSharedBytes = size_t(2) * kQueryBytes + 2 * kBufferBytes + size_t(kStages) * kStageBytes + 1024 + kStateBytes;
static_assert(kBoxes == 2, "a tile's boxes are looked at one by one");
static_assert(kSpanSharedBytes <= 227 * 1024, "a block's buffers fit an SM");

struct SpanShared {
  uint64_t full[kStages], empty[kStages];
  uint64_t first;                     // the first K
  uint64_t queries[2];                // a query tile is in shared memory
  uint64_t scores[2][2];              // [half][tile & 1]: S computed, and the product of the tile before the last one added
  uint64_t weights[2][2];             // [half][tile & 1]: P written
  uint64_t finished[2];               // of a half: all products added
  uint64_t done;                      // every MMA issued has completed
  uint32_t tmem_base;
  volatile int abort;
  int issued, query_tiles;            // stages, and a bit for each query tile, whose copies were requested
};
static_assert(sizeof(SpanShared) <= kStateBytes, "the block's state lies behind the ring");

__device__ __forceinline__ void tmem_request32(uint32_t address, uint32_t* r) {
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(address)
      : "memory");
}
// The lowest `count` bits, of any sign and size.
__device__ __forceinline__ uint32_t below(int count) { return count >= 32 ? 0xffffffffu : count <= 0 ? 0u : (1u << count) - 1; }
// Waits for the loads requested; the registers pass through so that nothing reads them earlier.
__device__ __forceinline__ void tmem_loaded32(uint32_t* r) {
  __syncwarp();
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                 "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                 "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}

__device__ uint32_t expired_waits;  // blocks that have given up since the library was loaded

__global__ void __launch_bounds__(kThreads, 1) span_attention_kernel(const __grid_constant__ SpanAttentionParams p) {
  extern __shared__ unsigned char span_smem_raw[];
  unsigned char* const smem = span_smem_raw + ((1024u - (smem_address(span_smem_raw) & 1023u)) & 1023u);
  unsigned char* const first_keys = smem + 2 * kQueryBytes;
  unsigned char* const ring = first_keys + 2 * kBufferBytes;
  SpanShared* const sh = reinterpret_cast<SpanShared*>(ring + kStages * kStageBytes);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 9 * 32) {
    prefetch_map(&p.k_tile_map), prefetch_map(&p.v_tile_map);
    if (p.copied_queries) prefetch_map(&p.q_map);  // encoded only then
  }
  const int kv_head = blockIdx.x, sequence = blockIdx.z;
  const int group = p.heads / p.kv_heads, stacked = p.rows * group;

  // ---- what this block does ----
  int length = p.lengths ? p.lengths[sequence] : p.length;
  if (length < 0 || length > p.capacity) length = 0;
  const uint32_t rank = cluster_rank(), blocks = cluster_size();
  const int y = blockIdx.y / blocks;
  int first_tile;             // query tile of half 0
  bool shared_tokens = true;  // both halves read every tile of tokens (of two query tiles); else every other (of one)
  int partial_index = 0;      // of this stretch's result among the prefix's
  int box_begin = 0, low = 0, sink_end = 0, sink_boxes = 0, box_end, end;
  int first_position0, last_position0, first_position1, last_position1;  // of the halves' rows
  const int base = length - p.rows;
  if (p.together) {
    int splits = p.splits.pair_splits;
    if (y < p.splits.pairs * splits) {
      first_tile = y / splits * 2;
      partial_index = y - first_tile / 2 * splits;
    } else {
      first_tile = p.splits.pairs * 2;
      shared_tokens = false;
      splits = p.splits.single_splits;
      partial_index = y - p.splits.pairs * p.splits.pair_splits;
    }
    const int tiles = (length + kSpanTile - 1) / kSpanTile;
    box_begin = int((long long)tiles * partial_index / splits) * kBoxes;
    end = length;
    box_end = min(int((long long)tiles * (partial_index + 1) / splits) * kBoxes, (end + kSpanBox - 1) / kSpanBox);
    first_position0 = first_position1 = last_position0 = last_position1 = length - 1;
  } else {
    first_tile = (int(gridDim.y / blocks) - 1 - y) * 2;  // the longest histories first
    shared_tokens = (first_tile + 1) * kSpanRows < stacked;
    auto position_of = [&](int i) { return base + min(i, stacked - 1) / group; };
    const int from = first_tile * kSpanRows;
    first_position0 = position_of(from), last_position0 = position_of(from + kSpanRows - 1);
    first_position1 = shared_tokens ? position_of(from + kSpanRows) : first_position0;
    last_position1 = shared_tokens ? position_of(from + 2 * kSpanRows - 1) : last_position0;
    end = max(0, last_position1 + 1);
    low = max(0, min(first_position0 - p.window + 1, end));
    sink_end = min(p.sinks, low);
    sink_boxes = (sink_end + kSpanBox - 1) / kSpanBox;
    box_end = sink_boxes + (end - low + kSpanBox - 1) / kSpanBox;
  }
  {
    // This block's share of the cluster's tiles.
    const int tiles = (box_end - box_begin + kBoxes - 1) / kBoxes, begin = box_begin;
    box_begin = begin + int((long long)tiles * rank / blocks) * kBoxes;
    box_end = min(box_end, begin + int((long long)tiles * (rank + 1) / blocks) * kBoxes);
  }
  const int items = (max(0, box_end - box_begin) + kBoxes - 1) / kBoxes;  // tiles of tokens
  auto start_of = [&](int box) { return box < sink_boxes ? box * kSpanBox : low + (box - sink_boxes) * kSpanBox; };
  auto stop_of = [&](int box) { return box >= box_end ? 0 : box < sink_boxes ? sink_end : end; };
  // Tiles that a half takes: all up to its last row's position, or every other.
  auto tiles_of = [&](int half) {
    if (!shared_tokens) return (items + 1 - half) / 2;
    if (p.together) return items;
    const int position = half ? last_position1 : last_position0;
    if (position < 0) return 0;
    const int boxes = position < low ? (min(sink_end, position + 1) + kSpanBox - 1) / kSpanBox : sink_boxes + (position - low) / kSpanBox + 1;
    return min(items, (max(0, boxes - box_begin) + kBoxes - 1) / kBoxes);
  };
  const int tiles0 = tiles_of(0), tiles1 = tiles_of(1);
  auto item_of = [&](int half, int t) { return shared_tokens ? t : 2 * t + half; };

  auto query_tile_of = [&](int half) { return shared_tokens ? first_tile + half : first_tile; };
  const long long row0 = (long long)sequence * p.rows;
  const int most = shared_tokens ? max(tiles0, tiles1) : items, ahead = shared_tokens ? 1 : 2;
  if (threadIdx.x == 8 * 32) {
    for (int b = 0; b < kStages; ++b) {
      mbarrier_init(&sh->full[b], 1);
      mbarrier_init(&sh->empty[b], shared_tokens ? 2 : 1);
    }
    mbarrier_init(&sh->first, 1);
    for (int i = 0; i < 2; ++i) {
      mbarrier_init(&sh->queries[i], p.copied_queries ? 1 : 4);
      mbarrier_init(&sh->finished[i], 1);
      for (int place = 0; place < 2; ++place) {
        mbarrier_init(&sh->scores[i][place], 1);
        mbarrier_init(&sh->weights[i][place], 4);
      }
    }
    mbarrier_init(&sh->done, 2);
    sh->abort = 0;
    sh->issued = sh->query_tiles = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 11) tmem_alloc(&sh->tmem_base, 512);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = sh->tmem_base;
  if (p.together) {  // launched in plain stream order: the wait is over at once
    grid_dependency_wait();
    grid_launch_dependents();
  }
  const uint32_t wait_limit = p.wait_limit ? p.wait_limit : kTmaWaitLimit;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbarrier_test_wait(bar, parity)) return true;
    for (uint32_t polls = 0; polls < wait_limit; ++polls) {
      if (mbarrier_try_wait(bar, parity)) return true;
      if (sh->abort) return false;
    }
    sh->abort = 1;
    return false;
  };
  // The same for a whole warp.
  auto wait_all = [&](uint64_t* bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, mbarrier_test_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, wait(bar, parity)) != 0;
  };

  // The row of a softmax thread.
  const int half = (warp >> 2) & 1, row_of_tile = threadIdx.x & (kSpanRows - 1);
  const int index = query_tile_of(half) * kSpanRows + row_of_tile;
  const bool live = warp < 8 && index < stacked;
  const int row = live ? index / group : 0, head = kv_head * group + (live ? index - row * group : 0);
  auto partial_of_row = [&] {
    return p.partial + ((size_t(partial_index) * p.sequences * p.rows + row0 + row) * p.heads + head) * kStepPartial;
  };
  auto out_of_row = [&] { return p.out + (row0 + row) * p.out_stride + size_t(head) * kDim; };

  // Of the row: running maximum, sum of the weights relative to it.
  float maximum = -INFINITY, sum = 0.0f;
  const float exponent_scale = rsqrtf(float(kDim)) * kLog2e;
  // Results of other blocks of the cluster, or of the other half, belong to the same rows.
  const bool join = blocks > 1 || !shared_tokens;
  const int own_tiles = ((warp >> 2) & 1) ? tiles1 : tiles0;

  if (warp < 8) {
    // ---- weights: thread = query row ----
    if (!p.copied_queries && (shared_tokens || half == 0)) {
      unsigned char* const own = smem + half * kQueryBytes + row_of_tile * 128;
      const bf16* q = p.q + (row0 + row) * p.q_stride + size_t(head) * kDim;
#pragma unroll 1
      for (int part = 0; part < 2; ++part) {
        uint4 held[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) held[i] = live ? reinterpret_cast<const uint4*>(q + part * 64)[i] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(own + part * kSpanRows * 128 + ((i ^ (row_of_tile & 7)) << 4)) = held[i];
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbarrier_arrive(&sh->queries[half]);
    }
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t places = tmem + lanes + half * 256, outputs = places + 128;
    const int last = p.together ? length - 1 : base + row;
    const bool some_live = __any_sync(0xffffffffu, live);
    const int tiles = own_tiles;
    // Boxes that every row of the half sees whole.
    const int clean_begin = sink_boxes + (max(0, (half ? last_position1 : last_position0) - p.window + 1 - low) + kSpanBox - 1) / kSpanBox;
    const int clean_end = sink_boxes + max(0, min(end, (half ? first_position1 : first_position0) + 1) - low) / kSpanBox;
    bool ok = true;
    for (int t = 0; t < tiles; ++t) {
      const int item = item_of(half, t), box0 = box_begin + item * kBoxes;
      const bool clean = box0 >= clean_begin && box0 + kBoxes <= clean_end;
      const uint32_t at = places + (t & 1) * 64;
      ok = wait_all(&sh->scores[half][t & 1], (t >> 1) & 1);
      if (!ok) break;
      tcgen05_fence_after();
      uint32_t s[2][32];
      float2 scales = make_float2(exponent_scale, exponent_scale), shifts = make_float2(0.0f, 0.0f);
      float rescale = 1.0f;
      bool moved_some = false;
      if (some_live) {
        tmem_request32(at, s[0]);
        tmem_request32(at + 32, s[1]);
        tmem_loaded32(s[0]);
        tmem_loaded32(s[1]);
        float tops[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!clean) {
            const int start = start_of(box0 + i);
            const uint32_t seen = below(min(stop_of(box0 + i), last + 1) - start) &
                                  (below(p.sinks - start) | ~below(last - p.window + 1 - start));
#pragma unroll
            for (int j = 0; j < 32; ++j) s[i][j] = seen >> j & 1 ? s[i][j] : 0xff800000u;
          }
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            float& most = tops[2 * i + part];
            most = __uint_as_float(s[i][16 * part]);
#pragma unroll
            for (int j = 1; j < 16; ++j) most = fmaxf(most, __uint_as_float(s[i][16 * part + j]));
          }
        }
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const bool moved = maximum == -INFINITY ? top != -INFINITY : (top - maximum) * exponent_scale > kSlack;
        const float previous = maximum;
        if (moved) maximum = top;
        // A row with nothing visible yet keeps -inf; 0 as the exponent's base then makes every weight 0.
        const float reference = maximum == -INFINITY ? 0.0f : maximum;
        if (fabsf(reference) >= kFarScore) scales.x = scales.y = kFarScale;
        shifts.x = shifts.y = -reference * scales.x;
        // From one rounded base of the exponents to the next.
        if (moved) rescale = power_of_two(__fadd_rn(__fmul_rn(previous, scales.x), shifts.x));
        moved_some = __any_sync(0xffffffffu, moved);
      }
      if (!clean && (stop_of(box0) - start_of(box0) < kSpanBox || stop_of(box0 + 1) - start_of(box0 + 1) < kSpanBox)) {
        // V's rows that are no token of the list are cleared: nothing there may pass through a zero weight. (Both halves'
        // warps do it before they hand over their weights, with the same zeros.)
        ok = wait_all(&sh->full[item % kStages], (item / kStages) & 1);
        if (!ok) break;
        unsigned char* values = ring + (item % kStages) * kStageBytes;
#pragma unroll 1
        for (int b = 0; b < kBoxes; ++b) {
          const int have = min(kSpanBox, max(0, stop_of(box0 + b) - start_of(box0 + b)));
          for (int i = row_of_tile; i < (kSpanBox - have) * 16; i += kSpanRows)
            *reinterpret_cast<uint4*>(values + (i & 1) * kHalfBytes + (b * kSpanBox + have + (i >> 4)) * 128 + ((i >> 1) & 7) * 16) =
                make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      if (some_live) {
        // In groups of 16, a group's exponentials ahead of the conversions of the one before it: taken pair by pair, each
        // conversion waited for its own two exponentials, 20 cycles a value instead of 8.
        float2 parts[2] = {};
        uint32_t packed[2][16];
        auto exponentials = [&](int group) {
          uint32_t* const v = &s[group >> 1][(group & 1) * 16];
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float2 x = fma_pair(make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), scales, shifts);
            v[j] = __float_as_uint(x.x), v[j + 1] = __float_as_uint(x.y);
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+r"(v[j]));
        };
        auto convert = [&](int group) {
          const uint32_t* const v = &s[group >> 1][(group & 1) * 16];
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            uint32_t both;
            asm volatile("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(both) : "f"(__uint_as_float(v[j + 1])), "f"(__uint_as_float(v[j])));
            packed[group >> 1][(group & 1) * 8 + j / 2] = both;
            parts[j / 2 & 1] = add_pair(parts[j / 2 & 1], make_float2(bf16_lo(both), bf16_hi(both)));
          }
        };
        exponentials(0);
        exponentials(1);
        convert(0);
        exponentials(2);
        convert(1);
        tmem_store16(at, packed[0]);
        exponentials(3);
        convert(2);
        convert(3);
        tmem_store16(at + 16, packed[1]);
        const float2 total = add_pair(parts[0], parts[1]);
        sum = sum * rescale + (total.x + total.y);
      }
      if (moved_some) {
        // The product of the tile before is added when the scores of the next one stand (or would, behind the last).
        ok = t == 0 || wait_all(&sh->scores[half][(t + 1) & 1], ((t + 1) >> 1) & 1);
        if (!ok) break;
        if (t > 0) {
          tcgen05_fence_after();
#pragma unroll 1
          for (int i = 0; i < 8; ++i) {
            uint32_t a[16];
            tmem_request16(outputs + i * 16, a);
            tmem_loaded(a);
#pragma unroll
            for (int j = 0; j < 16; ++j) a[j] = __float_as_uint(__uint_as_float(a[j]) * rescale);
            tmem_store16(outputs + i * 16, a);
          }
        }
      }
      tmem_stored();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbarrier_arrive(&sh->weights[half][t & 1]);
    }
    const bool any = tiles > 0;
    if (any) ok = ok && wait_all(&sh->finished[half], 0);
    if (ok && !join) {
      tcgen05_fence_after();
      float* const partial = partial_of_row();
      const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
      // Rows leave in whole lines, four at a time, by way of shared memory: queries of the half that are done with. A thread that stores its own row's 16 bytes at a time touches 32 lines at once:
      // 5.6 us instead of 1.5 for a block's partial results.
      unsigned char* const staged = smem + half * kQueryBytes + (warp & 3) * 4096;
      const uint64_t own_row = p.together ? reinterpret_cast<uint64_t>(partial) : reinterpret_cast<uint64_t>(out_of_row());
      const int parts = p.together ? 4 : 2;  // 128 bytes of a row each
      const uint32_t lives = __ballot_sync(0xffffffffu, live);
#pragma unroll 1
      for (int part = 0; part < parts; ++part) {
        uint32_t line[32];
        if (p.together) {
          if (any) {
            tmem_request32(outputs + part * 32, line);
            tmem_loaded32(line);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t v[16];
            if (any) {
              tmem_request16(outputs + part * 64 + i * 16, v);
              tmem_loaded(v);
            }
#pragma unroll
            for (int j = 0; j < 16; j += 2)  // an inverse of 0: nothing visible, whatever the sums are
              line[i * 8 + j / 2] = inverse == 0.0f ? 0u : pack_bf16(__uint_as_float(v[j]) * inverse, __uint_as_float(v[j + 1]) * inverse);
          }
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4*>(staged + lane * 128 + ((j ^ (lane & 7)) << 4)) =
              any ? make_uint4(line[4 * j], line[4 * j + 1], line[4 * j + 2], line[4 * j + 3]) : make_uint4(0, 0, 0, 0);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = 4 * j + (lane >> 3);
          const uint64_t to = __shfl_sync(0xffffffffu, own_row, r);
          if (lives >> r & 1)
            reinterpret_cast<uint4*>(to)[part * 8 + (lane & 7)] = *reinterpret_cast<const uint4*>(staged + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
        }
      }
      if (live && p.together) *reinterpret_cast<float2*>(partial + kDim) = make_float2(maximum * exponent_scale, sum);
    }
  } else if (warp == 8) {
    // ---- copies ----
    if (lane == 0) {
      // A tile whose tokens are neighbours is one copy, one that begins with sinks and goes on with the window four. (Of boxes of 32
      // tokens and half a head alone, a stage took eight, some 800 cycles to ask for.)
      auto copy = [&](const CUtensorMap& tiles, const CUtensorMap& boxes, int item, unsigned char* to, uint64_t* bar) {
        const int box = box_begin + item * kBoxes;
        if (box + 1 < sink_boxes || box >= sink_boxes || box + 1 >= box_end) {
          tma_load_5d(to, &tiles, 0, start_of(box), 0, kv_head, sequence, bar);
        } else {
          for (int j = 0; j < kBoxes; ++j)
            for (int part = 0; part < 2; ++part)
              tma_load_5d(to + part * kHalfBytes + j * kBoxBytes, &boxes, 0, start_of(box + j), part, kv_head, sequence, bar);
        }
      };
      if (p.copied_queries)
        for (int i = 0; i < (shared_tokens ? 2 : 1); ++i) {
          if ((i ? tiles1 : tiles0) == 0) continue;
          mbarrier_expect_tx(&sh->queries[i], uint32_t(kQueryBytes));
          for (int part = 0; part < 2; ++part)
            tma_load_5d(smem + i * kQueryBytes + part * kSpanRows * 128, &p.q_map, 0, 0, int(row0) + query_tile_of(i) * kSpanRows / group, part,
                        kv_head, &sh->queries[i]);
          sh->query_tiles |= 1 << i;
        }
      if (most > 0) {
        const bool faulty = sequence == 0 && rank == blocks - 1;
        mbarrier_expect_tx(&sh->first, uint32_t(min(ahead, most)) * kBufferBytes + (faulty ? p.fault_tx : 0));
        for (int i = 0; i < min(ahead, most); ++i) copy(p.k_tile_map, p.k_map, i, first_keys + i * kBufferBytes, &sh->first);
        sh->issued = 1;
      }
      for (int i = 0; i < most; ++i) {
        const int b = i % kStages;
        if (i >= kStages && !wait(&sh->empty[b], (i / kStages - 1) & 1)) break;
        mbarrier_expect_tx(&sh->full[b], uint32_t(i + ahead < most ? 2 : 1) * kBufferBytes);
        copy(p.v_tile_map, p.v_map, i, ring + b * kStageBytes, &sh->full[b]);
        if (i + ahead < most) copy(p.k_tile_map, p.k_map, i + ahead, ring + b * kStageBytes + kBufferBytes, &sh->full[b]);
        sh->issued = i + 2;
      }
    }
  } else if (warp < 11) {
    // ---- MMAs of one half ----
    const int mine = warp - 9, n = mine ? tiles1 : tiles0;
    const uint32_t leader = elect_one();
    constexpr uint32_t kScores = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(kSpanTile >> 3) << 17) | (uint32_t(kSpanRows >> 4) << 24);
    // The values' 128 columns are N-major: bit 16.
    constexpr uint32_t kOutputs = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (uint32_t(kDim >> 3) << 17) | (uint32_t(kSpanRows >> 4) << 24);
    const uint32_t query_desc = umma_desc_low(smem_address(smem) + (shared_tokens ? mine : 0) * kQueryBytes);
    const uint32_t outputs = tmem + mine * 256 + 128;
    // A loop of few instructions: with a barrier each for K, V and their buffers it took 1450 cycles a tile with nothing to wait
    // for, more than the products themselves.
    auto score = [&](const unsigned char* from, int place) {
      const uint32_t keys = umma_desc_low(smem_address(from));
#pragma unroll
      for (int k = 0; k < kDim / 16; ++k)
        umma_bf16_ss(tmem + mine * 256 + place * 64, query_desc + (k >> 2) * (kSpanRows * 128 >> 4) + (k & 3) * 2,
                     keys + (k >> 2) * (kHalfBytes >> 4) + (k & 3) * 2, kUmmaDescHigh, kScores, k > 0 ? 1u : 0u);
    };
    bool ok = n == 0 || (wait_all(&sh->queries[shared_tokens ? mine : 0], 0) && wait_all(&sh->first, 0));
    if (n > 0 && ok) {
      tcgen05_fence_after();
      if (leader) {
        score(first_keys + (shared_tokens ? 0 : mine) * kBufferBytes, 0);
        tcgen05_commit(&sh->scores[mine][0]);
      }
    }
    for (int i = shared_tokens ? 0 : mine, t = 0; i < most && ok; i += shared_tokens ? 1 : 2, ++t) {
      const int b = i % kStages;
      unsigned char* const stage = ring + b * kStageBytes;
      ok = wait_all(&sh->full[b], (i / kStages) & 1);
      if (!ok) break;
      if (t >= n) {
        // Both halves count this stage and only the other sees it: given back when it is there, not earlier, so that an arrival
        // cannot count for its previous tile.
        if (leader) mbarrier_arrive(&sh->empty[b]);
        continue;
      }
      tcgen05_fence_after();
      if (leader) {
        // The scores of the half's next tile, ahead of this one's product: they have a place of their own.
        if (t + 1 < n) score(stage + kBufferBytes, (t + 1) & 1);
        tcgen05_commit(&sh->scores[mine][(t + 1) & 1]);
      }
      ok = wait_all(&sh->weights[mine][t & 1], (t >> 1) & 1);
      if (!ok) break;
      tcgen05_fence_after();
      if (leader) {
        // 64 values of a token are a 128-byte row; the other 64 values' rows kHalfBytes on; eight tokens 1024 bytes.
        const uint32_t values = ((smem_address(stage) & 0x3ffffu) >> 4) | (uint32_t(kHalfBytes >> 4) << 16);
#pragma unroll
        for (int k = 0; k < kSpanTile / 16; ++k)
          umma_bf16_ts(outputs, tmem + mine * 256 + (t & 1) * 64 + k * 8, values + k * (16 * 128 >> 4), kUmmaDescHigh, kOutputs,
                       k > 0 ? 1u : uint32_t(t > 0));
        tcgen05_commit(&sh->empty[b]);
        if (t + 1 == n) tcgen05_commit(&sh->finished[mine]);
      }
    }
    if (leader) tcgen05_commit(&sh->done);
  }
  tcgen05_fence_before();
  __syncthreads();
  if (sh->abort) {  // no role is left to raise it: block-uniform
    if (threadIdx.x == 0) {
      atomicAdd(&expired_waits, 1u);
      for (uint32_t polls = 0; polls < wait_limit && !mbarrier_try_wait(&sh->done, 0); ++polls) {
      }
      for (int i = 0; i < 2; ++i)
        if (sh->query_tiles >> i & 1) mbarrier_wait(&sh->queries[i], 0, wait_limit);
      if (sh->issued > 0) mbarrier_wait(&sh->first, 0, wait_limit);
      for (int i = max(0, sh->issued - 1 - kStages); i < sh->issued - 1; ++i) mbarrier_wait(&sh->full[i % kStages], (i / kStages) & 1, wait_limit);
    }
    __syncthreads();
    if (live && !join) {
      const uint32_t nan = 0x7fffffffu;
      float* const partial = partial_of_row();
      bf16* const out = out_of_row();
      for (int j = 0; j < kDim; ++j) {
        if (p.together) partial[j] = __uint_as_float(nan);
        else reinterpret_cast<uint16_t*>(out)[j] = 0x7fff;
      }
      if (p.together) *reinterpret_cast<float2*>(partial + kDim) = make_float2(0.0f, __uint_as_float(nan));
    }
  }
  tcgen05_fence_after();
  if (join) {
    // Every row's sums, maximum and sum into shared memory (all copies and products are done with it), then a warp a row: its
    // parts relative to their common maximum, in the order of the blocks.
    unsigned char* const area = first_keys;  // [half][row][128] FP32, a row's 16-byte pieces turned by the row
    float2* const stats = reinterpret_cast<float2*>(area + 2 * kSpanRows * kDim * 4);
    const int place = half * kSpanRows + row_of_tile;
    if (warp < 8) {
      const uint32_t outputs = tmem + (uint32_t((warp & 3) * 32) << 16) + half * 256 + 128;
#pragma unroll 1
      for (int part = 0; part < 4; ++part) {
        uint32_t v[32];
        if (own_tiles > 0) {
          tmem_request32(outputs + part * 32, v);
          tmem_loaded32(v);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4*>(area + place * (kDim * 4) + (((part * 8 + j) ^ (row_of_tile & 31)) << 4)) =
              own_tiles > 0 ? make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]) : make_uint4(0, 0, 0, 0);
      }
      stats[place] = sh->abort ? make_float2(0.0f, __uint_as_float(0x7fffffffu)) : make_float2(maximum * exponent_scale, sum);
    }
    if (blocks > 1) cluster_sync();
    else __syncthreads();
    const int rows_here = shared_tokens ? 2 * kSpanRows : kSpanRows, sources = int(blocks) * (shared_tokens ? 1 : 2);
    for (int r = int(rank) * (kThreads / 32) + warp; r < rows_here; r += int(blocks) * (kThreads / 32)) {
      const int i = first_tile * kSpanRows + r;
      if (i >= stacked) break;  // whole warps
      const int source_place = [&](int source) { return shared_tokens ? r : (source & 1) * kSpanRows + r; }(lane);
      auto block_of = [&](int source) { return uint32_t(shared_tokens ? source : source >> 1); };
      float2 mine = make_float2(-INFINITY, 0.0f);
      if (lane < sources) mine = remote_float2(stats + source_place, block_of(lane));
      const float top = warp_max(mine.x);
      const float factor = mine.y == 0.0f ? 0.0f : power_of_two(mine.x - top);  // nothing visible there counts nothing
      const float total = warp_sum(mine.y == 0.0f ? 0.0f : mine.y * factor);
      float4 out4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
      for (int source = 0; source < sources; ++source) {
        const float weight = __shfl_sync(0xffffffffu, factor, source);
        const int from = shared_tokens ? r : (source & 1) * kSpanRows + r;
        const float4 v = remote_float4(area + from * (kDim * 4) + ((lane ^ (r & 31)) << 4), block_of(source));
        if (weight == 0.0f) continue;
        out4.x = fmaf(v.x, weight, out4.x), out4.y = fmaf(v.y, weight, out4.y);
        out4.z = fmaf(v.z, weight, out4.z), out4.w = fmaf(v.w, weight, out4.w);
      }
      const int to_row = i / group, to_head = kv_head * group + i - to_row * group;
      if (p.together) {
        float* const to = p.partial + ((size_t(partial_index) * p.sequences * p.rows + row0 + to_row) * p.heads + to_head) * kStepPartial;
        reinterpret_cast<float4*>(to)[lane] = out4;
        if (lane == 0) *reinterpret_cast<float2*>(to + kDim) = make_float2(top, total);
      } else {
        const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
        uint2 packed = make_uint2(0u, 0u);
        if (inverse != 0.0f) packed = make_uint2(pack_bf16(out4.x * inverse, out4.y * inverse), pack_bf16(out4.z * inverse, out4.w * inverse));
        reinterpret_cast<uint2*>(p.out + (row0 + to_row) * p.out_stride + size_t(to_head) * kDim)[lane] = packed;
      }
    }
    if (blocks > 1) cluster_sync();  // no block leaves while another reads its shared memory
  }
  if (warp == 11) {
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

void launch_span_attention(const SpanAttentionParams& given, cudaStream_t stream) {
  static PerDevice<bool> devices;
  int device = 0;
  EI_CUDA(cudaGetDevice(&device));
  devices.get(device, [] {
    EI_CUDA(cudaFuncSetAttribute(span_attention_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSpanSharedBytes)));
    return true;
  });
  SpanAttentionParams p = given;
  const int group = p.heads / p.kv_heads;
  const long long all_rows = (long long)p.rows * p.sequences;
  p.copied_queries = p.q_stride < (1ll << 31) && all_rows < (1ll << 31) &&
                     encode_query_map(&p.q_map, p.q, int(all_rows), int(p.q_stride), group, p.kv_heads, kDim);
  const size_t query_tiles = (size_t(p.rows) * group + kSpanRows - 1) / kSpanRows;
  const unsigned clusters = p.together ? unsigned(p.splits.clusters()) : unsigned((query_tiles + 1) / 2);
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(unsigned(p.kv_heads), clusters * unsigned(p.cluster), unsigned(p.sequences));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = kSpanSharedBytes;
  config.stream = stream;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = cluster.val.clusterDim.z = 1;
  cluster.val.clusterDim.y = unsigned(p.cluster);
  config.attrs = &cluster;
  config.numAttrs = 1;
  check_cuda(cudaLaunchKernelEx(&config, span_attention_kernel, p), "cudaLaunchKernelEx");
}

uint32_t span_expired_waits(cudaStream_t stream) {
  uint32_t count = 0;
  EI_CUDA(cudaMemcpyFromSymbolAsync(&count, expired_waits, sizeof(count), 0, cudaMemcpyDeviceToHost, stream));
  EI_CUDA(cudaStreamSynchronize(stream));
  return count;
}

}  // namespace ei
