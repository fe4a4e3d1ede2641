// Attention of few query rows over a batch of caches: a sliding window with first tokens that stay visible, the own part of
// sequences that share a prefix, and attention that also reports the weight every cached token received.
//
//   o_i = sum_t w_it v_t,  w_it = exp(q_i k_t / sqrt(128) - m_i) / l_i  over the tokens t that row i sees.
//
// A unit is 32 stacked query rows (row x query head of one KV head) of one sequence; 16 where no unit has more. The path is
// bound by the bytes of K and V, so each is fetched once per unit and every warp streams on its own: a warp walks every
// fourth (or eighth) tile of 32 tokens of its block with a private ring of three 8 KB buffers filled by TMA (K and V in turn: a
// tile's V and the next tile's K travel while the scores are made) on its own mbarriers, so that the loop has no barrier of the
// block and no empty barriers. Two blocks of four warps or one of eight fit an SM, some 128 KB under way. Scores and products
// are mma.sync (16 rows are all that a decode step has; a tcgen05 tile would be 128), weights are rounded to BF16 for the
// second product only and their sum is of the rounded ones, so that the weights used add up to one exactly (where weights
// are reported, in FP32, the sum is of the unrounded ones).
// The blocks of a unit form a cluster (up to 16): they join (sums, maximum, sum) through distributed shared memory, each
// finishing a part of the rows, so that there is no scratch, no second launch and a fixed order of every addition. What a block
// says of itself it writes to all blocks ahead of the cluster's barrier: read from one another behind it, block by block, that
// took 2.7 us of a single token's 10.
// 64 caches of 256 to 8192 tokens, window 4096, 32 / 8 heads: 129 to 134 us on different B200s = 6.2 to 6.4 TB/s, 94 to 98 % of the
// measured copy rate. One token over 1028 tokens
// of one cache: 7.6 us, a chain of launch, length, first copies, tile, join; over 30000 tokens 25 us = 4.9 TB/s. With weights
// reported, 64 caches of 2304: 100 to 103 us (84.5 without).
//
// Only tokens that some row of the unit sees are read: tiles start at the window's first token, sinks are a stretch of their
// own. What a box brings beyond a stretch (other tokens, rows never written) is masked in the scores and cleared in V.
//
// Every wait is bounded. A warp whose wait runs out waits (bounded) for its copies in flight and joins with NaN: its unit's rows come
// out as NaN and add nothing to reported weights, and the host can ask how often that happened.
#include "step_attention.cuh"

#include "cluster.cuh"
#include "per_device.hpp"
#include "span_choice.hpp"
#include "step_choice.hpp"

#include <algorithm>
#include <stdexcept>

namespace ei {
namespace {

constexpr int kDim = 128;
constexpr int kBuffer = kStepTile * kDim * 2;
constexpr int kBuffers = 3;

template <int kWarps>
struct StepShared {
  uint64_t full[kWarps][kBuffers];
  float maxima[kWarps][kStepRows], sums[kWarps][kStepRows];
  float2 blocks[kStepMaxSplits][kStepRows];  // maximum and sum of every block of the cluster; each block leaves its own everywhere
  long long out[kStepRows];                  // where a row's output goes
  uint32_t slot[kStepRows];                  // its place among the partial results
  int others[kStepRows];                     // results to be joined; -1: no row of the sequence
  float top[kStepRows], inverse[kStepRows];
};
constexpr size_t step_shared(int warps, int row_tiles) {
  return size_t(warps) * kBuffers * kBuffer + (row_tiles > 1 ? size_t(kStepRows) * kDim * 2 : 0) +
         (warps == 8 ? sizeof(StepShared<8>) : sizeof(StepShared<4>)) + 1024;
}
static_assert(2 * (step_shared(4, 2) + 1024) <= 228 * 1024 && step_shared(8, 2) <= 227 * 1024, "two small blocks or a large one fit an SM");
// When the ring is done with, a warp's part of it holds its sums in front, and behind the second warp's lies what joined results
// say of themselves.
static_assert(kStepRows * kDim * 4 + kSpanMostPartials * kStepRows * 8 <= kBuffers * kBuffer, "sums and joined results fit");

__device__ __forceinline__ int tile_offset(int token, int chunk) {
  return (chunk >> 3) * (kStepTile * 128) + token * 128 + (((chunk & 7) ^ (token & 7)) << 4);
}
__device__ __forceinline__ int query_offset(int row, int chunk) {
  return (chunk >> 3) * (kStepRows * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}
__device__ uint32_t expired_waits;  // warps that have given up since the library was loaded

// The larger of two, not a number if either is none.
__device__ __forceinline__ float fmaxf_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
template <int kWarps, int kRowTiles, bool kWeights>
__global__ void __launch_bounds__(kWarps * 32, kWarps == 8 ? 1 : 2) step_attention_kernel(const __grid_constant__ StepAttentionParams p) {
  constexpr int kThreads = kWarps * 32;
  extern __shared__ unsigned char step_smem_raw[];
  unsigned char* const smem = step_smem_raw + ((1024u - (smem_address(step_smem_raw) & 1023u)) & 1023u);
  unsigned char* const queries = smem + kWarps * kBuffers * kBuffer;
  using Shared = StepShared<kWarps>;
  Shared* const sh = reinterpret_cast<Shared*>(queries + (kRowTiles > 1 ? kStepRows * kDim * 2 : 0));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const uint32_t rank = cluster_rank(), splits = cluster_size();
  cluster_started();
  if (threadIdx.x == 32) prefetch_map(&p.k_map), prefetch_map(&p.v_map);
  const int kv_head = blockIdx.x / splits, sequence = blockIdx.y;
  const int group = p.heads / p.kv_heads, stacked = p.rows * group;
  const int first_stacked = (p.first_group + int(blockIdx.z)) * kStepRows;
  const int have = min(kStepRows, stacked - first_stacked);  // rows of this unit

  // Row i of the unit: stacked row first_stacked + i = query row * group + head of the group.
  const long long row0 = (long long)sequence * p.rows;
  auto row_of = [&](int i) { return (first_stacked + i) / group; };
  auto joined_of = [&](int i) { return p.joined_counts[row0 * group + first_stacked + i < p.joined_border ? 0 : 1]; };
  auto query_at = [&](int i) {
    const int r = row_of(i), h = first_stacked + i - r * group;
    return p.q + (row0 + r) * p.q_stride + size_t(kv_head * group + h) * kDim;
  };
  uint32_t qa[kRowTiles == 1 ? 8 : 1][4];
  if (kRowTiles == 1) {
    const bf16* lo = query_at(g < have ? g : 0);
    const bf16* hi = query_at(g + 8 < have ? g + 8 : 0);
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      qa[kRowTiles == 1 ? kk : 0][0] = g < have ? *reinterpret_cast<const uint32_t*>(lo + kk * 16 + 2 * c) : 0u;
      qa[kRowTiles == 1 ? kk : 0][1] = g + 8 < have ? *reinterpret_cast<const uint32_t*>(hi + kk * 16 + 2 * c) : 0u;
      qa[kRowTiles == 1 ? kk : 0][2] = g < have ? *reinterpret_cast<const uint32_t*>(lo + kk * 16 + 8 + 2 * c) : 0u;
      qa[kRowTiles == 1 ? kk : 0][3] = g + 8 < have ? *reinterpret_cast<const uint32_t*>(hi + kk * 16 + 8 + 2 * c) : 0u;
    }
  }

  int length = p.lengths ? p.lengths[sequence] : p.length;
  if (length < 0 || length > p.capacity) length = 0;
  // Position of the unit's first and last row; a negative one is no row of the sequence.
  const int base = length - p.rows;
  const int first_position = p.together ? length - 1 : base + first_stacked / group;
  const int last_position = p.together ? length - 1 : base + (first_stacked + have - 1) / group;
  const int end = kWeights ? length : last_position + 1;
  const int low = max(0, min(first_position - p.window + 1, end));
  const int sink_end = min(p.sinks, low);
  const int sink_tiles = (sink_end + kStepTile - 1) / kStepTile;
  const int tiles = sink_tiles + (max(0, end - low) + kStepTile - 1) / kStepTile;
  const int first_tile = int((long long)tiles * rank / splits), last_tile = int((long long)tiles * (rank + 1) / splits);

  const uint32_t wait_limit = p.wait_limit ? p.wait_limit : kTmaWaitLimit;
  unsigned char* const ring = smem + warp * kBuffers * kBuffer;
  uint64_t* const full = sh->full[warp];
  auto start_of = [&](int tile) { return tile < sink_tiles ? tile * kStepTile : low + (tile - sink_tiles) * kStepTile; };
  // Item 2n is K and 2n + 1 V of this warp's n-th tile; item i lies in buffer i % 3.
  auto request = [&](int item) {
    const int tile = first_tile + warp + (item >> 1) * kWarps;
    if (tile >= last_tile) return;
    uint64_t* bar = &full[item % kBuffers];
    const bool faulty = item == 0 && warp == 0 && sequence == 0 && rank == splits - 1;  // which has a tile if any block has
    mbarrier_expect_tx(bar, kBuffer + (faulty ? p.fault_tx : 0));
    tma_load_5d(ring + (item % kBuffers) * kBuffer, (item & 1) ? &p.v_map : &p.k_map, 0, start_of(tile), 0, kv_head, sequence, bar);
  };
  if (lane == 0) {
    for (int b = 0; b < kBuffers; ++b) mbarrier_init(&full[b], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int i = 0; i < kBuffers; ++i) request(i);
  }
  __syncwarp();
  if (p.partial) {  // launched in plain stream order: the wait is over at once
    grid_dependency_wait();
    grid_launch_dependents();
  }

  if (kRowTiles > 1) {
    for (int i = threadIdx.x; i < kStepRows * 16; i += kThreads) {
      const int row = i >> 4, chunk = i & 15;
      const uint4 v = row < have ? reinterpret_cast<const uint4*>(query_at(row))[chunk] : make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(queries + query_offset(row, chunk)) = v;
    }
    __syncthreads();
  }

  constexpr int kUnitRows = kRowTiles * 16;
  if (threadIdx.x < kUnitRows) {  // read behind the loop
    const int i = threadIdx.x;
    const int r = i < have ? row_of(i) : 0, h = kv_head * group + (i < have ? first_stacked + i - r * group : 0);
    const bool real = i < have && (p.together || base + r >= 0);
    sh->slot[i] = uint32_t((row0 + r) * p.heads + h);
    sh->out[i] = (row0 + r) * p.out_stride + (long long)h * kDim;
    sh->others[i] = !real ? -1 : p.joined ? joined_of(i) : 0;
  }

  // Rows' positions: what a row sees is t <= limit and (t >= floor or t < sinks).
  int limit[kRowTiles][2];
#pragma unroll
  for (int rt = 0; rt < kRowTiles; ++rt)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int i = rt * 16 + half * 8 + g;
      limit[rt][half] = i < have ? (p.together ? length - 1 : base + row_of(i)) : -1;
    }
  const float exponent_scale = rsqrtf(float(kDim)) * kLog2e;
  float* const raw =
      kWeights ? p.raw + ((size_t(sequence) * p.kv_heads + kv_head) * p.raw_rows + size_t(blockIdx.z) * kStepRows) * p.raw_stride : nullptr;

  float o[kRowTiles][16][4];
  float m[kRowTiles][2], l[kRowTiles][2];
#pragma unroll
  for (int rt = 0; rt < kRowTiles; ++rt) {
#pragma unroll
    for (int d = 0; d < 16; ++d) o[rt][d][0] = o[rt][d][1] = o[rt][d][2] = o[rt][d][3] = 0.0f;
    m[rt][0] = m[rt][1] = -INFINITY;
    l[rt][0] = l[rt][1] = 0.0f;
  }

  bool ok = true;
  int item = 0, buffer = 0;
  uint32_t parity = 0;
  for (int tile = first_tile + warp; tile < last_tile; tile += kWarps) {
    ok = __all_sync(0xffffffffu, mbarrier_wait(&full[buffer], parity, wait_limit));
    if (!ok) break;
    const unsigned char* ks = ring + buffer * kBuffer;
    const int first = start_of(tile);
    const int stop = tile < sink_tiles ? sink_end : end;  // of the tile's stretch

    float s[kRowTiles][4][4];
#pragma unroll
    for (int rt = 0; rt < kRowTiles; ++rt)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[rt][j][0] = s[rt][j][1] = s[rt][j][2] = s[rt][j][3] = 0.0f;
#pragma unroll
    for (int pair = 0; pair < 4; ++pair) {
      uint32_t a[kRowTiles][2][4];
#pragma unroll
      for (int rt = 0; rt < kRowTiles; ++rt)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          if (kRowTiles == 1) {
#pragma unroll
            for (int x = 0; x < 4; ++x) a[rt][kk][x] = qa[kRowTiles == 1 ? 2 * pair + kk : 0][x];
          } else {
            ldmatrix_x4(a[rt][kk][0], a[rt][kk][1], a[rt][kk][2], a[rt][kk][3],
                        queries + query_offset(rt * 16 + (lane & 15), 2 * (2 * pair + kk) + (lane >> 4)));
          }
        }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4(b0, b1, b2, b3, ks + tile_offset(j * 8 + (lane & 7), 4 * pair + (lane >> 3)));
#pragma unroll
        for (int rt = 0; rt < kRowTiles; ++rt) {
          mma_bf16_16816(s[rt][j], a[rt][0][0], a[rt][0][1], a[rt][0][2], a[rt][0][3], b0, b1);
          mma_bf16_16816(s[rt][j], a[rt][1][0], a[rt][1][1], a[rt][1][2], a[rt][1][3], b2, b3);
        }
      }
    }
    __syncwarp();
    if (lane == 0) request(item + kBuffers);  // K has been read: its buffer takes the next tile's V
    __syncwarp();

    if (first + kStepTile > min(first_position + 1, stop) || (tile >= sink_tiles && first <= last_position - p.window)) {
#pragma unroll
      for (int rt = 0; rt < kRowTiles; ++rt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int t = first + j * 8 + 2 * c + (x & 1), at = limit[rt][x >> 1];
            if (t >= stop || t > at || (t <= at - p.window && t >= p.sinks)) s[rt][j][x] = -INFINITY;
          }
    }
    // Scores as powers of two, rounded once here: relative to a maximum that is one of them, the largest weight is 1 whatever its
    // size, and the weights that are reported and their sum are made of the same numbers.
#pragma unroll
    for (int rt = 0; rt < kRowTiles; ++rt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[rt][j][x] *= exponent_scale;
    if (kWeights) {
      // For the weights when the row's maximum and sum are known.
#pragma unroll
      for (int rt = 0; rt < kRowTiles; ++rt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int i = rt * 16 + half * 8 + g;
          if (i < have) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<float2*>(raw + size_t(i) * p.raw_stride + size_t(tile) * kStepTile + j * 8 + 2 * c) =
                  make_float2(s[rt][j][2 * half], s[rt][j][2 * half + 1]);
          }
        }
    }

    uint32_t pa[kRowTiles][4][2];
#pragma unroll
    for (int rt = 0; rt < kRowTiles; ++rt) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float top = m[rt][half];
#pragma unroll
        for (int j = 0; j < 4; ++j) top = fmaxf(top, fmaxf(s[rt][j][2 * half], s[rt][j][2 * half + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // A row with nothing visible yet keeps -inf; 0 as the exponent's base then makes every weight 0.
        const float reference = top == -INFINITY ? 0.0f : top;
        if (__any_sync(0xffffffffu, top != m[rt][half])) {
          const float rescale = power_of_two(m[rt][half] - reference);  // exactly 1 where it stayed
          l[rt][half] *= rescale;
#pragma unroll
          for (int d = 0; d < 16; ++d) {
            o[rt][d][2 * half] *= rescale;
            o[rt][d][2 * half + 1] *= rescale;
          }
          m[rt][half] = top;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float w0 = power_of_two(s[rt][j][2 * half] - reference);
          const float w1 = power_of_two(s[rt][j][2 * half + 1] - reference);
          const uint32_t both = pack_bf16(w0, w1);
          l[rt][half] += kWeights ? w0 + w1 : bf16_lo(both) + bf16_hi(both);
          pa[rt][j][half] = both;
        }
      }
    }

    ++item;
    if (++buffer == kBuffers) buffer = 0, parity ^= 1;
    ok = __all_sync(0xffffffffu, mbarrier_wait(&full[buffer], parity, wait_limit));
    if (!ok) break;
    unsigned char* vs = ring + buffer * kBuffer;
    if (stop - first < kStepTile) {
      // Nothing beyond the stretch may pass through a zero weight.
      const int live = stop - first;
      for (int i = lane; i < (kStepTile - live) * 16; i += 32)
        *reinterpret_cast<uint4*>(vs + tile_offset(live + (i >> 4), i & 15)) = make_uint4(0, 0, 0, 0);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the buffer is a copy's again after this tile
      __syncwarp();
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int d = 0; d < 16; d += 2) {
        const int matrix = lane >> 3;
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4_trans(b0, b1, b2, b3, vs + tile_offset(t * 16 + (matrix & 1) * 8 + (lane & 7), d + (matrix >> 1)));
#pragma unroll
        for (int rt = 0; rt < kRowTiles; ++rt) {
          mma_bf16_16816(o[rt][d], pa[rt][2 * t][0], pa[rt][2 * t][1], pa[rt][2 * t + 1][0], pa[rt][2 * t + 1][1], b0, b1);
          mma_bf16_16816(o[rt][d + 1], pa[rt][2 * t][0], pa[rt][2 * t][1], pa[rt][2 * t + 1][0], pa[rt][2 * t + 1][1], b2, b3);
        }
      }
    }
    __syncwarp();
    if (lane == 0) request(item + kBuffers);
    __syncwarp();
    ++item;
    if (++buffer == kBuffers) buffer = 0, parity ^= 1;
  }
  if (!ok) {
    // A copy did not arrive within the bound. Those requested are waited for (bounded) before their buffers are used for
    // anything else, and the unit's rows come out as NaN. A maximum that is no number, which no scores make, says so to the
    // other warps and blocks.
    if (lane == 0) {
      atomicAdd(&expired_waits, 1u);
      for (int i = item; i < item + kBuffers; ++i) {
        if (first_tile + warp + (i >> 1) * kWarps < last_tile) mbarrier_wait(&full[i % kBuffers], (i / kBuffers) & 1, wait_limit);
      }
    }
    __syncwarp();
#pragma unroll
    for (int rt = 0; rt < kRowTiles; ++rt) l[rt][0] = l[rt][1] = m[rt][0] = m[rt][1] = __int_as_float(0x7fffffff);
  }
  grid_dependency_wait();  // what is joined below may be the preceding kernel's

  // The warps' results: maxima first, then each warp's sums relative to the block's maximum.
#pragma unroll
  for (int rt = 0; rt < kRowTiles; ++rt)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      l[rt][half] += __shfl_xor_sync(0xffffffffu, l[rt][half], 1);
      l[rt][half] += __shfl_xor_sync(0xffffffffu, l[rt][half], 2);
      if (c == 0) {
        sh->maxima[warp][rt * 16 + half * 8 + g] = m[rt][half];
        sh->sums[warp][rt * 16 + half * 8 + g] = l[rt][half];
      }
    }
  __syncthreads();
  const size_t slots = size_t(p.sequences) * p.rows * p.heads;
  // Results to be joined say their maximum and sum: requested by all threads at once.
  float2(*const others)[kStepRows] =
      reinterpret_cast<float2(*)[kStepRows]>(smem + 2 * kBuffers * kBuffer - kSpanMostPartials * kStepRows * sizeof(float2));
  if (p.joined) {
    for (int e = threadIdx.x; e < kSpanMostPartials * kUnitRows; e += kThreads) {
      const int j = e / kUnitRows, i = e % kUnitRows;
      if (j < sh->others[i]) others[j][i] = *reinterpret_cast<const float2*>(p.joined + (j * slots + sh->slot[i]) * kStepPartial + kDim);
    }
  }
  cluster_wait_started();
  // The block's maximum and sum of a row go to every block of the cluster, so that joining starts with values at hand.
  for (int e = threadIdx.x; e < kUnitRows * int(splits); e += kThreads) {
    const int i = e % kUnitRows;
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf_nan(top, sh->maxima[w][i]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float part = sh->sums[w][i];
      if (part != 0.0f) sum += part * power_of_two(sh->maxima[w][i] - top);  // a warp without a visible token has none
    }
    remote_store(&sh->blocks[rank][i], e / kUnitRows, make_float2(top, sum));
  }
  float* const area = reinterpret_cast<float*>(ring);  // [rows][128]
#pragma unroll
  for (int rt = 0; rt < kRowTiles; ++rt)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int i = rt * 16 + half * 8 + g;
      float top = sh->maxima[0][i];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sh->maxima[w][i]);
      const float factor = m[rt][half] == -INFINITY ? 0.0f : power_of_two(m[rt][half] - top);
#pragma unroll
      for (int d = 0; d < 16; ++d)
        *reinterpret_cast<float2*>(area + i * kDim + ((d * 8 + 2 * c) ^ ((i & 3) << 3))) =
            make_float2(o[rt][d][2 * half] * factor, o[rt][d][2 * half + 1] * factor);
    }
  __syncthreads();
  float* const block_area = reinterpret_cast<float*>(smem);
  for (int i = threadIdx.x; i < min(kUnitRows, have) * (kDim / 4); i += kThreads) {
    float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float4 v = reinterpret_cast<const float4*>(smem + w * kBuffers * kBuffer)[i];
      total.x += v.x, total.y += v.y, total.z += v.z, total.w += v.w;
    }
    reinterpret_cast<float4*>(block_area)[i] = total;
  }
  if (splits > 1) cluster_sync();
  else __syncthreads();

  // Joined over the cluster and with what other kernels left: the common maximum, every part's factor and share of the sum
  // (in place of its maximum and sum), the sum.
  if (threadIdx.x < kUnitRows) {
    const int i = threadIdx.x, count = sh->others[i];
    float top = -INFINITY;
    for (uint32_t r = 0; r < splits; ++r) top = fmaxf_nan(top, sh->blocks[r][i].x);
#pragma unroll 4
    for (int j = 0; j < count; ++j) top = fmaxf_nan(top, others[j][i].x);
    sh->top[i] = top;
  }
  __syncthreads();
  {
    auto weigh = [&](float2& part, float top) {
      const float factor = part.y == 0.0f ? 0.0f : power_of_two(part.x - top);  // nothing visible there counts nothing
      part = make_float2(factor, part.y == 0.0f ? 0.0f : part.y * factor);
    };
    for (int e = threadIdx.x; e < kUnitRows * int(splits); e += kThreads) weigh(sh->blocks[e / kUnitRows][e % kUnitRows], sh->top[e % kUnitRows]);
    if (p.joined)
      for (int e = threadIdx.x; e < kSpanMostPartials * kUnitRows; e += kThreads) {
        const int j = e / kUnitRows, i = e % kUnitRows;
        if (j < sh->others[i]) weigh(others[j][i], sh->top[i]);
      }
  }
  __syncthreads();
  if (threadIdx.x < kUnitRows) {
    const int i = threadIdx.x, count = sh->others[i];
    float sum = 0.0f;
    for (uint32_t r = 0; r < splits; ++r) sum += sh->blocks[r][i].y;
#pragma unroll 4
    for (int j = 0; j < count; ++j) sum += others[j][i].y;
    const float inverse = count < 0 || sum == 0.0f ? 0.0f : p.partial ? sum : 1.0f / sum;
    sh->inverse[i] = inverse;
    if (kWeights && p.row_stats && rank == 0 && i < have)
      p.row_stats[(size_t(sequence) * p.kv_heads + kv_head) * p.raw_rows + size_t(blockIdx.z) * kStepRows + i] =
          make_float2(sh->top[i], sh->top[i] != sh->top[i] ? 0.0f : inverse);
  }
  __syncthreads();
  {
    const int quads = have * (kDim / 4);
    const int from = int((long long)quads * rank / splits), to = int((long long)quads * (rank + 1) / splits);
    for (int e = from + int(threadIdx.x); e < to; e += kThreads) {
      const int i = e / (kDim / 4), quad = e % (kDim / 4);
      const float* own = block_area + i * kDim + ((quad * 4) ^ ((i & 3) << 3));
      float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      auto add = [&](float4 v, float factor) {
        if (factor == 0.0f) return;  // nothing visible there: not even a product that is no number counts
        total.x = fmaf(v.x, factor, total.x), total.y = fmaf(v.y, factor, total.y);
        total.z = fmaf(v.z, factor, total.z), total.w = fmaf(v.w, factor, total.w);
      };
#pragma unroll 1
      for (uint32_t r0 = 0; r0 < splits; r0 += 8) {
        float4 v[8];
#pragma unroll
        for (uint32_t u = 0; u < 8; ++u)
          if (r0 + u < splits) v[u] = remote_float4(own, r0 + u);
#pragma unroll
        for (uint32_t u = 0; u < 8; ++u)
          if (r0 + u < splits) add(v[u], sh->blocks[r0 + u][i].x);
      }
      const size_t slot = sh->slot[i];
      const int count = p.joined ? sh->others[i] : 0;
#pragma unroll 1
      for (int j0 = 0; j0 < count; j0 += 16) {
        float4 v[16];
#pragma unroll
        for (int u = 0; u < 16; ++u)
          if (j0 + u < count) v[u] = *reinterpret_cast<const float4*>(p.joined + ((j0 + u) * slots + slot) * kStepPartial + quad * 4);
#pragma unroll
        for (int u = 0; u < 16; ++u)
          if (j0 + u < count) add(v[u], others[j0 + u][i].x);
      }
      const float inverse = sh->inverse[i];
      if (p.partial) {
        float* to_slot = p.partial + slot * kStepPartial;
        *reinterpret_cast<float4*>(to_slot + quad * 4) = total;
        if (quad == 0) *reinterpret_cast<float2*>(to_slot + kDim) = make_float2(sh->top[i], inverse);
      } else {
        uint2 packed = make_uint2(0u, 0u);
        if (inverse != 0.0f) {  // also a NaN
          packed.x = pack_bf16(total.x * inverse, total.y * inverse);
          packed.y = pack_bf16(total.z * inverse, total.w * inverse);
        }
        *reinterpret_cast<uint2*>(p.out + sh->out[i] + quad * 4) = packed;
      }
    }
  }
  if (kWeights && !p.row_stats) {
    // This block's tokens: the sum over the rows, in their order. A thread has kQuads times four neighbours, of four rows, under way:
    // behind a saturated memory a trip to the L2 takes 2 us.
    constexpr int kQuads = 4;
    const float* scores = p.scores ? p.scores + sequence * p.scores_sequence + kv_head * p.scores_head : nullptr;
    float* scores_out = p.scores_out + sequence * p.out_sequence + kv_head * p.out_head;
    const bool whole = ((reinterpret_cast<uintptr_t>(scores) | reinterpret_cast<uintptr_t>(scores_out)) & 15) == 0;
    const int stop = min(last_tile * kStepTile, end);
    for (int t0 = first_tile * kStepTile + 4 * int(threadIdx.x); t0 < stop; t0 += 4 * kQuads * kThreads) {
      float sum[kQuads][4] = {}, old[kQuads][4] = {};
#pragma unroll
      for (int u = 0; u < kQuads; ++u) {
        const int t = t0 + u * 4 * kThreads;
        if (!scores) continue;
        if (whole && t + 3 < stop) {
          *reinterpret_cast<float4*>(old[u]) = *reinterpret_cast<const float4*>(scores + t);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (t + x < stop) old[u][x] = scores[t + x];
        }
      }
      for (int i0 = 0; i0 < have; i0 += 4) {
        float4 score[4][kQuads];  // whole tiles of them are there
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int u = 0; u < kQuads; ++u) {
            const int t = t0 + u * 4 * kThreads;
            if (i0 + i < have && t < stop) score[i][u] = *reinterpret_cast<const float4*>(raw + size_t(i0 + i) * p.raw_stride + t);
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i0 + i >= have) break;
          const float inverse = sh->inverse[i0 + i], top = sh->top[i0 + i];
          if (inverse == 0.0f || top != top) continue;  // a row that gave up adds nothing
#pragma unroll
          for (int u = 0; u < kQuads; ++u) {
            sum[u][0] = fmaf(power_of_two(score[i][u].x - top), inverse, sum[u][0]);
            sum[u][1] = fmaf(power_of_two(score[i][u].y - top), inverse, sum[u][1]);
            sum[u][2] = fmaf(power_of_two(score[i][u].z - top), inverse, sum[u][2]);
            sum[u][3] = fmaf(power_of_two(score[i][u].w - top), inverse, sum[u][3]);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kQuads; ++u) {
        const int t = t0 + u * 4 * kThreads;
        if (whole && t + 3 < stop) {
          *reinterpret_cast<float4*>(scores_out + t) =
              make_float4(old[u][0] + sum[u][0], old[u][1] + sum[u][1], old[u][2] + sum[u][2], old[u][3] + sum[u][3]);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (t + x < stop) scores_out[t + x] = old[u][x] + sum[u][x];
        }
      }
    }
  }
  if (splits > 1) cluster_sync();  // no block leaves while another reads its shared memory
}

// Weights of more than one unit's rows: block (128 tokens, KV head, sequence), a warp takes every eighth row, the warps' sums are
// added in their order.
constexpr int kWeightWarps = 8;
__global__ void __launch_bounds__(kWeightWarps * 32) step_weights_kernel(const __grid_constant__ StepAttentionParams p, int rows) {
  __shared__ float4 sums[kWeightWarps][32];
  const int kv_head = blockIdx.y, sequence = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  int length = p.lengths ? p.lengths[sequence] : p.length;
  if (length < 0 || length > p.capacity) length = 0;
  const int first = blockIdx.x * 128, t = first + lane * 4;
  if (first >= length) return;
  const size_t unit = (size_t(sequence) * p.kv_heads + kv_head) * p.raw_rows;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  constexpr int kAtOnce = 8;
  for (int i0 = warp; i0 < rows; i0 += kWeightWarps * kAtOnce) {
    float4 score[kAtOnce];
    float2 stats[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int i = i0 + u * kWeightWarps;
      stats[u] = make_float2(0.0f, 0.0f);
      if (i < rows && t < length) {  // whole tiles of scores are there
        stats[u] = p.row_stats[unit + i];
        score[u] = *reinterpret_cast<const float4*>(p.raw + (unit + i) * p.raw_stride + t);
      }
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (stats[u].y == 0.0f) continue;
      sum.x = fmaf(power_of_two(score[u].x - stats[u].x), stats[u].y, sum.x);
      sum.y = fmaf(power_of_two(score[u].y - stats[u].x), stats[u].y, sum.y);
      sum.z = fmaf(power_of_two(score[u].z - stats[u].x), stats[u].y, sum.z);
      sum.w = fmaf(power_of_two(score[u].w - stats[u].x), stats[u].y, sum.w);
    }
  }
  sums[warp][lane] = sum;
  __syncthreads();
  if (threadIdx.x < 128 && first + int(threadIdx.x) < length) {
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWeightWarps; ++w) total += reinterpret_cast<const float*>(sums[w])[threadIdx.x];
    const int token = first + int(threadIdx.x);
    const float old = p.scores ? p.scores[sequence * p.scores_sequence + kv_head * p.scores_head + token] : 0.0f;
    p.scores_out[sequence * p.out_sequence + kv_head * p.out_head + token] = old + total;
  }
}

template <int kWarps>
auto step_kernel(bool two, bool weights) {
  return two ? (weights ? step_attention_kernel<kWarps, 2, true> : step_attention_kernel<kWarps, 2, false>)
             : (weights ? step_attention_kernel<kWarps, 1, true> : step_attention_kernel<kWarps, 1, false>);
}
auto step_kernel(int warps, bool two, bool weights) { return warps == 8 ? step_kernel<8>(two, weights) : step_kernel<4>(two, weights); }

cudaLaunchConfig_t step_config(const StepShape& shape, bool two, unsigned heads, unsigned sequences, unsigned groups,
                               cudaLaunchAttribute* cluster) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(heads * unsigned(shape.splits), sequences, groups);
  config.blockDim = dim3(unsigned(shape.warps * 32));
  config.dynamicSmemBytes = step_shared(shape.warps, two ? 2 : 1);
  cluster->id = cudaLaunchAttributeClusterDimension;
  cluster->val.clusterDim.x = unsigned(shape.splits);
  cluster->val.clusterDim.y = cluster->val.clusterDim.z = 1;
  config.attrs = cluster;
  config.numAttrs = 1;
  return config;
}

// Sets the kernels up on the current device and says how many clusters it runs at once.
const StepCapacity& configure_step_kernels() {
  static PerDevice<StepCapacity> devices;
  int device = 0;
  EI_CUDA(cudaGetDevice(&device));
  return devices.get(device, [] {
    StepCapacity capacity;
    for (const int warps : {4, 8}) {
      for (const bool two : {false, true})
        for (const bool weights : {false, true}) {
          EI_CUDA(cudaFuncSetAttribute(step_kernel(warps, two, weights), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       int(step_shared(warps, two ? 2 : 1))));
          EI_CUDA(cudaFuncSetAttribute(step_kernel(warps, two, weights), cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        }
      for (int power = 0; power < 5; ++power) {
        cudaLaunchAttribute cluster{};
        const cudaLaunchConfig_t config = step_config({1 << power, warps}, true, 64, 1, 1, &cluster);
        EI_CUDA(cudaOccupancyMaxActiveClusters(&(warps == 4 ? capacity.four : capacity.eight)[power], step_kernel(warps, true, true), &config));
      }
    }
    return capacity;
  });
}

}  // namespace

void encode_cache_map(CUtensorMap* map, const CacheStrides& cache, size_t capacity, size_t kv_heads, size_t sequences, int box_tokens,
                      int box_halves) {
  const cuuint64_t dims[5] = {64, cuuint64_t(capacity), 2, cuuint64_t(kv_heads), cuuint64_t(sequences)};
  // An axis of extent 1 is not stepped along; its stride only has to be one that the encoder takes.
  const cuuint64_t strides[4] = {cuuint64_t(capacity > 1 ? cache.token : kDim) * 2, 128, cuuint64_t(kv_heads > 1 ? cache.head : kDim) * 2,
                                 cuuint64_t(sequences > 1 ? cache.sequence : kDim) * 2};
  const cuuint32_t box[5] = {64, cuuint32_t(box_tokens), cuuint32_t(box_halves), 1, 1};
  encode_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, cache.data, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, "K / V cache");
}

void launch_step_attention(const StepAttentionParams& p, size_t tokens, cudaStream_t stream, bool pdl) {
  const StepCapacity& capacity = configure_step_kernels();
  const int group = p.heads / p.kv_heads;
  const bool two = size_t(p.rows) * group > 16;
  const StepShape shape = step_shape(size_t(p.kv_heads) * p.sequences * p.groups, tokens, two, capacity);
  cudaLaunchAttribute attributes[2]{};
  cudaLaunchConfig_t config = step_config(shape, two, unsigned(p.kv_heads), unsigned(p.sequences), unsigned(p.groups), attributes);
  config.stream = stream;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  if (pdl) config.numAttrs = 2;
  check_cuda(cudaLaunchKernelEx(&config, step_kernel(shape.warps, two, p.raw != nullptr), p), "cudaLaunchKernelEx");
}

uint32_t step_expired_waits(cudaStream_t stream) {
  uint32_t count = 0;
  EI_CUDA(cudaMemcpyFromSymbolAsync(&count, expired_waits, sizeof(count), 0, cudaMemcpyDeviceToHost, stream));
  EI_CUDA(cudaStreamSynchronize(stream));
  return count;
}

void launch_step_weights(const StepAttentionParams& p, size_t tokens, cudaStream_t stream) {
  if (tokens == 0) return;  // no token to add to, and no launch without blocks
  const int rows = std::min(p.groups * kStepRows, p.rows * (p.heads / p.kv_heads) - p.first_group * kStepRows);
  launch(step_weights_kernel, dim3(unsigned((tokens + 127) / 128), unsigned(p.kv_heads), unsigned(p.sequences)), dim3(kWeightWarps * 32), 0, stream, true,
         p, rows);
}

}  // namespace ei
