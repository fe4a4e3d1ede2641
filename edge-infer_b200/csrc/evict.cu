// A cache cut to a budget: per sequence and KV head the first `sinks` tokens, the last `recent` and, of the others, those with
// the largest accumulated weight, moved in order of position into another cache.
//
// Selection is exact: the place-th largest score is found digit by digit (11, 11 and 10 bits of the order-preserving integer key,
// a histogram each of the keys that share the digits before), scores above it stay, of those equal to it the ones with the
// lowest positions. Bound: the scores once, the kept rows in and out. The selection is a chain of some microseconds however few
// tokens there are, so that the blocks which share a head's rows each repeat it (from their own copy of the keys in shared
// memory) instead of waiting for one another, and then move a part of the rows each. 64 caches of 2304 tokens and 8 heads to 2048:
// 176 us = 6.07 TB/s; one of 8191 to 1024: 13.7 us (46 with the place-th key found two bits a step by counting all keys).
#include "context_kernels.cuh"
#include "per_device.hpp"

#include <algorithm>

namespace ei {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMoves = 4;          // tokens a warp has under way
// Keys that a block holds itself (160 KB); further ones are made from the scores again. The room goes by the capacity, the lengths
// being on the device: at a capacity of 40960 one block fits an SM, and 64 caches of 2304 tokens take 246 us instead of 182.
constexpr int kCachedKeys = 40960;

constexpr int kBins = 2048;

struct EvictShared {
  int4 bins[kBins / 4];
  int totals[kWarps];
  int digit, before;
  int above[kWarps], ties[kWarps];
};

// Larger scores have larger keys; -0 is 0, and what is not a number comes last.
__device__ __forceinline__ uint32_t key_of(float score) {
  if (score != score) return 0u;
  const uint32_t bits = __float_as_uint(score + 0.0f);
  return bits ^ ((bits >> 31) ? 0xffffffffu : 0x80000000u);
}

// The digit of the place-th largest of the histogram's keys, and how many keys have a larger one; the histogram is cleared.
__device__ __forceinline__ int2 find_digit(EvictShared* sh, int place) {
  static_assert(kBins == 4 * kThreads, "a thread has four bins");
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = kThreads - 1 - int(threadIdx.x);  // the largest digits first
  const int4 bins = sh->bins[mine];
  sh->bins[mine] = make_int4(0, 0, 0, 0);
  const int own = bins.x + bins.y + bins.z + bins.w;
  int sum = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += other;
  }
  if (lane == 31) sh->totals[warp] = sum;
  __syncthreads();
  int before = sum - own;
#pragma unroll
  for (int w = 0; w < kWarps; ++w)
    if (w < warp) before += sh->totals[w];
  if (before < place && place <= before + own) {
    const int counts[4] = {bins.w, bins.z, bins.y, bins.x};
    int digit = 4 * mine + 3;
    for (int i = 0; i < 3 && before + counts[i] < place; ++i, --digit) before += counts[i];
    sh->digit = digit;
    sh->before = before;
  }
  __syncthreads();
  return make_int2(sh->digit, sh->before);
}

// Block (part of the kept rows, KV head, sequence).
__global__ void __launch_bounds__(kThreads) evict_kernel(const EvictParams p, int cached, int part_rows) {
  extern __shared__ uint32_t evict_smem[];
  EvictShared* const sh = reinterpret_cast<EvictShared*>(evict_smem);
  int* const rows = reinterpret_cast<int*>(sh + 1);                    // [part_rows] tokens of this block's part
  uint32_t* const keys = reinterpret_cast<uint32_t*>(rows + part_rows);  // [cached]
  const int kv_head = blockIdx.y, sequence = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int length = p.lengths ? p.lengths[sequence] : p.length;
  if (length < 0 || length > p.capacity) length = 0;
  const int stay = min(length, p.budget);  // tokens of the result
  const int part_first = blockIdx.x * part_rows, part_last = min(part_first + part_rows, p.budget);
  const float* scores = p.scores + sequence * p.scores_sequence + kv_head * p.scores_head;
  if (blockIdx.x == 0 && kv_head == 0 && threadIdx.x == 0) p.lengths_out[sequence] = stay;

  if (length <= p.budget) {
    for (int i = part_first + int(threadIdx.x); i < min(part_last, stay); i += kThreads) rows[i - part_first] = i;
  } else {
    // The tokens that compete: [sinks, length - recent).
    const int from = p.sinks, to = length - p.recent;
    auto key_at = [&](int t) { return t - from < cached ? keys[t - from] : key_of(scores[t]); };
    int* const bins = reinterpret_cast<int*>(sh->bins);
    const int place = p.budget - p.sinks - p.recent;  // of them stay
    uint32_t threshold = 0;                            // the place-th largest key
    sh->bins[threadIdx.x] = make_int4(0, 0, 0, 0);
    __syncthreads();
    if (place > 0) {
#pragma unroll 4
      for (int t = from + int(threadIdx.x); t < to; t += kThreads) {
        const uint32_t key = key_of(scores[t]);
        if (t - from < cached) keys[t - from] = key;
        atomicAdd(&bins[key >> 21], 1);
      }
      const int2 high = find_digit(sh, place);
#pragma unroll 4
      for (int t = from + int(threadIdx.x); t < to; t += kThreads) {
        const uint32_t key = key_at(t);
        if (key >> 21 == uint32_t(high.x)) atomicAdd(&bins[key >> 10 & 2047], 1);
      }
      const int2 middle = find_digit(sh, place - high.y);
      const uint32_t leading = uint32_t(high.x) << 11 | uint32_t(middle.x);
#pragma unroll 4
      for (int t = from + int(threadIdx.x); t < to; t += kThreads) {
        const uint32_t key = key_at(t);
        if (key >> 10 == leading) atomicAdd(&bins[key & 1023], 1);
      }
      threshold = leading << 10 | uint32_t(find_digit(sh, place - high.y - middle.y).x);
    }
    // Positions: a warp takes a stretch of tokens; how many before it stay comes from the other warps' counts.
    const int span = ((to - from + kWarps - 1) / kWarps + 31) / 32 * 32;
    const int first = min(from + warp * span, to), last = min(first + span, to);
    int above = 0, ties = 0;
    for (int t0 = first; t0 < last && place > 0; t0 += 32) {
      const int t = t0 + lane;
      const uint32_t key = t < last ? key_at(t) : 0u;
      above += __popc(__ballot_sync(0xffffffffu, t < last && key > threshold));
      ties += __popc(__ballot_sync(0xffffffffu, t < last && key == threshold));
    }
    if (lane == 0) sh->above[warp] = above, sh->ties[warp] = ties;
    __syncthreads();
    int above_before = 0, ties_before = 0, above_all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) above_before += sh->above[w], ties_before += sh->ties[w];
      above_all += sh->above[w];
    }
    const int ties_stay = place > 0 ? place - above_all : 0;
    auto put = [&](int index, int token) {
      if (index >= part_first && index < part_last) rows[index - part_first] = token;
    };
    if (place > 0) {
      for (int t0 = first; t0 < last; t0 += 32) {
        const int t = t0 + lane;
        const uint32_t key = t < last ? key_at(t) : 0u;
        const uint32_t over = __ballot_sync(0xffffffffu, t < last && key > threshold);
        const uint32_t equal = __ballot_sync(0xffffffffu, t < last && key == threshold);
        const uint32_t below = (1u << lane) - 1;
        const int tie = ties_before + __popc(equal & below);  // ties before this token
        if ((over >> lane & 1) || ((equal >> lane & 1) && tie < ties_stay))
          put(p.sinks + above_before + __popc(over & below) + min(tie, ties_stay), t);
        above_before += __popc(over);
        ties_before += __popc(equal);
      }
    }
    for (int i = threadIdx.x; i < p.sinks; i += kThreads) put(i, i);
    for (int i = threadIdx.x; i < p.recent; i += kThreads) put(p.budget - p.recent + i, length - p.recent + i);
  }
  __syncthreads();

  const int moved = max(0, min(part_last, stay) - part_first);
  for (int i = threadIdx.x; i < part_last - part_first; i += kThreads) {
    const size_t at = size_t(part_first + i);
    p.kept[sequence * p.kept_sequence + kv_head * p.kept_head + at] = i < moved ? rows[i] : -1;
    if (i < moved) p.scores_out[sequence * p.scores_out_sequence + kv_head * p.scores_out_head + at] = scores[rows[i]];
  }
  // A warp moves a token's K (lanes 0-15) and V (16-31).
  const CacheStrides& cache = lane < 16 ? p.k : p.v;
  const bf16* source = cache.data + sequence * cache.sequence + kv_head * cache.head + (lane & 15) * 8;
  bf16* target = lane < 16 ? p.k_out + sequence * p.k_out_sequence + kv_head * p.k_out_head
                           : p.v_out + sequence * p.v_out_sequence + kv_head * p.v_out_head;
  target += (lane & 15) * 8;
  const size_t step = lane < 16 ? p.k_out_token : p.v_out_token;
  for (int i0 = warp * kMoves; i0 < moved; i0 += kWarps * kMoves) {
    uint4 held[kMoves];
#pragma unroll
    for (int u = 0; u < kMoves; ++u)
      if (i0 + u < moved) held[u] = ldg_stream(source + size_t(rows[i0 + u]) * cache.token);
#pragma unroll
    for (int u = 0; u < kMoves; ++u)
      if (i0 + u < moved) *reinterpret_cast<uint4*>(target + size_t(part_first + i0 + u) * step) = held[u];
  }
}

}  // namespace

void launch_evict(const EvictParams& p, int multiprocessors, cudaStream_t stream) {
  const int units = p.sequences * p.kv_heads;
  const int cached = std::max(0, std::min(p.capacity - p.sinks - p.recent, kCachedKeys));
  // Parts of a head's rows: a block for every SM and, so that one block's selection hides behind others' copies, no more than
  // some 512 rows (64 caches of 2304 tokens and 8 heads cut to 2048, parts of 2048, 1024, 512, 256, 128 rows: 196, 182, 176, 177,
  // 214 us); 32 rows at least and 8192 at most (their list is in shared memory).
  int parts = std::max(multiprocessors / units, p.budget / 512);
  parts = std::max(1, std::min(parts, p.budget / 32));
  parts = std::max(parts, (p.budget + 8191) / 8192);
  const int part_rows = (p.budget + parts - 1) / parts;
  const size_t shared = sizeof(EvictShared) + size_t(part_rows) * 4 + size_t(cached) * 4;
  static PerDevice<bool> devices;
  int device = 0;
  EI_CUDA(cudaGetDevice(&device));
  devices.get(device, [] {
    EI_CUDA(cudaFuncSetAttribute(evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 int(sizeof(EvictShared) + (8192 + kCachedKeys) * 4)));
    return true;
  });
  launch(evict_kernel, dim3(unsigned((p.budget + part_rows - 1) / part_rows), unsigned(p.kv_heads), unsigned(p.sequences)), dim3(kThreads),
         shared, stream, false, p, cached, part_rows);
}

}  // namespace ei
