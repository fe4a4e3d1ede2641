// Few-row attention over batches of key / value caches: parameters and launch (step_attention.cu).
#pragma once

#include "kernels.cuh"
#include "step_choice.hpp"

namespace ei {

constexpr int kStepPartial = 132;  // floats of a partial result: 128 sums, maximum (power of two), sum, padding

// A cache of any strides: token t, KV head j, sequence s at data + t * token + j * head + s * sequence (elements).
struct CacheStrides {
  const bf16* data;
  size_t token, head, sequence;
};
// Map of a cache for boxes of one head's tokens: (64 values, token, half of the head, KV head, sequence), so that a box lands as
// [half][token][128 B] with the 128-byte swizzle. Tokens from `capacity` on read as zero.
void encode_cache_map(CUtensorMap* map, const CacheStrides& cache, size_t capacity, size_t kv_heads, size_t sequences, int box_tokens,
                      int box_halves);

struct StepAttentionParams {
  CUtensorMap k_map, v_map;   // boxes of kStepTile tokens
  const bf16* q;              // row r, head h at q + r * q_stride + h * 128; sequence s owns rows [s * rows, (s + 1) * rows)
  long long q_stride;
  bf16* out;
  long long out_stride;
  int rows, heads, kv_heads, sequences;
  int capacity;
  const int32_t* lengths;     // tokens of each sequence (device) or null -> length
  int length;
  int window, sinks;          // a row at position p sees t <= p with t > p - window or t < sinks
  bool together;              // every row stands at the last token (a prefix that all rows see)
  int first_group, groups;    // groups of kStepRows stacked rows that this launch takes
  // Results of other stretches of tokens to be joined: [joined][sequences * rows][heads][kStepPartial]. Of all sequences' stacked
  // rows of a KV head (all_row * group + head of the group) those below joined_border have joined_counts[0], the others [1].
  const float* joined;
  int joined_border, joined_counts[2];
  float* partial;             // leave (sums, maximum, sum) here in that layout instead of normalised rows in `out`
  // Weights: scores_out[s][j][t] = scores[s][j][t] + the weights of token t, summed over this launch's rows and the group's
  // heads; every token of the sequence is written. raw: [sequences][kv_heads][raw_rows][raw_stride] FP32. Rows of one unit (one
  // group) are added up by its own blocks; of more, row_stats [sequences][kv_heads][raw_rows] receives each row's maximum and
  // inverse sum, and launch_step_weights adds up.
  const float* scores;
  float* scores_out;
  size_t scores_sequence, scores_head, out_sequence, out_head;
  float* raw;
  size_t raw_rows, raw_stride;  // the launch's stacked rows; tokens, whole tiles
  float2* row_stats;
  // Polls before a bounded wait gives up (0: the default), and bytes more than it brings that the first copy of each unit of the
  // first sequence is told to expect (0 but for tests). What gives up leaves NaN rows, a NaN maximum in partial results and the
  // accumulated weights without its rows'.
  uint32_t wait_limit, fault_tx;
};
inline int step_groups(int rows, int group) { return int((size_t(rows) * group + kStepRows - 1) / kStepRows); }
// k_map, v_map, first_group and groups are the caller's; tokens: the most a unit may read.
void launch_step_attention(const StepAttentionParams& p, size_t tokens, cudaStream_t stream, bool pdl);
constexpr int kStepWeightGroups = 8;  // that may share a launch with weights (their scores take scratch)
// Waits that have run out in this kernel on the current device, read when the stream gets there.
uint32_t step_expired_waits(cudaStream_t stream);
void launch_step_weights(const StepAttentionParams& p, size_t tokens, cudaStream_t stream);

}  // namespace ei
