// Launch functions of the rotation with norms (qk_rope.cu) and of cache eviction (evict.cu).
#pragma once

#include "step_attention.cuh"

namespace ei {

struct QkRopeParams {
  const bf16 *q, *k, *q_weight, *k_weight;  // weights may be null: no norm
  bf16 *q_out, *k_out;
  long long q_row, k_row, q_out_row, k_out_row;  // elements between rows; heads are adjacent
  int rows, heads, kv_heads, width, rotary;
  const float* table;  // [positions][rotary], sine and cosine side by side
  int table_rows;
  const int32_t* positions;  // per row, or null: offset + row
  int offset;
  float epsilon, inverse_width;
  bool interleaved;
};
void launch_qk_norm_rope(const QkRopeParams& p, cudaStream_t stream);

struct EvictParams {
  CacheStrides k, v;
  bf16 *k_out, *v_out;
  size_t k_out_token, k_out_head, k_out_sequence, v_out_token, v_out_head, v_out_sequence;
  const float* scores;
  size_t scores_head, scores_sequence;
  float* scores_out;
  size_t scores_out_head, scores_out_sequence;
  int32_t* kept;
  size_t kept_head, kept_sequence;
  const int32_t* lengths;
  int length;
  int32_t* lengths_out;
  int sequences, kv_heads, capacity, budget, sinks, recent;
};
void launch_evict(const EvictParams& p, int multiprocessors, cudaStream_t stream);

}  // namespace ei
