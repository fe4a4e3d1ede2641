// Many-row attention over caches on the 5th-generation tensor cores: parameters and launch (span_attention.cu).
#pragma once

#include "span_choice.hpp"
#include "step_attention.cuh"

namespace ei {

struct SpanAttentionParams {
  CUtensorMap k_map, v_map;            // boxes of kSpanBox tokens, half a head
  CUtensorMap k_tile_map, v_tile_map;  // boxes of kSpanTile tokens
  CUtensorMap q_map;                   // filled by the launch function where query tiles are boxes of the queries
  bool copied_queries;
  const bf16* q;             // as StepAttentionParams
  long long q_stride;
  bf16* out;
  long long out_stride;
  int rows, heads, kv_heads, sequences, capacity;
  const int32_t* lengths;
  int length, window, sinks;
  // Every row sees all `length` tokens of the only sequence: results are left in
  // partial[splits.partials()][rows][heads][kStepPartial], not normalised.
  bool together;
  SpanSplits splits;
  int cluster;  // blocks that share the tokens of two query tiles (of a stretch), joined through distributed shared memory
  float* partial;
  uint32_t wait_limit, fault_tx;  // as StepAttentionParams
};
void launch_span_attention(const SpanAttentionParams& p, cudaStream_t stream);
uint32_t span_expired_waits(cudaStream_t stream);  // as step_expired_waits

}  // namespace ei
