// Which of the two attention kernels over caches takes a call, in a plain header so that it is tested without a GPU.
#pragma once

#include "span_choice.hpp"
#include "step_choice.hpp"

namespace ei {

// Up to so many stacked rows (rows x query heads of a KV head) the few-row kernel is bound by the bytes alone.
constexpr size_t kFewRows = 16;

// Most tokens that `rows` neighbouring rows see, of a cache with up to `tokens`.
inline size_t window_tokens(size_t tokens, size_t window, size_t sinks, size_t rows) { return std::min(tokens, window + sinks + rows); }

// Whichever kernel is the faster by its estimate. If it is the many-row kernel, `span` says how its blocks are joined; its query
// tiles have 128 rows, two a block.
inline bool window_on_tensor_cores(size_t sequences, size_t kv_heads, size_t rows, size_t group, size_t tokens, size_t window, size_t sinks,
                                   SpanWindow* span) {
  const size_t stacked = rows * group;
  if (stacked <= kFewRows) return false;
  *span = span_window(sequences, kv_heads, stacked, window_tokens(tokens, window, sinks, (2 * kSpanRows + group - 1) / group));
  const size_t units = sequences * kv_heads * ((stacked + kStepRows - 1) / kStepRows);
  return span->microseconds < step_microseconds(units, window_tokens(tokens, window, sinks, (kStepRows + group - 1) / group));
}

// The same for a prefix that all sequences' stacked rows see, and how the many-row kernel cuts it.
inline bool prefix_on_tensor_cores(size_t stacked, size_t prefix, size_t kv_heads, SpanSplits* splits) {
  if (stacked <= kFewRows) return false;
  *splits = span_splits((stacked + kSpanRows - 1) / kSpanRows, prefix, int(kv_heads));
  return splits->microseconds < step_microseconds(kv_heads * ((stacked + kStepRows - 1) / kStepRows), prefix);
}

}  // namespace ei
