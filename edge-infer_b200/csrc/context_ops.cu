// C-ABI entry points of the operators for long contexts: rotation with norms, attention with a window, over a shared prefix and
// with accumulated weights, eviction. Validation before any write, no allocation, launches on the context's stream.
#include "abi_checks.cuh"
#include "abi_util.cuh"
#include "attention_choice.hpp"
#include "context_kernels.cuh"
#include "span_attention.cuh"
#include "view_overlap.hpp"

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <vector>

using namespace ei;

namespace {

constexpr size_t kHeadWidth = 128;
constexpr size_t kMostTokens = size_t(1) << 30;  // of a cache: positions and windows stay clear of 2^31

// The context's device has to be the current one: launches, tensor maps and kernel attributes go there. Asked for last, so
// that a malformed call is refused as such on any machine.
void expect_current_device(const ei_context* ctx) {
  int device = -1;
  EI_CUDA(cudaGetDevice(&device));
  if (device != ctx->device) reject("the execution context belongs to another CUDA device than the current one");
}

// `out` is written while others read or write the rest.
void expect_apart(const Region& out, std::initializer_list<Region> others, const char* what) {
  for (const Region& other : others)
    if (may_meet(out, other)) reject(what);
}
Region region_of_rows(const ei_view3& v) { return region_of(v, sizeof(bf16), 2); }
Region region_of_cache(const ei_view4& v) { return region_of(v, sizeof(bf16), 1); }
Region region_of_scores(const ei_view3& v) { return region_of(v, sizeof(float), 1); }
// Values in device memory that the kernels read or write one by one; null is the caller's to look at.
void expect_integers(const int32_t* values, const char* name) {
  if (reinterpret_cast<uintptr_t>(values) & 3) reject(std::string(name) + " must be 4-byte aligned");
}
Region region_of_lengths(const int32_t* lengths, size_t sequences) { return region_of(lengths, sequences * sizeof(int32_t)); }

// [rows, heads, width]: heads of a row adjacent, rows 16-byte aligned and disjoint.
void expect_rows(const ei_view3& v, const char* name) {
  if (v.data == nullptr || elements(v) == 0) reject(std::string(name) + " have no storage or are empty");
  for (size_t extent : v.shape) kernel_extent(extent, name);
  if ((v.shape[2] > 1 && v.stride[2] != 1) || (v.shape[1] > 1 && v.stride[1] != v.shape[2]))
    reject(std::string(name) + " must keep the heads of a row packed and adjacent");
  if (v.shape[0] > 1 && (v.stride[0] < v.shape[1] * v.shape[2] || v.stride[0] % 8 || v.stride[0] > (size_t(1) << 40)))
    reject(std::string(name) + " must have disjoint rows a multiple of 16 bytes apart");
  if (!aligned16(v.data)) reject(std::string(name) + " must be 16-byte aligned");
}
long long row_stride(const ei_view3& v) { return v.shape[0] > 1 ? (long long)v.stride[0] : (long long)(v.shape[1] * v.shape[2]); }

// [sequences, capacity, kv_heads, 128] of any strides that are whole 16 bytes and step over at least a head row each. (Inputs may
// show one storage twice; outputs are looked at by may_fold as well.)
CacheStrides expect_cache(const ei_view4& v, const char* name) {
  if (v.data == nullptr || elements(v) == 0) reject(std::string(name) + " have no storage or are empty");
  if (v.shape[3] != kHeadWidth || v.stride[3] != 1) reject(std::string(name) + " must have packed heads of 128 values");
  if (v.shape[0] > 65535 || v.shape[2] > 65535) reject(std::string(name) + " have too many sequences or heads");
  if (v.shape[1] > kMostTokens) reject(std::string(name) + " have too many tokens");
  size_t stride[3];
  for (int axis = 0; axis < 3; ++axis) {
    stride[axis] = v.shape[axis] > 1 ? v.stride[axis] : kHeadWidth;
    if (stride[axis] < kHeadWidth || stride[axis] % 8 || stride[axis] >= (size_t(1) << 38))
      reject(std::string(name) + " must step over whole head rows, a multiple of 16 bytes");
  }
  if (!aligned16(v.data)) reject(std::string(name) + " must be 16-byte aligned");
  return {static_cast<const bf16*>(v.data), stride[1], stride[2], stride[0]};
}
ei_view4 as_cache(const ei_view3& v) {
  return {v.data, {1, v.shape[0], v.shape[1], v.shape[2]}, {kHeadWidth, v.stride[0], v.stride[1], v.stride[2]}};
}

// Scores [sequences, kv_heads, tokens], packed along the tokens.
void expect_scores(const ei_view3& v, size_t sequences, size_t kv_heads, size_t tokens, const char* name) {
  if (v.data == nullptr) reject(std::string(name) + " has no storage");
  if (v.shape[0] != sequences || v.shape[1] != kv_heads || v.shape[2] != tokens)
    reject(std::string(name) + " must be [sequences, kv_heads, tokens]");
  if ((tokens > 1 && v.stride[2] != 1) || (kv_heads > 1 && v.stride[1] < tokens) || (sequences > 1 && v.stride[0] < tokens))
    reject(std::string(name) + " must be packed along its tokens, rows apart");
  if ((kv_heads > 1 && v.stride[1] > (size_t(1) << 40)) || (sequences > 1 && v.stride[0] > (size_t(1) << 40)))
    reject(std::string(name) + " has rows too far apart");
  if (reinterpret_cast<uintptr_t>(v.data) & 3) reject(std::string(name) + " must be 4-byte aligned");
}

// Test hook: poll limit for the next attention that this thread calls (0: none is armed).
thread_local uint32_t injected_polls = 0;
void take_injected(StepAttentionParams* p) {
  if (!injected_polls) return;
  p->wait_limit = injected_polls;
  p->fault_tx = 16;
  injected_polls = 0;
}

// What every attention of this file checks and fills in: queries [sequences * rows, heads, 128] over caches.
StepAttentionParams attention_of(const ei_view3& q, const ei_view4& k, const ei_view4& v, const ei_view3& out, const int32_t* lengths,
                                 size_t length, CacheStrides* keys, CacheStrides* values) {
  expect_rows(q, "attention queries");
  expect_rows(out, "attention outputs");
  *keys = expect_cache(k, "attention keys");
  *values = expect_cache(v, "attention values");
  for (int axis = 0; axis < 3; ++axis)
    if (q.shape[axis] != out.shape[axis]) reject("attention outputs must have the queries' shape");
  for (int axis = 0; axis < 4; ++axis)
    if (k.shape[axis] != v.shape[axis]) reject("attention keys and values must have one shape");
  if (q.shape[2] != kHeadWidth) reject("attention heads must be 128 wide");
  if (q.shape[1] % k.shape[2]) reject("query heads must be a whole multiple of KV heads");
  if (q.shape[0] % k.shape[0]) reject("query rows must be the same number for every sequence");
  const size_t rows = q.shape[0] / k.shape[0], group = q.shape[1] / k.shape[2];
  if (rows > kMostTokens / group || (rows * group + kStepRows - 1) / kStepRows > 65535) reject("too many query rows");
  if (q.shape[0] > (size_t(1) << 31) / q.shape[1]) reject("too many query rows");
  if (!lengths && length > k.shape[1]) reject("the length exceeds the caches' capacity");
  expect_integers(lengths, "lengths");
  // A row's queries are read by the blocks that write it and, as part of their boxes, by others that do not use them.
  if (q.data != out.data || row_stride(q) != row_stride(out))
    expect_apart(region_of_rows(out), {region_of_rows(q)}, "attention outputs must be the queries' own view or lie apart from them");
  expect_apart(region_of_rows(out), {region_of_cache(k), region_of_cache(v), region_of_lengths(lengths, k.shape[0])},
               "attention outputs must lie apart from keys, values and lengths");
  StepAttentionParams p{};
  p.q = static_cast<const bf16*>(q.data);
  p.q_stride = row_stride(q);
  p.out = static_cast<bf16*>(out.data);
  p.out_stride = row_stride(out);
  p.rows = int(rows);
  p.heads = int(q.shape[1]);
  p.kv_heads = int(k.shape[2]);
  p.sequences = int(k.shape[0]);
  p.capacity = int(k.shape[1]);
  p.lengths = lengths;
  p.length = int(length);
  p.window = int(kMostTokens);
  p.groups = step_groups(p.rows, int(group));
  return p;
}
void encode_maps(StepAttentionParams* p, const CacheStrides& keys, const CacheStrides& values) {
  encode_cache_map(&p->k_map, keys, size_t(p->capacity), size_t(p->kv_heads), size_t(p->sequences), kStepTile, 2);
  encode_cache_map(&p->v_map, values, size_t(p->capacity), size_t(p->kv_heads), size_t(p->sequences), kStepTile, 2);
}
// The same rows and caches for the many-row kernel.
SpanAttentionParams span_of(const StepAttentionParams& p, const CacheStrides& keys, const CacheStrides& values) {
  SpanAttentionParams s{};
  s.q = p.q, s.q_stride = p.q_stride, s.out = p.out, s.out_stride = p.out_stride;
  s.rows = p.rows, s.heads = p.heads, s.kv_heads = p.kv_heads, s.sequences = p.sequences, s.capacity = p.capacity;
  s.wait_limit = p.wait_limit, s.fault_tx = p.fault_tx;
  s.lengths = p.lengths, s.length = p.length, s.window = p.window, s.sinks = p.sinks, s.together = p.together;
  encode_cache_map(&s.k_map, keys, size_t(p.capacity), size_t(p.kv_heads), size_t(p.sequences), kSpanBox, 1);
  encode_cache_map(&s.v_map, values, size_t(p.capacity), size_t(p.kv_heads), size_t(p.sequences), kSpanBox, 1);
  encode_cache_map(&s.k_tile_map, keys, size_t(p.capacity), size_t(p.kv_heads), size_t(p.sequences), kSpanTile, 2);
  encode_cache_map(&s.v_tile_map, values, size_t(p.capacity), size_t(p.kv_heads), size_t(p.sequences), kSpanTile, 2);
  return s;
}
size_t most_tokens(const StepAttentionParams& p) { return size_t(p.lengths ? p.capacity : p.length); }

size_t raw_rows(size_t rows, size_t group) { return std::min<size_t>(kStepWeightGroups * kStepRows, rows * group); }
size_t raw_stride(size_t capacity) { return (capacity + kStepTile - 1) / kStepTile * kStepTile; }

}  // namespace

extern "C" {

ei_status ei_build_rope_table_scaled(float* host_table, size_t max_positions, size_t rotary_dim, double theta,
                                     const ei_rope_scaling* scaling) {
  return guarded([&] {
    if (!host_table || !max_positions || !rotary_dim || rotary_dim % 2 || !std::isfinite(theta) || theta <= 0.0)
      reject("RoPE table requires positive extents, an even rotated width and a positive theta");
    const ei_rope_scaling none{};
    const ei_rope_scaling& s = scaling ? *scaling : none;
    if (s.kind < EI_ROPE_PLAIN || s.kind > EI_ROPE_BANDS) reject("unknown RoPE scaling");
    const bool scaled = s.kind != EI_ROPE_PLAIN, banded = s.kind == EI_ROPE_YARN || s.kind == EI_ROPE_BANDS;
    if (scaled && !(std::isfinite(s.factor) && s.factor > 0.0)) reject("RoPE scaling needs a positive factor");
    if (banded && !(std::isfinite(s.original_positions) && s.original_positions > 0.0 && std::isfinite(s.fast) && std::isfinite(s.slow) &&
                    s.slow > 0.0 && s.fast > s.slow))
      reject("RoPE scaling by frequency needs the original length and fast > slow > 0");
    if (s.kind == EI_ROPE_YARN && theta == 1.0) reject("RoPE scaling by frequency needs a theta other than 1");
    if (!(std::isfinite(s.length) && s.length >= 0.0)) reject("RoPE vectors' length must not be negative");
    const double pi = 3.14159265358979323846;
    const size_t pairs = rotary_dim / 2;
    std::vector<double> frequencies(pairs);
    double low = 0.0, high = 0.0;
    if (s.kind == EI_ROPE_YARN) {
      // Pair whose angle turns so often over the original length.
      const auto pair_of = [&](double turns) {
        return double(rotary_dim) * std::log(s.original_positions / (2.0 * pi * turns)) / (2.0 * std::log(theta));
      };
      low = std::max(std::floor(pair_of(s.fast)), 0.0);
      high = std::min(std::ceil(pair_of(s.slow)), double(rotary_dim - 1));
    }
    for (size_t i = 0; i < pairs; ++i) {
      const double f = std::pow(theta, -2.0 * double(i) / double(rotary_dim));
      double divided = 0.0;  // part of the frequency that is divided by the factor
      if (s.kind == EI_ROPE_LINEAR) divided = 1.0;
      if (s.kind == EI_ROPE_YARN) divided = std::min(std::max((double(i) - low) / std::max(high - low, 0.001), 0.0), 1.0);
      if (s.kind == EI_ROPE_BANDS) divided = std::min(std::max((s.fast - s.original_positions * f / (2.0 * pi)) / (s.fast - s.slow), 0.0), 1.0);
      frequencies[i] = scaled ? f / s.factor * divided + f * (1.0 - divided) : f;
    }
    double length = s.length;
    if (length == 0.0) length = s.kind == EI_ROPE_YARN && s.factor > 1.0 ? 0.1 * std::log(s.factor) + 1.0 : 1.0;
    for (size_t pos = 0; pos < max_positions; ++pos)
      for (size_t i = 0; i < pairs; ++i) {
        const double angle = double(pos) * frequencies[i];
        host_table[pos * rotary_dim + 2 * i] = float(length * std::sin(angle));
        host_table[pos * rotary_dim + 2 * i + 1] = float(length * std::cos(angle));
      }
  });
}

ei_status ei_qk_norm_rope_bf16(const ei_context* ctx, ei_view3 q, ei_view3 k, ei_view2 table, const int32_t* positions, size_t offset,
                               ei_view1 q_weight, ei_view1 k_weight, float epsilon, int32_t interleaved, ei_view3 q_out,
                               ei_view3 k_out) {
  return guarded([&] {
    cudaStream_t stream = stream_of(ctx);
    expect_rows(q, "queries");
    expect_rows(k, "keys");
    expect_rows(q_out, "rotated queries");
    expect_rows(k_out, "rotated keys");
    for (int axis = 0; axis < 3; ++axis)
      if (q.shape[axis] != q_out.shape[axis] || k.shape[axis] != k_out.shape[axis]) reject("rotated queries and keys must have the inputs' shapes");
    const size_t rows = q.shape[0], width = q.shape[2];
    if (k.shape[0] != rows || k.shape[2] != width) reject("queries and keys must share rows and head width");
    if (width % 16 || width > 512) reject("the head width must be a multiple of 16 up to 512");
    expect_packed(table, "RoPE table");
    const size_t rotary = table.shape[1];
    if (rotary % 16 || rotary > width) reject("the rotated width must be a multiple of 16 within the head");
    if (!aligned16(table.data)) reject("the RoPE table must be 16-byte aligned");
    const int table_rows = kernel_extent(table.shape[0], "RoPE positions");
    expect_integers(positions, "positions");
    if (!positions && (offset > table.shape[0] || rows > table.shape[0] - offset))
      throw std::out_of_range("RoPE positions exceed the table");
    for (const ei_view1* weight : {&q_weight, &k_weight}) {
      if (weight->data == nullptr) continue;
      if (weight->shape[0] != width || weight->stride[0] != 1 || !aligned16(weight->data))
        reject("a norm weight must have one packed, 16-byte aligned value per value of a head");
    }
    // In place, or apart: a thread reads its own values before it writes them, others' at any time.
    const char* apart = "rotated heads must replace their inputs or lie apart from them and from all else";
    for (const ei_view3* to : {&q_out, &k_out}) {
      const ei_view3 &from = to == &q_out ? q : k, &other = to == &q_out ? k : q;
      const Region out = region_of_rows(*to);
      if (from.data != to->data || row_stride(from) != row_stride(*to)) expect_apart(out, {region_of_rows(from)}, apart);
      expect_apart(out,
                   {region_of_rows(other), region_of(table.data, table.shape[0] * rotary * sizeof(float)), region_of(positions, rows * sizeof(int32_t)),
                    region_of(q_weight.data, width * sizeof(bf16)), region_of(k_weight.data, width * sizeof(bf16))},
                   apart);
    }
    expect_apart(region_of_rows(q_out), {region_of_rows(k_out)}, apart);
    if ((q_weight.data || k_weight.data) && !(std::isfinite(epsilon) && epsilon >= 0.0f)) reject("the norm's epsilon must not be negative");
    if (q.shape[1] + k.shape[1] > size_t(1) << 20) reject("too many heads");
    expect_current_device(ctx);
    QkRopeParams p{};
    p.q = static_cast<const bf16*>(q.data);
    p.k = static_cast<const bf16*>(k.data);
    p.q_weight = static_cast<const bf16*>(q_weight.data);
    p.k_weight = static_cast<const bf16*>(k_weight.data);
    p.q_out = static_cast<bf16*>(q_out.data);
    p.k_out = static_cast<bf16*>(k_out.data);
    p.q_row = row_stride(q), p.k_row = row_stride(k), p.q_out_row = row_stride(q_out), p.k_out_row = row_stride(k_out);
    p.rows = int(rows), p.heads = int(q.shape[1]), p.kv_heads = int(k.shape[1]), p.width = int(width), p.rotary = int(rotary);
    p.table = static_cast<const float*>(table.data);
    p.table_rows = table_rows;
    p.positions = positions;
    p.offset = positions ? 0 : int(offset);
    p.epsilon = epsilon;
    p.inverse_width = 1.0f / float(width);
    p.interleaved = interleaved != 0;
    launch_qk_norm_rope(p, stream);
  });
}

ei_status ei_attention_window_bf16(const ei_context* ctx, ei_view3 q, ei_view4 k, ei_view4 v, ei_view3 out, const int32_t* lengths,
                                   size_t length, size_t window, size_t sinks) {
  return guarded([&] {
    cudaStream_t stream = stream_of(ctx);
    CacheStrides keys, values;
    StepAttentionParams p = attention_of(q, k, v, out, lengths, length, &keys, &values);
    if (window < 1) reject("the window must hold at least the row's own token");
    p.window = int(std::min(window, kMostTokens));
    p.sinks = int(std::min(sinks, kMostTokens));
    expect_current_device(ctx);
    take_injected(&p);
    const size_t group = size_t(p.heads / p.kv_heads), tokens = most_tokens(p);
    SpanWindow choice;
    if (window_on_tensor_cores(size_t(p.sequences), size_t(p.kv_heads), size_t(p.rows), group, tokens, size_t(p.window), size_t(p.sinks), &choice)) {
      SpanAttentionParams span = span_of(p, keys, values);
      span.cluster = choice.cluster;
      launch_span_attention(span, stream);
      return;
    }
    encode_maps(&p, keys, values);
    launch_step_attention(p, window_tokens(tokens, size_t(p.window), size_t(p.sinks), kStepRows), stream, false);
  });
}

ei_status ei_context_expired_waits(const ei_context* ctx, uint64_t* count) {
  return guarded([&] {
    cudaStream_t stream = stream_of(ctx);
    if (!count) reject("the count of expired waits needs a place");
    expect_current_device(ctx);
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    EI_CUDA(cudaStreamIsCapturing(stream, &capturing));
    if (capturing != cudaStreamCaptureStatusNone) reject("expired waits are counted when the stream gets there, which a captured one does not");
    *count = uint64_t(step_expired_waits(stream)) + span_expired_waits(stream);
  });
}

ei_status ei_context_inject_wait_timeout(uint32_t polls) {
  return guarded([&] { injected_polls = polls; });
}

size_t ei_attention_shared_prefix_scratch_bytes(size_t q_rows, size_t query_heads, size_t kv_heads, size_t prefix_length) {
  if (!prefix_length || !kv_heads) return 0;
  SpanSplits splits;
  const size_t partials = prefix_on_tensor_cores(q_rows * (query_heads / kv_heads), prefix_length, kv_heads, &splits) ? size_t(splits.partials()) : 1;
  return partials * q_rows * query_heads * kStepPartial * sizeof(float);
}

ei_status ei_attention_shared_prefix_bf16(const ei_context* ctx, ei_view3 q, ei_view3 prefix_k, ei_view3 prefix_v, ei_view4 k, ei_view4 v,
                                          ei_view3 out, const int32_t* lengths, size_t length, void* scratch, size_t scratch_bytes) {
  return guarded([&] {
    cudaStream_t stream = stream_of(ctx);
    CacheStrides keys, values;
    StepAttentionParams own = attention_of(q, k, v, out, lengths, length, &keys, &values);
    const size_t prefix = prefix_k.shape[0];
    if (prefix_v.shape[0] != prefix) reject("prefix keys and values must have one shape");
    CacheStrides first_keys{}, first_values{};
    if (prefix) {
      first_keys = expect_cache(as_cache(prefix_k), "prefix keys");
      first_values = expect_cache(as_cache(prefix_v), "prefix values");
      if (prefix_k.shape[1] != k.shape[2] || prefix_v.shape[1] != k.shape[2]) reject("the prefix must have the caches' KV heads");
      if (!scratch || !aligned16(scratch) ||
          scratch_bytes < ei_attention_shared_prefix_scratch_bytes(q.shape[0], q.shape[1], k.shape[2], prefix))
        reject("shared prefix attention needs 16-byte aligned scratch of the size it names");
      if ((q.shape[0] * (q.shape[1] / k.shape[2]) + kStepRows - 1) / kStepRows > 65535) reject("too many query rows");
      const Region first_k = region_of(prefix_k, sizeof(bf16), 1), first_v = region_of(prefix_v, sizeof(bf16), 1);
      expect_apart(region_of_rows(out), {first_k, first_v}, "attention outputs must lie apart from the prefix");
      expect_apart(region_of(scratch, ei_attention_shared_prefix_scratch_bytes(q.shape[0], q.shape[1], k.shape[2], prefix)),
                   {first_k, first_v, region_of_rows(q), region_of_cache(k), region_of_cache(v), region_of_lengths(lengths, k.shape[0]),
                    region_of_rows(out)},
                   "scratch must lie apart from all else");
    }
    expect_current_device(ctx);
    encode_maps(&own, keys, values);
    take_injected(&own);
    if (prefix) {
      StepAttentionParams first = own;
      own.wait_limit = own.fault_tx = 0;  // of the call's first launch alone
      first.rows = int(q.shape[0]);
      first.sequences = 1;
      first.capacity = first.length = int(prefix);
      first.lengths = nullptr;
      first.together = true;
      first.groups = step_groups(first.rows, first.heads / first.kv_heads);
      first.partial = static_cast<float*>(scratch);
      own.joined = first.partial;
      own.joined_border = 0;
      own.joined_counts[1] = 1;
      SpanSplits splits;
      if (prefix_on_tensor_cores(q.shape[0] * (q.shape[1] / k.shape[2]), prefix, k.shape[2], &splits)) {
        SpanAttentionParams span = span_of(first, first_keys, first_values);
        span.splits = splits;
        span.partial = first.partial;
        own.joined_border = span.splits.pairs * 2 * kSpanRows;
        own.joined_counts[0] = span.splits.pair_splits;
        own.joined_counts[1] = span.splits.single_splits;
        span.cluster = span.splits.cluster;
        launch_span_attention(span, stream);
      } else {
        encode_maps(&first, first_keys, first_values);
        launch_step_attention(first, prefix, stream, false);
      }
    }
    launch_step_attention(own, most_tokens(own), stream, prefix > 0);
  });
}

size_t ei_attention_accumulate_scratch_bytes(size_t sequences, size_t rows, size_t query_heads, size_t kv_heads, size_t capacity) {
  if (!kv_heads) return 0;
  const size_t stored = sequences * kv_heads * raw_rows(rows, query_heads / kv_heads);
  return stored * (raw_stride(capacity) * sizeof(float) + sizeof(float2));
}

ei_status ei_attention_accumulate_bf16(const ei_context* ctx, ei_view3 q, ei_view4 k, ei_view4 v, ei_view3 out, const int32_t* lengths,
                                       size_t length, ei_view3 scores, ei_view3 scores_out, void* scratch, size_t scratch_bytes) {
  return guarded([&] {
    cudaStream_t stream = stream_of(ctx);
    CacheStrides keys, values;
    StepAttentionParams p = attention_of(q, k, v, out, lengths, length, &keys, &values);
    if (scores.data) expect_scores(scores, k.shape[0], k.shape[2], k.shape[1], "accumulated weights");
    expect_scores(scores_out, k.shape[0], k.shape[2], k.shape[1], "new accumulated weights");
    const bool same = scores.data == scores_out.data && scores.stride[0] == scores_out.stride[0] && scores.stride[1] == scores_out.stride[1];
    if (may_fold(region_of_scores(scores_out))) reject("new accumulated weights must have storage for every token of every head");
    const Region old_weights = region_of_scores(scores), new_weights = region_of_scores(scores_out);
    if (!same) expect_apart(new_weights, {old_weights}, "new accumulated weights must replace the old ones or lie apart from them");
    expect_apart(new_weights, {region_of_rows(q), region_of_cache(k), region_of_cache(v), region_of_lengths(lengths, k.shape[0])},
                 "new accumulated weights must lie apart from queries, keys, values and lengths");
    expect_apart(region_of_rows(out), {old_weights, new_weights}, "attention outputs must lie apart from accumulated weights");
    const size_t group = q.shape[1] / k.shape[2];
    const size_t needed = ei_attention_accumulate_scratch_bytes(k.shape[0], size_t(p.rows), q.shape[1], k.shape[2], k.shape[1]);
    if (!scratch || !aligned16(scratch) || scratch_bytes < needed)
      reject("attention with accumulated weights needs 16-byte aligned scratch of the size it names");
    expect_apart(region_of(scratch, needed),
                 {region_of_rows(q), region_of_cache(k), region_of_cache(v), region_of_lengths(lengths, k.shape[0]), region_of_rows(out),
                  old_weights, new_weights},
                 "scratch must lie apart from all else");
    expect_current_device(ctx);
    encode_maps(&p, keys, values);
    take_injected(&p);
    p.raw = static_cast<float*>(scratch);
    p.raw_rows = raw_rows(size_t(p.rows), group);
    p.raw_stride = raw_stride(k.shape[1]);
    p.scores = static_cast<const float*>(scores.data);
    p.scores_sequence = scores.stride[0], p.scores_head = scores.stride[1];
    p.scores_out = static_cast<float*>(scores_out.data);
    p.out_sequence = scores_out.stride[0], p.out_head = scores_out.stride[1];
    // Up to eight groups of 32 stacked rows at a time, each time adding to what the one before left, in a fixed order.
    const int groups = p.groups;
    if (groups > 1) p.row_stats = reinterpret_cast<float2*>(p.raw + size_t(p.sequences) * p.kv_heads * p.raw_rows * p.raw_stride);
    for (p.first_group = 0; p.first_group < groups; p.first_group += kStepWeightGroups) {
      p.groups = std::min(kStepWeightGroups, groups - p.first_group);
      launch_step_attention(p, most_tokens(p), stream, false);
      if (p.row_stats) launch_step_weights(p, most_tokens(p), stream);
      p.wait_limit = p.fault_tx = 0;
      p.scores = p.scores_out;
      p.scores_sequence = p.out_sequence, p.scores_head = p.out_head;
    }
  });
}

ei_status ei_evict_kv_bf16(const ei_context* ctx, ei_view4 k, ei_view4 v, ei_view3 scores, const int32_t* lengths, size_t length, size_t sinks,
                           size_t recent, ei_view4 k_out, ei_view4 v_out, ei_view3 scores_out, ei_view3 kept, int32_t* lengths_out) {
  return guarded([&] {
    cudaStream_t stream = stream_of(ctx);
    EvictParams p{};
    p.k = expect_cache(k, "cached keys");
    p.v = expect_cache(v, "cached values");
    const CacheStrides k_to = expect_cache(k_out, "kept keys"), v_to = expect_cache(v_out, "kept values");
    const size_t sequences = k.shape[0], kv_heads = k.shape[2], budget = k_out.shape[1];
    for (int axis = 0; axis < 4; ++axis)
      if (k.shape[axis] != v.shape[axis] || k_out.shape[axis] != v_out.shape[axis] || (axis != 1 && k_out.shape[axis] != k.shape[axis]))
        reject("cached and kept keys and values must agree in all but their tokens");
    expect_scores(scores, sequences, kv_heads, k.shape[1], "accumulated weights");
    expect_scores(scores_out, sequences, kv_heads, budget, "kept weights");
    expect_scores(kept, sequences, kv_heads, budget, "kept positions");
    if (sinks > budget || recent > budget - sinks) reject("first and latest tokens must fit the budget");
    if (!lengths && length > k.shape[1]) reject("the length exceeds the caches' capacity");
    expect_integers(lengths, "lengths");
    expect_integers(lengths_out, "new lengths");
    if (!lengths_out || lengths_out == lengths) reject("new lengths need storage of their own");
    const Region from[] = {region_of_cache(k), region_of_cache(v), region_of_scores(scores), region_of_lengths(lengths, sequences)};
    const Region to[] = {region_of_cache(k_out), region_of_cache(v_out), region_of_scores(scores_out), region_of_scores(kept),
                         region_of_lengths(lengths_out, sequences)};
    for (const Region& out : to)
      expect_apart(out, {from[0], from[1], from[2], from[3]}, "kept keys, values, weights, positions and lengths must lie apart from all inputs");
    for (int i = 0; i < 4; ++i)
      if (may_fold(to[i])) reject("kept keys, values, weights and positions must have storage for every token of every head");
    for (int i = 0; i < 5; ++i)
      for (int j = 0; j < i; ++j) expect_apart(to[i], {to[j]}, "kept keys, values, weights, positions and lengths must not share storage, but lie apart");
    p.k_out = const_cast<bf16*>(k_to.data), p.k_out_token = k_to.token, p.k_out_head = k_to.head, p.k_out_sequence = k_to.sequence;
    p.v_out = const_cast<bf16*>(v_to.data), p.v_out_token = v_to.token, p.v_out_head = v_to.head, p.v_out_sequence = v_to.sequence;
    p.scores = static_cast<const float*>(scores.data);
    p.scores_sequence = scores.stride[0], p.scores_head = scores.stride[1];
    p.scores_out = static_cast<float*>(scores_out.data);
    p.scores_out_sequence = scores_out.stride[0], p.scores_out_head = scores_out.stride[1];
    p.kept = static_cast<int32_t*>(kept.data);
    p.kept_sequence = kept.stride[0], p.kept_head = kept.stride[1];
    p.lengths = lengths;
    p.length = int(length);
    p.lengths_out = lengths_out;
    p.sequences = int(sequences), p.kv_heads = int(kv_heads), p.capacity = int(k.shape[1]), p.budget = int(budget);
    p.sinks = int(sinks), p.recent = int(recent);
    expect_current_device(ctx);
    launch_evict(p, device_multiprocessors(), stream);
  });
}

}  // extern "C"
