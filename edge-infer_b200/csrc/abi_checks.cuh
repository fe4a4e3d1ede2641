// Argument checks shared by the translation units of the direct operators.
#pragma once

#include <limits>
#include <string>

#include "common.cuh"

namespace ei {

// ---- argument checks ------------------------------------------------------------------------------------
// Every operator rejects a malformed call with std::invalid_argument (EI_INVALID_ARGUMENT across the ABI)
// before it writes anything, as the reference's operators do (operators/src/cuda/execution.cu:23-58).

[[noreturn]] inline void reject(const std::string& what) { throw std::invalid_argument(what); }

// Extents cross the ABI as size_t and index the kernels as int.
inline int kernel_extent(size_t extent, const char* name) {
  if (extent < 1 || extent > size_t(std::numeric_limits<int>::max()))
    reject(std::string(name) + " must lie between 1 and 2^31 - 1");
  return int(extent);
}

template <typename View>
constexpr int rank_of(const View& v) {
  return int(sizeof(v.shape) / sizeof(v.shape[0]));
}

template <typename View>
size_t elements(const View& v) {
  size_t product = 1;
  for (int axis = 0; axis < rank_of(v); ++axis) product *= v.shape[axis];
  return product;
}

// Packed: walking the axes from the innermost outwards, each axis steps over exactly what lies inside it.
// An axis of extent 1 is never stepped along, so its stride is not looked at.
template <typename View>
bool packed(const View& v) {
  size_t step = 1;
  for (int axis = rank_of(v) - 1; axis >= 0; --axis) {
    if (v.shape[axis] > 1 && v.stride[axis] != step) return false;
    step *= v.shape[axis];
  }
  return true;
}

// An operand the kernels index as one dense array.
template <typename View>
void expect_packed(const View& v, const char* name) {
  if (v.data == nullptr) reject(std::string(name) + " has no storage");
  if (elements(v) == 0) reject(std::string(name) + " is empty");
  if (!packed(v)) reject(std::string(name) + " must be a packed row-major view");
}

// [rows, heads, width] with every head row packed and the heads of a row adjacent; rows may be strided
// (a slice of a wider projection output, a window of a cache).
inline void expect_head_rows(const ei_view3& v, const char* name) {
  if (v.data == nullptr || elements(v) == 0) reject(std::string(name) + " has no storage or is empty");
  const bool heads_adjacent = v.stride[2] == 1 && v.stride[1] == v.shape[2];
  const bool rows_disjoint = v.stride[0] >= v.shape[1] * v.shape[2];
  if (!heads_adjacent || !rows_disjoint) reject(std::string(name) + " must keep the heads of a row packed and adjacent");
  kernel_extent(v.shape[0], "rows");
  kernel_extent(v.shape[1], "heads");
  kernel_extent(v.shape[2], "head width");
}

// A bias is optional; when present it has one packed value per output feature.
inline void expect_bias(const ei_view1& bias, size_t outputs, const char* name) {
  if (bias.data == nullptr) return;
  if (bias.shape[0] != outputs) reject(std::string(name) + " must have one value per output feature");
  if (outputs > 1 && bias.stride[0] != 1) reject(std::string(name) + " must be packed");
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline cudaStream_t stream_of(const ei_context* ctx) {
  if (!ctx) throw std::invalid_argument("execution context is null");
  return static_cast<cudaStream_t>(ctx->stream);
}

inline size_t smem_limit_of(const ei_context* ctx) {
  return ctx->shared_memory_limit ? ctx->shared_memory_limit : size_t(227) * 1024;
}

}  // namespace ei
