// Whether what two views touch can meet in memory, in a plain header so that it is tested without a GPU.
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>
#include <limits>

namespace ei {

// Items of `item` bytes at `at` + a sum of multiples of `step` (bytes), 0 .. count - 1 each.
struct Region {
  uintptr_t at;
  size_t item;
  int rank;
  size_t count[4], step[4];
};

// `packed` of a view's last axes are one item: the caller knows that they are adjacent.
template <typename View>
Region region_of(const View& v, size_t element, int packed) {
  constexpr int rank = int(sizeof(v.shape) / sizeof(v.shape[0]));
  Region r{reinterpret_cast<uintptr_t>(v.data), element, rank - packed, {}, {}};
  for (int axis = 0; axis < rank; ++axis) {
    if (axis >= rank - packed) r.item *= v.shape[axis];
    else r.count[axis] = v.shape[axis], r.step[axis] = v.stride[axis] * element;
  }
  return r;
}
inline Region region_of(const void* data, size_t bytes) { return {reinterpret_cast<uintptr_t>(data), bytes, 0, {}, {}}; }

// Bytes from the first to behind the last, of the axes whose step is no multiple of `period`; the largest size_t for more.
inline size_t reach_of(const Region& r, size_t period = 0) {
  unsigned __int128 bytes = r.item;
  for (int axis = 0; axis < r.rank; ++axis)
    if (r.count[axis] > 1 && (period == 0 || r.step[axis] % period)) bytes += (unsigned __int128)(r.count[axis] - 1) * r.step[axis];
  const size_t most = std::numeric_limits<size_t>::max();
  return bytes > most ? most : size_t(bytes);
}

// False only where they are known to lie apart: one behind the other, or interleaved, in different parts of a period that all
// their longer steps are multiples of (the queries and keys of one projection's rows, the keys and values of one cache).
inline bool may_meet(const Region& a, const Region& b) {
  if (!a.at || !b.at || !a.item || !b.item) return false;
  const Region& low = a.at <= b.at ? a : b;
  const Region& high = a.at <= b.at ? b : a;
  const size_t distance = high.at - low.at;
  if (reach_of(low) <= distance) return false;
  for (const Region* from : {&a, &b})
    for (int axis = 0; axis < from->rank; ++axis) {
      const size_t period = from->step[axis];
      if (from->count[axis] <= 1 || period == 0) continue;
      const size_t low_part = reach_of(low, period), high_part = reach_of(high, period), offset = distance % period;
      if (low_part <= offset && high_part <= period - offset) return false;
    }
  return true;
}

// False only where no two items meet because every axis steps over all that shorter steps reach.
inline bool may_fold(const Region& r) {
  unsigned __int128 reach = r.item;
  bool taken[4] = {};
  for (int i = 0; i < r.rank; ++i) {
    int shortest = -1;
    for (int axis = 0; axis < r.rank; ++axis)
      if (!taken[axis] && (shortest < 0 || r.step[axis] < r.step[shortest])) shortest = axis;
    taken[shortest] = true;
    // An axis of one is not stepped along: where it comes in the order does not matter.
    if (r.count[shortest] <= 1) continue;
    if (r.step[shortest] < reach) return true;
    reach += (unsigned __int128)(r.count[shortest] - 1) * r.step[shortest];
  }
  return false;
}

}  // namespace ei
