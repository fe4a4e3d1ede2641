// How the few-row attention over caches is cut into blocks, in a plain header so that it is tested without a GPU.
#pragma once

#include <algorithm>
#include <cstddef>

namespace ei {

constexpr int kStepTile = 32;   // tokens of a tile
constexpr int kStepWarps = 4;   // of a block, a tile each at a time
constexpr int kStepMaxSplits = 16;

// Blocks (one cluster) that share one unit's tokens: a power of two, at most 16. `units` = sequences x KV heads x groups of
// rows, `tokens` = most tokens a unit may read. Two blocks fit on an SM.
inline int step_splits(size_t units, size_t tokens, int multiprocessors) {
  const size_t tiles = (tokens + kStepTile - 1) / kStepTile;
  int splits = 1;
  while (splits < kStepMaxSplits && units * size_t(splits) < size_t(2 * multiprocessors) && tiles >= size_t(splits) * 2 * kStepWarps)
    splits *= 2;
  return splits;
}

}  // namespace ei
