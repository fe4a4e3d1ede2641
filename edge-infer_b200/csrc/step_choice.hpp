// How the few-row attention over caches is cut into blocks, in a plain header so that it is tested without a GPU.
#pragma once

#include <algorithm>
#include <cstddef>

namespace ei {

constexpr int kStepTile = 32;   // tokens of a tile; a warp has one at a time
constexpr int kStepMaxSplits = 16;

// A unit's tokens are shared by the blocks of one cluster: a power of two of them, at most 16. `units` = sequences x KV heads x
// groups of rows, `tokens` = most tokens a unit may read. One block of eight warps or two of four fit an SM.
struct StepShape {
  int splits, warps;
};
inline StepShape step_shape(size_t units, size_t tokens, int multiprocessors) {
  const size_t tiles = (tokens + kStepTile - 1) / kStepTile;
  // Few units: eight warps a block, as many blocks as fit at once while every warp has a tile.
  if (units <= size_t(multiprocessors)) {
    int splits = 1;
    while (splits < kStepMaxSplits && units * splits * 2 <= size_t(multiprocessors) && tiles > size_t(splits) * 8) splits *= 2;
    return {splits, 8};
  }
  return {1, 4};
}

}  // namespace ei
