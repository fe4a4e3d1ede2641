// How the few-row attention over caches is cut into blocks, in a plain header so that it is tested without a GPU.
#pragma once

#include <algorithm>
#include <cstddef>

namespace ei {

constexpr int kStepRows = 32;   // stacked query rows (row x query head of one KV head) of a unit
constexpr int kStepTile = 32;   // tokens of a tile; a warp has one at a time
constexpr int kStepMaxSplits = 16;

// A unit's tokens are shared by the blocks of one cluster: a power of two of them, at most 16, of four warps (two blocks fit
// an SM) or eight.
struct StepShape {
  int splits, warps;
};
// Clusters of 1, 2, 4, 8, 16 blocks that run at once. (A cluster stays within one group of SMs, and their sizes differ: of 16
// blocks of eight warps a B200 takes 7, of four warps 14; an eighth of the former started 26 us late.)
struct StepCapacity {
  int four[5], eight[5];
};

// `units` = sequences x KV heads x groups of rows, `tokens` = most tokens a unit may read: as many warps at work as there are
// while all clusters run at once and no warp is without a tile; of equal shapes the one of fewer, larger blocks, whose clusters
// are smaller (8 units of 30000 tokens, 16 blocks of four warps or 8 of eight: 28.7 and 26.7 us). With more than 16 stacked rows
// a warp's arithmetic counts, and the smaller blocks, which lie on more SMs, are ahead (16 units of 4096 tokens: 15.6 and 16.6).
inline StepShape step_shape(size_t units, size_t tokens, bool two_row_tiles, const StepCapacity& capacity) {
  const size_t tiles = (tokens + kStepTile - 1) / kStepTile;
  StepShape best{1, 4};
  for (const int warps : {4, 8})
    for (int power = 0; power < 5; ++power) {
      const int splits = 1 << power;
      const int fit = (warps == 4 ? capacity.four : capacity.eight)[power];
      if (units > size_t(fit) || size_t(splits) * warps > std::max<size_t>(tiles, 4)) continue;
      const bool better = two_row_tiles ? splits * warps > best.splits * best.warps : splits * warps >= best.splits * best.warps;
      if (better) best = {splits, warps};
    }
  return best;
}

// What the few-row kernel takes for units of more than 16 stacked rows, in microseconds: 9 for a block's start and join, in as many
// waves as there are, and 2.1 ns for 32 rows times 32 tokens with 1184 warps at work, as many as fit a B200; few units do not
// get as many.
inline float step_microseconds(size_t units, size_t tokens) {
  size_t warps = units > 14 ? 32 : 64;  // of a unit
  while (warps > 4 && warps * units > 1184) warps /= 2;
  const float busy = std::min(1.0f, float(warps * units) / 1184.0f);
  return 9.0f * std::max(1.0f, float(units) / 296.0f) + 0.0021f * float(units) * float((tokens + kStepTile - 1) / kStepTile) / busy;
}

}  // namespace ei
