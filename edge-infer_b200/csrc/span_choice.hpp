// How the many-row attention is cut into blocks, in a plain header so that it is tested without a GPU.
#pragma once

#include <algorithm>
#include <cstddef>
#include <utility>

namespace ei {

constexpr int kSpanTile = 64;    // tokens of a tile
constexpr int kSpanBox = 32;     // tokens of a box: a tile may be put together from two stretches
constexpr int kSpanRows = 128;   // stacked query rows of a query tile; a block has two, or both halves of it work on one
constexpr int kSpanMostCluster = 8;
constexpr int kSpanMostPartials = 32;

// Clusters of 1, 2, 4 and 8 such blocks that a B200 runs at once (a cluster stays within a group of SMs).
inline int span_clusters(int size) { return size == 1 ? 148 : size == 2 ? 74 : size == 4 ? 33 : 15; }

// What a block takes, in microseconds: to set itself up and to leave, per tile of tokens for two query tiles (for one, whose
// tiles the halves take in turn, two at a time), to join a cluster's results, and a partial result for who joins it. Fitted to
// blocks of 2 to 66 tiles: of 44 sizes timed with both kernels, the choice by this and the few-row kernel's estimate was the
// slower one four times, by 3, 3, 16 and 20 %.
constexpr float kSpanFixed = 10.0f, kSpanPerTile = 1.15f, kSpanJoin = 3.0f, kSpanPerPartial = 0.25f;

// A prefix that all rows see, `query_tiles` query tiles per KV head. Pairs of query tiles share the tiles of tokens they read
// and are cut into `pair_splits` stretches, an odd last one into `single_splits`; the blocks of a cluster share a stretch and
// join their results. Every stretch leaves a partial result of its rows.
struct SpanSplits {
  int cluster, pairs, pair_splits, single_splits;  // single_splits 0: no odd tile
  float microseconds;
  int clusters() const { return pairs * pair_splits + single_splits; }
  int partials() const { return std::max(pairs ? pair_splits : 0, single_splits); }  // of a row, at most
};
inline SpanSplits span_splits(size_t query_tiles, size_t tokens, int kv_heads) {
  const int tiles = int((tokens + kSpanTile - 1) / kSpanTile);
  SpanSplits best{};
  for (const int cluster : {1, 2, 4}) {
    SpanSplits s{cluster, int(query_tiles / 2), 1, int(query_tiles % 2), 0.0f};
    auto longest = [&](const SpanSplits& t) {  // tiles of a block
      const int pair = t.pairs ? (tiles + t.pair_splits * cluster - 1) / (t.pair_splits * cluster) : 0;
      const int single = t.single_splits ? (tiles + 2 * t.single_splits * cluster - 1) / (2 * t.single_splits * cluster) : 0;
      return std::make_pair(pair, single);
    };
    // More stretches, always of the kind whose blocks are longer, while the clusters fit the chip at once and blocks keep tiles.
    for (;;) {
      const auto length = longest(s);
      SpanSplits next = s;
      if (length.first >= length.second) ++next.pair_splits;
      else ++next.single_splits;
      if (std::max(length.first, length.second) < 2 || next.partials() > kSpanMostPartials ||
          (long long)next.clusters() * kv_heads > span_clusters(cluster))
        break;
      s = next;
    }
    const auto length = longest(s);
    const long long waves = ((long long)s.clusters() * kv_heads + span_clusters(cluster) - 1) / span_clusters(cluster);
    s.microseconds = float(waves) * (kSpanFixed + kSpanPerTile * float(std::max(length.first, length.second)) + (cluster > 1 ? kSpanJoin : 0.0f)) +
                     kSpanPerPartial * float(s.partials());
    if (cluster == 1 || s.microseconds < best.microseconds) best = s;
  }
  return best;
}

// Rows that see up to `tokens` tokens each: blocks of a cluster for every two query tiles, and the time.
struct SpanWindow {
  int cluster;
  float microseconds;
};
inline SpanWindow span_window(size_t sequences, size_t kv_heads, size_t stacked, size_t tokens) {
  const size_t query_tiles = (stacked + kSpanRows - 1) / kSpanRows, blocks = sequences * kv_heads * ((query_tiles + 1) / 2);
  const size_t tiles = (tokens + kSpanTile - 1) / kSpanTile;
  const size_t steps = query_tiles == 1 ? (tiles + 1) / 2 : tiles;
  SpanWindow best{1, 0.0f};
  for (int cluster = 1; cluster <= kSpanMostCluster; cluster *= 2) {
    const size_t waves = (blocks + span_clusters(cluster) - 1) / span_clusters(cluster);
    const float time = float(waves) * (kSpanFixed + kSpanPerTile * float((steps + cluster - 1) / cluster) +
                                       (cluster > 1 || query_tiles == 1 ? kSpanJoin : 0.0f));
    if (cluster == 1 || time < best.microseconds) best = {cluster, time};
  }
  return best;
}

}  // namespace ei
