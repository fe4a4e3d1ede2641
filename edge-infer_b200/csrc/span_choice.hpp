// How the many-row attention over one stretch of tokens is cut into blocks, in a plain header so that it is tested without a GPU.
#pragma once

#include <algorithm>
#include <cstddef>

namespace ei {

constexpr int kSpanTile = 64;    // tokens of a tile
constexpr int kSpanBox = 32;     // tokens of a copy: a tile may be put together from several stretches
constexpr int kSpanRows = 128;   // stacked query rows of a query tile; a block has two

// A prefix that all rows see, `query_tiles` query tiles per KV head. Pairs of query tiles share the tiles of tokens they read
// and are cut into `pair_splits` stretches; an odd last one has both halves of its blocks to itself, every other tile of
// tokens each, and is cut into `single_splits`. So that no block has much more to do than another, a single's stretch is
// twice as long.
struct SpanSplits {
  int pairs, pair_splits, single_splits;  // single_splits 0: no odd tile
  int blocks() const { return pairs * pair_splits + single_splits; }
  int partials() const { return std::max(pairs ? pair_splits : 0, 2 * single_splits); }  // of a row, at most
};
constexpr int kSpanMostPartials = 32;
inline SpanSplits span_splits(size_t query_tiles, size_t tokens, int kv_heads, int multiprocessors) {
  const int tiles = int((tokens + kSpanTile - 1) / kSpanTile);
  SpanSplits s{int(query_tiles / 2), 1, int(query_tiles % 2)};
  // Grow the number of stretches, always of the kind whose blocks are longer, while the blocks still fit the chip at once
  // and a stretch keeps two tiles (of a single: two for each half).
  for (;;) {
    const int pair_length = s.pairs ? (tiles + s.pair_splits - 1) / s.pair_splits : 0;
    const int single_length = s.single_splits ? (tiles + 2 * s.single_splits - 1) / (2 * s.single_splits) : 0;
    SpanSplits next = s;
    if (pair_length >= single_length) ++next.pair_splits;
    else ++next.single_splits;
    if (std::max(pair_length, single_length) < 2 || next.partials() > kSpanMostPartials ||
        (long long)next.blocks() * kv_heads > multiprocessors)
      return s;
    s = next;
  }
}

}  // namespace ei
