// How paged attention is cut into pieces.  Plain arithmetic, for the kernel and for tests on the host.
//
// An item is a KV head of a sequence with a tile of its query rows (all query heads of that KV head); it walks over tiles of
// kTokens cached tokens.  An item of n token tiles counts as 1 + n units, the first for what it costs whatever its length
// (queries in, results out).  Items in the order sequence, KV head, query tile form one line of units, which is cut into equal
// ranges, one for each block; an item that a cut divides is computed in pieces and joined afterwards.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define GW_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define GW_HOST_DEVICE inline
#endif

namespace gw {

constexpr int kTokens = 128;      // cached tokens of a tile

// sum of (a * i + b) / kTokens over i < n, n up to 2^24 and a up to kTokens, by the steps of Euclid's algorithm.  After the first one
// 32 bits hold everything but the sum, and 32-bit divisions take a fifth of the time that 64-bit ones take.
GW_HOST_DEVICE int64_t floor_sum(int32_t count, int32_t slope, int64_t start) {
  int64_t sum = int64_t(count) * (count - 1) / 2 * (slope / kTokens) + count * (start / kTokens);
  uint32_t n = uint32_t(count), m = kTokens, a = uint32_t(slope % kTokens), b = uint32_t(start % kTokens);
  while (true) {
    const uint32_t last = a * n + b;              // a, b < m <= kTokens
    if (last < m) return sum;
    n = last / m;
    b = last % m;
    const uint32_t t = m;
    m = a;
    a = t;
    sum += int64_t(n) * (n - 1) / 2 * (a / m) + int64_t(n) * (b / m);
    a %= m;
    b %= m;
  }
}

// One sequence: `rows` query rows, the first at position `base` (below 0: no token), `per_tile` rows a query tile, and a window of
// `window` tokens (0: none).
struct SequenceWork {
  int32_t base, rows, per_tile, window;

  GW_HOST_DEVICE int32_t query_tiles() const { return (rows + per_tile - 1) / per_tile; }
  // the tokens that a query tile reads: [low, high)
  GW_HOST_DEVICE int32_t low(int32_t tile) const {
    const int64_t at = int64_t(base) + int64_t(tile) * per_tile - window + 1;
    return window == 0 || at < 0 ? 0 : int32_t(at);
  }
  GW_HOST_DEVICE int32_t high(int32_t tile) const {
    const int64_t end = int64_t(tile + 1) * per_tile, at = int64_t(base) + (end < rows ? end : rows);
    return at < 0 ? 0 : int32_t(at);
  }
  GW_HOST_DEVICE int32_t first_token_tile(int32_t tile) const { return low(tile) / kTokens; }
  GW_HOST_DEVICE int32_t token_tiles(int32_t tile) const { return int32_t((int64_t(high(tile)) + kTokens - 1) / kTokens) - first_token_tile(tile); }
  // units of the query tiles in front of `tile`
  GW_HOST_DEVICE int64_t units_before(int32_t tile) const {
    if (tile <= 0) return 0;
    const int32_t whole = tile < query_tiles() ? tile : tile - 1;       // the last one may have fewer rows
    int64_t units = tile;
    if (whole < tile) units += token_tiles(whole);
    const int64_t skip_high = base >= 0 ? 0 : -int64_t(base) / per_tile;      // tiles without any token
    if (whole > skip_high) units += floor_sum(int32_t(whole - skip_high), per_tile, base + (skip_high + 1) * per_tile + kTokens - 1);
    if (window != 0) {
      const int64_t start = int64_t(base) - window + 1, skip_low = start >= 0 ? 0 : (-start + per_tile - 1) / per_tile;
      if (whole > skip_low) units -= floor_sum(int32_t(whole - skip_low), per_tile, start + skip_low * per_tile);
    }
    return units;
  }
  GW_HOST_DEVICE int64_t units() const { return units_before(query_tiles()); }
};

// Range `part` of `parts` equal ones.
GW_HOST_DEVICE int64_t range_start(int64_t units, int64_t part, int64_t parts) { return units * part / parts; }
// The part that has unit `at`.
GW_HOST_DEVICE int32_t part_with(int64_t units, int64_t at, int64_t parts) {
  int64_t part = at * parts / units;
  while (part + 1 < parts && range_start(units, part + 1, parts) <= at) ++part;
  while (part > 0 && range_start(units, part, parts) > at) --part;
  return int32_t(part);
}

// What the range [from, to) has of an item whose units start at `item`: token tiles [begin, end) of its `tiles`.
struct Piece {
  int32_t begin, end;
  bool here;          // false: nothing of it is computed in this range
};
GW_HOST_DEVICE Piece piece_of(int64_t item, int32_t tiles, int64_t from, int64_t to) {
  const int64_t begin = from - item - 1 > 0 ? from - item - 1 : 0, end = to - item - 1 < tiles ? to - item - 1 : tiles;
  return {int32_t(begin < tiles ? begin : tiles), int32_t(end > 0 ? end : 0), tiles == 0 ? from <= item && item < to : begin < end};
}

}  // namespace gw
