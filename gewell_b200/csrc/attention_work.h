// How paged attention is cut into pieces.  Plain arithmetic, for the kernel and for tests on the host.
//
// An item is a KV head of a sequence with a tile of its query rows (all query heads of that KV head); it walks over tiles of
// kTokens cached tokens.  An item of n token tiles counts as 1 + n units, the first for what it costs whatever its length
// (queries in, results out).  Items in the order sequence, KV head, query tile form one line of units, which is cut into equal
// ranges, one for each block; an item that a cut divides is computed in pieces and joined afterwards.
#pragma once

#include <cmath>
#include <cstdint>

#ifdef __CUDACC__
#define GW_HOST_DEVICE __host__ __device__ __forceinline__
#define GW_HOST_DEVICE_CALL __host__ __device__ __noinline__      // long code that runs once, in several places
#else
#define GW_HOST_DEVICE inline
#define GW_HOST_DEVICE_CALL inline
#endif

namespace gw {

constexpr int kTokens = 128;      // cached tokens of a tile

// sum of (slope * i + start) / kTokens over i < count, count up to 2^24, slope up to kTokens and the sum below 2^31, by the steps of
// Euclid's algorithm.  In 32 bits: a 64-bit division is 120 instructions.
GW_HOST_DEVICE uint32_t floor_sum(uint32_t count, uint32_t slope, uint32_t start) {
  uint32_t sum = uint32_t(uint64_t(count) * (count - 1) / 2 * (slope / kTokens)) + count * (start / kTokens);
  uint32_t n = count, m = kTokens, a = slope % kTokens, b = start % kTokens;
  while (true) {
    const uint32_t last = a * n + b;              // a, b < m <= kTokens
    if (last < m) return sum;
    n = last / m;
    b = last % m;
    const uint32_t t = m;
    m = a;
    a = t;
    sum += uint32_t(uint64_t(n) * (n - 1) / 2) * (a / m) + n * (b / m);
    a %= m;
    b %= m;
  }
}

// One sequence: `rows` query rows (up to 2^24), the first at position `base` (below 0: no token; up to 2^30), `per_tile` rows a
// query tile, and a window of `window` tokens (0: none; up to 2^30).
struct SequenceWork {
  int32_t base, rows, per_tile, window;

  GW_HOST_DEVICE int32_t query_tiles() const { return (rows + per_tile - 1) / per_tile; }
  // the tokens that a query tile reads: [low, high)
  GW_HOST_DEVICE int32_t low(int32_t tile) const {
    const int32_t at = base + tile * per_tile - window + 1;
    return window == 0 || at < 0 ? 0 : at;
  }
  GW_HOST_DEVICE int32_t high(int32_t tile) const {
    const int32_t end = (tile + 1) * per_tile, at = base + (end < rows ? end : rows);
    return at < 0 ? 0 : at;
  }
  GW_HOST_DEVICE int32_t first_token_tile(int32_t tile) const { return low(tile) / kTokens; }
  GW_HOST_DEVICE int32_t token_tiles(int32_t tile) const { return (high(tile) + kTokens - 1) / kTokens - first_token_tile(tile); }
  // units of the query tiles in front of `tile`
  GW_HOST_DEVICE_CALL uint32_t units_before(int32_t tile) const {
    if (tile <= 0) return 0;
    const int32_t whole = tile < query_tiles() ? tile : tile - 1;       // the last one may have fewer rows
    uint32_t units = tile;
    if (whole < tile) units += token_tiles(whole);
    const int32_t skip_high = base >= 0 ? 0 : -base / per_tile;         // tiles without any token
    if (whole > skip_high) units += floor_sum(whole - skip_high, per_tile, uint32_t(base + (skip_high + 1) * per_tile + kTokens - 1));
    if (window != 0) {
      const int32_t start = base - window + 1, skip_low = start >= 0 ? 0 : (-start + per_tile - 1) / per_tile;
      if (whole > skip_low) units -= floor_sum(whole - skip_low, per_tile, uint32_t(start + skip_low * per_tile));
    }
    return units;
  }
  // perhaps 2^31 units or more, which the sums here cannot hold
  GW_HOST_DEVICE bool too_many() const {
    const float tokens = fmaxf(0.F, float(base) + float(rows)), span = float(window) + float(per_tile);
    const float tiles = float(query_tiles()), with_tokens = fminf(tiles, tokens / float(per_tile) + 1.F);
    return tiles + with_tokens * ((window != 0 ? fminf(span, tokens) : tokens) * (1.F / kTokens) + 3.F) >= 2147483648.F;
  }
  GW_HOST_DEVICE uint32_t units() const { return rows <= 0 ? 0 : rows <= per_tile ? 1 + token_tiles(0) : units_before(query_tiles()); }
};

// `units` in `parts` equal ranges (parts <= units < 2^31, parts up to 2^15).
struct Ranges {
  uint32_t whole, rest, parts;      // units / parts, units % parts
  GW_HOST_DEVICE Ranges(uint32_t units, uint32_t parts) : whole(units / parts), rest(units - units / parts * parts), parts(parts) {}
  GW_HOST_DEVICE uint32_t start(uint32_t part) const { return whole * part + rest * part / parts; }
  // the range that has unit `at`
  GW_HOST_DEVICE uint32_t with(uint32_t at) const {
    uint32_t part = at / whole < parts ? at / whole : parts - 1;
    while (start(part) > at) --part;
    return part;
  }
};

// What the range [from, to) has of an item whose units start at `item`: token tiles [begin, end) of its `tiles`.
struct Piece {
  int32_t begin, end;
  bool here;          // false: nothing of it is computed in this range
};
GW_HOST_DEVICE Piece piece_of(uint32_t item, int32_t tiles, uint32_t from, uint32_t to) {
  const int32_t begin = int32_t(from - item) - 1, end = int32_t(to - item) - 1;
  const int32_t first = begin > 0 ? begin : 0, last = end < tiles ? end : tiles;
  return {first, last, tiles == 0 ? from <= item && item < to : first < last};
}

}  // namespace gw
