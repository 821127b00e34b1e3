// Every token tile of every item lies in exactly one block's range; sums in closed form equal loops.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "attention_work.h"

using namespace gw;

#define REQUIRE(c) do { if (!(c)) { std::printf("FAIL %s:%d %s\n", __FILE__, __LINE__, #c); return 1; } } while (0)

static uint32_t state = 1;
static int draw(int low, int high) {
  state = state * 1664525u + 1013904223u;
  return low + int((state >> 8) % uint32_t(high - low + 1));
}

int main() {
  for (int i = 0; i < 20000; ++i) {
    const int n = draw(1, 300), a = draw(1, kTokens), b = draw(0, 5000);
    uint32_t sum = 0;
    for (int k = 0; k < n; ++k) sum += uint32_t(a * k + b) / kTokens;
    REQUIRE(floor_sum(n, a, b) == sum);
  }
  for (int round = 0; round < 3000; ++round) {
    const int sequences = draw(1, 9), heads = draw(1, 4), per_tile = draw(1, 128), window = draw(0, 2) ? 0 : draw(1, 700);
    std::vector<SequenceWork> all;
    uint32_t units = 0;
    for (int s = 0; s < sequences; ++s) {
      const int rows = draw(0, 3) ? draw(0, 6) : draw(0, 900), context = draw(0, 4) ? rows + draw(0, 3000) : draw(0, rows);
      all.push_back({context - rows, rows, per_tile, window});
      const SequenceWork& w = all.back();
      uint32_t before = 0;
      for (int t = 0; t < w.query_tiles(); ++t) {
        REQUIRE(w.units_before(t) == before);
        REQUIRE(w.token_tiles(t) >= 0 && w.low(t) <= w.high(t));
        before += 1 + w.token_tiles(t);
      }
      REQUIRE(w.units() == before);
      units += before * heads;
    }
    if (units == 0) continue;
    const int parts = int(units < 148 ? draw(1, int(units)) : draw(1, 148));
    const Ranges ranges(units, parts);
    REQUIRE(ranges.start(0) == 0 && ranges.start(parts) == units);
    std::vector<std::vector<int>> taken;       // by item: how often each token tile
    std::vector<int> owners, zeros;
    for (int part = 0; part < parts; ++part) {
      const uint32_t from = ranges.start(part), to = ranges.start(part + 1);
      REQUIRE(from < to && ranges.with(from) == uint32_t(part) && ranges.with(to - 1) == uint32_t(part));
      uint32_t item = 0;
      size_t number = 0;
      int first_pieces = 0, later_pieces = 0;
      for (const SequenceWork& w : all)
        for (int h = 0; h < heads; ++h)
          for (int t = 0; t < w.query_tiles(); ++t, ++number) {
            const int tiles = w.token_tiles(t);
            if (taken.size() <= number) { taken.push_back(std::vector<int>(size_t(tiles))); owners.push_back(0); zeros.push_back(0); }
            const Piece p = piece_of(item, tiles, from, to);
            if (p.here) {
              for (int k = p.begin; k < p.end; ++k) ++taken[number][size_t(k)];
              if (tiles == 0) ++zeros[number];
              if (p.begin > 0) ++later_pieces;
              if (p.begin == 0 && p.end < tiles) {
                ++first_pieces;
                ++owners[number];
                // the blocks of the other pieces are the ones up to that of the last unit
                const int last = int(ranges.with(item + tiles));
                REQUIRE(last > part);
                for (int other = part + 1; other <= last; ++other) {
                  const Piece q = piece_of(item, tiles, ranges.start(other), ranges.start(other + 1));
                  REQUIRE(q.here && q.begin > 0 && (other == last) == (q.end == tiles));
                }
              }
            }
            item += 1 + tiles;
          }
      REQUIRE(item == units && first_pieces <= 1 && later_pieces <= 1);
    }
    for (size_t i = 0; i < taken.size(); ++i) {
      for (int n : taken[i]) REQUIRE(n == 1);
      REQUIRE(owners[i] <= 1 && zeros[i] == (taken[i].empty() ? 1 : 0));
    }
  }
  const SequenceWork far{(1 << 30) - 4096, 4096, 64, 0}, wide{0, 1 << 24, 128, 1 << 20};
  uint32_t units = 0;
  for (int t = 0; t < far.query_tiles(); ++t) units += 1 + far.token_tiles(t);
  REQUIRE(far.units() == units);
  units = 0;
  for (int t = 0; t < wide.query_tiles(); ++t) units += 1 + wide.token_tiles(t);
  REQUIRE(wide.units() == units);
  std::puts("PASS");
  return 0;
}
