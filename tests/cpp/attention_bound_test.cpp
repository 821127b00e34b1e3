// The bound that keeps an item's units within 31 bits lies above the units, and not far above.
#include <cstdint>
#include <cstdio>
#include <initializer_list>

#include "attention_work.h"

using namespace gw;

int main() {
  const int rows[] = {1, 2, 63, 64, 65, 1000, 1 << 16, (1 << 24) - 1, 1 << 24}, contexts[] = {1, 200, 1 << 20, 1 << 24, (1 << 30) - 5, 1 << 30};
  int refused = 0, taken = 0;
  for (int r : rows)
    for (int c : contexts)
      for (int per_tile : {1, 8, 64})
        for (int window : {0, 1, 1000, 1 << 20, 1 << 30}) {
          const SequenceWork w{c - r, r, per_tile, window};
          uint64_t units = 0;
          for (int t = 0; t < w.query_tiles(); ++t) units += 1 + uint64_t(w.token_tiles(t));
          if (w.too_many()) {
            ++refused;
            if (units < 500000000ull) { std::printf("FAIL refused %d %d %d %d: %llu\n", r, c, per_tile, window, (unsigned long long)units); return 1; }
          } else {
            ++taken;
            if (w.units() != units) { std::printf("FAIL %d %d %d %d: %u, not %llu\n", r, c, per_tile, window, w.units(), (unsigned long long)units); return 1; }
          }
        }
  if (refused < 20 || taken < 100) { std::printf("FAIL %d %d\n", refused, taken); return 1; }
  std::printf("PASS\n");
}
