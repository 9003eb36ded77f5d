// Checks of the paged cache's index arithmetic (csrc/kv8_index.h) on the CPU:
// every tile a kernel reads lies within its sequence, every visible key lies
// in exactly one tile, and the split over blocks covers each tile once.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "kv8_index.h"

using namespace vcb;

#define CHECK(c)                                                       \
  do {                                                                 \
    if (!(c)) {                                                        \
      std::printf("FAIL line %d: %s\n", __LINE__, #c);                 \
      std::exit(1);                                                    \
    }                                                                  \
  } while (0)

static void tiles(int len, int window, int sinks, int tile) {
  const VisibleKeys v = visible_keys(len, window, sinks);
  const VisibleTiles t = visible_tiles(v, tile);
  CHECK(t.count >= 0 && t.head >= 0);
  std::vector<int> seen(len > 0 ? len + tile : tile, 0);
  int last = -1;
  for (int i = 0; i < t.count; ++i) {
    const int k0 = tile_key(t, i, tile);
    CHECK(k0 % tile == 0 && k0 > last && k0 < len);
    last = k0;
    for (int k = k0; k < k0 + tile && k < len; ++k) ++seen[k];
  }
  for (int k = 0; k < len; ++k) {
    const bool see = window <= 0 || k >= len - window || k < sinks;
    CHECK(key_visible(v, k) == see);
    CHECK(seen[k] <= 1);
    if (see) CHECK(seen[k] == 1);
  }
  CHECK(!key_visible(v, len > 0 ? len : 0));
}

int main() {
  const int lens[] = {0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 500, 1000, 1023};
  const int windows[] = {0, 1, 2, 15, 16, 17, 64, 100, 128, 511, 1000, 5000};
  const int sinks[] = {0, 1, 4, 16, 17, 63, 64, 65, 130, 2000};
  for (int len : lens)
    for (int w : windows)
      for (int s : sinks)
        for (int tile : {16, 32, 64, 128}) tiles(len, w, s, tile);
  // The largest lengths: no overflow.
  const VisibleTiles big = visible_tiles(visible_keys(2147483647, 0, 0), 64);
  CHECK(big.count == 33554432);

  for (int64_t total : {(int64_t)1, (int64_t)2, (int64_t)7, (int64_t)147, (int64_t)148, (int64_t)149,
                        (int64_t)1000, (int64_t)4099, (int64_t)1 << 33})
    for (int most : {1, 2, 3, 148, 296, 444, 592}) {
      const TileSplit sp(total, most);
      CHECK(sp.blocks >= 1 && sp.blocks <= most && sp.blocks <= total);
      CHECK(sp.start(0) == 0 && sp.start(sp.blocks) == total);
      for (int c = 0; c < sp.blocks; ++c) {
        const int64_t n = sp.start(c + 1) - sp.start(c);
        CHECK(n == total / sp.blocks || n == total / sp.blocks + 1);
        CHECK(sp.owner(sp.start(c)) == c && sp.owner(sp.start(c + 1) - 1) == c);
        if (total < 5000)
          for (int64_t t = sp.start(c); t < sp.start(c + 1); ++t) CHECK(sp.owner(t) == c);
      }
    }

  for (int e = -140; e < 128; ++e)
    for (float m : {1.0f, 1.25f, 1.75f, 1.7500001f, 1.9999999f}) {
      const float a = std::ldexp(m, e), s = e4m3_block_scale(a);
      int want = -100;
      while (want < 119 && (double)a > 448.0 * std::ldexp(1.0, want)) ++want;
      CHECK((double)s == std::ldexp(1.0, want));
    }
  CHECK(e4m3_block_scale(0.0f) == std::ldexp(1.0f, -100));
  std::printf("PASS\n");
  return 0;
}
