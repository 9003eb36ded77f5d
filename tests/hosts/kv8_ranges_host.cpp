// Checks of csrc/kv8_index.h at the ends of its ranges, on the CPU: spans that
// pass 64 bits, the longest sequences with the longest windows and sinks, and
// the masks that the kernel takes its keys by.
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "kv8_index.h"

using namespace vcb;

#define CHECK(c)                                                       \
  do {                                                                 \
    if (!(c)) {                                                        \
      std::printf("FAIL line %d: %s\n", __LINE__, #c);                 \
      std::exit(1);                                                    \
    }                                                                  \
  } while (0)

static void spans() {
  const int64_t ns[] = {1, 2, 3, 1000, (1 << 25) + 1, 2147483647}, strides[] = {0, 1, 64, 4096, (int64_t)1 << 38, (int64_t)1 << 40},
                lasts[] = {1, 64, 1 << 20, kNoMemory};
  for (int64_t n : ns)
    for (int64_t s : strides)
      for (int64_t last : lasts) {
        const __int128 want = (__int128)(n - 1) * s + last;
        CHECK(row_span(n, s, last) == (want >= kNoMemory ? kNoMemory : (int64_t)want));
      }
  // 2^25 pages 2^39 bytes apart are 2^64 bytes, which wrap to none.
  CHECK(row_span((1 << 25) + 1, (int64_t)1 << 39, 1 << 20) == kNoMemory);
  CHECK(row_span(2, (int64_t)1 << 39, row_span((1 << 25) + 1, (int64_t)1 << 39, 1)) == kNoMemory);
}

// The tiles of a sequence, by their borders: within it, each once, and the
// visible keys at the borders of the sinks and the window in one of them.
static void tiles(int len, int window, int sinks, int tile) {
  const VisibleKeys v = visible_keys(len, window, sinks);
  const VisibleTiles t = visible_tiles(v, tile);
  const int64_t end = ((int64_t)len + tile - 1) / tile;
  CHECK(t.head >= 0 && t.head <= t.first && t.first < end && t.count == t.head + (end - t.first));
  auto has = [&](int key) { return key / tile < t.head || key / tile >= t.first; };
  for (int key : {0, v.sink - 1, v.sink, v.lo - 1, v.lo, len - 1}) {
    if (key < 0 || key >= len) continue;
    const bool see = window <= 0 || key >= (int64_t)len - window || key < sinks;
    CHECK(key_visible(v, key) == see);
    if (see) CHECK(has(key));
  }
  // A warp's 32 keys of a tile, bit by bit, at every tile of short sequences and
  // around the borders of long ones.
  auto mask = [&](int64_t tile0) {
    for (int64_t key = tile0; key < tile0 + 128 && key + 31 <= 2147483647; key += 32)
      for (int i = 0; i < 32; ++i)
        CHECK((visible_mask(v, (int)key) >> i & 1) == (uint32_t)key_visible(v, (int)key + i));
  };
  if (len <= 1100)
    for (int64_t k = 0; k < end * tile; k += 128) mask(k);
  else
    for (int64_t key : {(int64_t)0, (int64_t)v.sink, (int64_t)v.lo, (int64_t)len - 1}) mask(key / 128 * 128);
  CHECK(tile_key(t, 0, tile) == (t.head || !t.first ? 0 : t.first * tile));
  CHECK(tile_key(t, t.count - 1, tile) == (end - 1) * tile);
}

int main() {
  spans();
  const int most = 2147483647;
  for (int len : {1, 31, 32, 33, 127, 128, 129, 500, 1023, 1100})
    for (int window : {0, 1, 2, 17, 31, 32, 33, 100, 128, 511, 5000})
      for (int sinks : {0, 1, 4, 31, 32, 33, 64, 130, 2000}) tiles(len, window, sinks, 128);
  for (int len : {1, 100, 128, 129, most - 128, most - 127, most - 15, most - 1, most})
    for (int window : {0, 1, 64, 128, 1 << 30, most - 1, most})
      for (int sinks : {0, 1, 128, 1 << 30, most - 127, most - 126, most - 1, most})
        for (int tile : {16, 64, 128}) tiles(len, window, sinks, tile);
  std::printf("PASS\n");
  return 0;
}
