// Checks of csrc/kv8_index.h at the ends of its ranges, on the CPU: spans that
// pass 64 bits.
#include <cstdio>
#include <cstdlib>

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

int main() {
  spans();
  std::printf("PASS\n");
  return 0;
}
