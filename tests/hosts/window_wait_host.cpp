// The prompt kernel's longest waits, on the CPU: a pair of row tiles over the
// most keys that the entry takes, at twice the time that a step takes, ends
// before they do.
#include <cstdio>

#include "internal.h"

int main() {
  for (int64_t Nk = 1; Nk <= 1 << 30; Nk *= 2)
    if (vcb::window_pair_wait_ns((int)Nk) < (uint64_t)(Nk + 127) / 128 * 4000) {
      std::printf("FAIL at %d keys\n", (int)Nk);
      return 1;
    }
  std::printf("PASS\n");
  return 0;
}
