// kv8_index.h - index arithmetic of the 8-bit paged K/V cache, shared by its
// kernels and (compiled as plain C++) by the CPU tests: which keys a token
// sees, in which tiles they lie, how the tiles of a ragged batch are split
// over blocks, and the exponent of a block's scale.
#pragma once
#include <cstdint>
#include <cstring>

#ifdef __CUDACC__
#define VCB_HD __host__ __device__ __forceinline__
#else
#define VCB_HD inline
#endif

namespace vcb {

// Keys that the last token of a sequence of `len` tokens sees: [0, sink) and
// [lo, len), sink <= lo. window <= 0: all of them (sink = lo = 0).
struct VisibleKeys {
  int sink, lo, len;
};
VCB_HD VisibleKeys visible_keys(int len, int window, int sinks) {
  VisibleKeys v{0, 0, len > 0 ? len : 0};
  if (window > 0 && window < v.len) {
    v.lo = v.len - window;
    v.sink = sinks < v.lo ? sinks : v.lo;
  }
  return v;
}
VCB_HD bool key_visible(const VisibleKeys &v, int key) {
  return key < v.len && (key >= v.lo || key < v.sink);
}
// The low n bits.
VCB_HD uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1; }
// The same for the 32 keys from `key` on, one bit each.
VCB_HD uint32_t visible_mask(const VisibleKeys &v, int key) {
  return low_bits(v.len - key) & (~low_bits(v.lo - key) | low_bits(v.sink - key));
}

// Those keys as tiles of `tile` keys aligned to multiples of `tile`: first
// `head` tiles from key 0 (the sinks), then the window's from tile `first`.
struct VisibleTiles {
  int head, first, count;
};
VCB_HD VisibleTiles visible_tiles(const VisibleKeys &v, int tile) {
  VisibleTiles t;
  t.first = v.lo / tile;
  const int end = (int)(((int64_t)v.len + tile - 1) / tile);
  t.head = (int)(((int64_t)v.sink + tile - 1) / tile);
  if (t.head > t.first) t.head = t.first;  // the window's first tile holds the rest
  t.count = t.head + end - t.first;
  return t;
}
// First key of tile `i` (0 <= i < count).
VCB_HD int tile_key(const VisibleTiles &t, int i, int tile) {
  return (i < t.head ? i : t.first + (i - t.head)) * tile;
}

// Entries from the first of `n` rows to the end of the last, which takes `last`:
// rows lie `stride` >= 0 apart. What is longer than any memory counts as
// kNoMemory, in sums over several axes too.
constexpr int64_t kNoMemory = (int64_t)1 << 60;
VCB_HD int64_t row_span(int64_t n, int64_t stride, int64_t last) {
  if (n > 1 && stride > (kNoMemory - last) / (n - 1)) return kNoMemory;
  return n > 1 ? (n - 1) * stride + last : last;
}

// Split of `total` > 0 tiles over at most `most` blocks, as even as it gets:
// block c takes [start(c), start(c + 1)), the first `more` blocks one tile more.
struct TileSplit {
  int64_t each;
  int blocks, more;
  VCB_HD TileSplit(int64_t total, int most) {
    blocks = total < most ? (int)total : most;
    each = total / blocks;
    more = (int)(total - each * blocks);
  }
  VCB_HD int64_t start(int c) const { return each * c + (c < more ? c : more); }
  // The block that takes tile t.
  VCB_HD int owner(int64_t t) const {
    const int64_t head = (each + 1) * more;
    return t < head ? (int)(t / (each + 1)) : more + (int)((t - head) / each);
  }
};

// Scale of a block whose largest finite magnitude is `amax`: 2^e, e the
// smallest exponent with amax <= 448 * 2^e (448: the largest e4m3 value,
// 1.75 * 2^8), kept within [-100, 119]. A power of two makes x / scale exact,
// so that the only rounding is the one to 8 bits, and tokens whose scale
// grows later move without a second rounding but in e4m3's subnormals.
constexpr int kScaleMinExp = -100, kScaleMaxExp = 119;
VCB_HD float e4m3_block_scale(float amax) {
  uint32_t b;
#ifdef __CUDA_ARCH__
  b = __float_as_uint(amax);
#else
  std::memcpy(&b, &amax, 4);
#endif
  int e = (int)((b >> 23) & 0xFFu) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  e = e < kScaleMinExp ? kScaleMinExp : e > kScaleMaxExp ? kScaleMaxExp : e;
  const uint32_t s = (uint32_t)(e + 127) << 23;
#ifdef __CUDA_ARCH__
  return __uint_as_float(s);
#else
  float f;
  std::memcpy(&f, &s, 4);
  return f;
#endif
}

}  // namespace vcb
