// kv8_pages.cu - writing and moving the pages of the 8-bit paged K/V cache.
//
// A page holds page_size tokens of every K/V head, [heads][page_size][d] e4m3
// codes, with one fp32 scale per head, for K and V apart: x = code * scale.
//
// kv8_append_kernel: new 16-bit K/V tokens into the pages behind each
// sequence's end. A block takes some of the (head, K or V) items of one page:
// it loads an item's new tokens once into registers, takes their largest
// magnitude, raises the page's scale to it where needed (tokens already in the
// page are then re-expressed at the new scale), rounds and stores, while the
// next item's tokens are on their way. 2 bytes are read and 1 written per
// element: bound by HBM, once the pages are enough to fill the GPU.
//
// kv8_copy_kernel: whole pages src[i] -> dst[i], codes and scales, in every
// layer with one launch; bound by HBM.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <mutex>

#include "dependent_launch.cuh"
#include "internal.h"
#include "kv8_index.h"
#include "ptx.cuh"

namespace vcb {
namespace {

template <bool BF16>
__device__ __forceinline__ float2 widen2(uint32_t p) {
  if constexpr (BF16)
    return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xFFFF0000u));
  else
    return __half22float2(*reinterpret_cast<__half2 *>(&p));
}

// Two floats to e4m3 codes (nearest, ties to even; beyond +-448 the largest
// code, NaN stays NaN), the first in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)codes));
  return __half22float2(*reinterpret_cast<__half2 *>(&h));
}

struct AppendParams {
  const void *src[2];  // K, V: [T][heads][d]
  int64_t src_stride[2];
  uint8_t *codes[2];
  float *scales[2];
  int64_t page_stride, scale_stride;
  const int32_t *table, *start, *cu;
  int32_t *lens_out;
  int num_pages, page_size, table_width, max_new, pages_per_seq, T;
  int heads, per_block;  // (K or V, head) items of a block
};

// D / 8 threads per token (8 elements each), PASSES * THREADS * 8 = page_size * D.
// Item i of a page: head i / 2 of K (i even) or V.
template <int D, int THREADS, int PASSES, bool BF16>
__global__ void __launch_bounds__(THREADS) kv8_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kLanes = D / 8;                    // threads per token
  constexpr int kRows = THREADS / kLanes;          // tokens per pass
  const int b = blockIdx.x / p.pages_per_seq;
  const int pi = blockIdx.x % p.pages_per_seq;
  const int P = p.page_size;
  const int item0 = blockIdx.y * p.per_block, item1 = min(item0 + p.per_block, p.heads * 2);

  grid_dependency_wait();
  grid_launch_dependents();

  const int start = p.start[b];
  int64_t row0 = p.cu ? p.cu[b] : (int64_t)b * p.max_new;
  int64_t n = p.cu ? (int64_t)p.cu[b + 1] - row0 : p.max_new;
  // What the caller's arrays say is checked before anything is read by it.
  const int64_t room = (int64_t)p.table_width * P;
  bool bad = start < 0 || n < 0 || n > p.max_new || row0 < 0 || row0 + n > p.T;
  if (bad) n = 0;
  if (!bad && start + n > room) {
    bad = true;
    n = start < room ? room - start : 0;
  }
  const bool first_block = pi == 0 && item0 == 0 && threadIdx.x == 0;
  if (first_block && p.lens_out) p.lens_out[b] = (int32_t)(bad && n == 0 ? (start < 0 ? 0 : start) : start + n);
  if (first_block && bad) record_error(kErrOutOfBounds);
  const int64_t pos0 = start > 0 ? start : 0;
  const int64_t page_idx = pos0 / P + pi;
  if (n == 0 || page_idx * P >= pos0 + n) return;
  // Slots [s0, s1) of this page are new.
  const int s0 = (int)(pos0 > page_idx * P ? pos0 - page_idx * P : 0);
  const int s1 = (int)(pos0 + n - page_idx * P < P ? pos0 + n - page_idx * P : P);
  const int page = p.table[(int64_t)b * p.table_width + page_idx];
  if (page < 0 || page >= p.num_pages) {
    if (threadIdx.x == 0) record_error(kErrOutOfBounds);
    return;
  }
  // Token of slot s: row0 + (page_idx * P + s - pos0).
  const int64_t tok0 = row0 + page_idx * P - pos0;
  const int lane = threadIdx.x % kLanes;
  const int row = threadIdx.x / kLanes;
  __shared__ uint32_t warp_max[2][THREADS / 32];

  auto load = [&](int item, uint4 (&x)[PASSES], float &old) {
    const int kv = item & 1, head = item >> 1;
    const char *src = static_cast<const char *>(p.src[kv]) +
                      (tok0 * p.src_stride[kv] + (int64_t)head * D + lane * 8) * 2;
    old = s0 > 0 ? p.scales[kv][(int64_t)page * p.scale_stride + head] : 0.0f;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int s = i * kRows + row;
      x[i] = make_uint4(0, 0, 0, 0);
      if (s >= s0 && s < s1) x[i] = __ldcs(reinterpret_cast<const uint4 *>(src + s * p.src_stride[kv] * 2));
    }
  };
  uint4 x[PASSES], next[PASSES];
  float old_raw, old_next = 0.0f;
  load(item0, x, old_raw);
#pragma unroll 1
  for (int item = item0; item < item1; ++item) {
    if (item + 1 < item1) load(item + 1, next, old_next);  // while this one is worked on
    const int kv = item & 1, head = item >> 1;
    uint8_t *codes = p.codes[kv] + (int64_t)page * p.page_stride + (int64_t)head * P * D;
    // Magnitudes of 16-bit floats order as their bits do, infinity and NaN on
    // top: one packed maximum per pair, and a second look only where it meets
    // one of those (an infinity saturates instead of setting the scale).
    constexpr uint32_t kInf = BF16 ? 0x7F80u : 0x7C00u;
    uint32_t top2 = 0;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      top2 = __vmaxu2(top2, x[i].x & 0x7FFF7FFFu);
      top2 = __vmaxu2(top2, x[i].y & 0x7FFF7FFFu);
      top2 = __vmaxu2(top2, x[i].z & 0x7FFF7FFFu);
      top2 = __vmaxu2(top2, x[i].w & 0x7FFF7FFFu);
    }
    uint32_t *const tops = warp_max[item & 1];  // the item before may still be read
    auto block_max = [&](uint32_t v) {
      v = __reduce_max_sync(0xffffffffu, v);
      if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = v;
      __syncthreads();  // also: every thread has read the old scale
#pragma unroll
      for (int i = 0; i < THREADS / 32; ++i) v = max(v, tops[i]);
      return v;
    };
    uint32_t top = block_max(max(top2 & 0xFFFFu, top2 >> 16));
    if (top >= kInf) {
      uint32_t finite = 0;
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t lo = w[j] & 0x7FFFu, hi = w[j] >> 16 & 0x7FFFu;
          if (lo < kInf) finite = max(finite, lo);
          if (hi < kInf) finite = max(finite, hi);
        }
      }
      __syncthreads();  // every thread has read the first maxima
      top = block_max(finite);
    }
    const float amax = widen2<BF16>(top).x;

    const float old = old_raw > 0.0f && old_raw < INFINITY ? old_raw : 0.0f;
    const float sc = fmaxf(e4m3_block_scale(amax), old);
    if (threadIdx.x == 0) p.scales[kv][(int64_t)page * p.scale_stride + head] = sc;
    if (s0 > 0 && sc != old) {
      // The page's earlier tokens at the larger scale.
      for (int s = row; s < s0; s += kRows) {
        uint2 *at = reinterpret_cast<uint2 *>(codes + s * D + lane * 8);
        const uint2 q = *at;
        uint32_t out[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t w = j ? q.y : q.x;
          const float2 a = from_e4m3x2(w & 0xFFFFu), c = from_e4m3x2(w >> 16);
          out[j] = to_e4m3x2(a.x * old / sc, a.y * old / sc) |
                   to_e4m3x2(c.x * old / sc, c.y * old / sc) << 16;
        }
        *at = make_uint2(out[0], out[1]);
      }
    }
    // x / sc: a multiplication where sc is a power of two (exact), else the
    // correctly rounded quotient. fp16 pairs multiply and convert packed where
    // 1 / sc is an fp16 number: what underflows there is zero in e4m3 as well.
    auto store = [&](auto codes_of) {
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int s = i * kRows + row;
        if (s < s0 || s >= s1) continue;
        *reinterpret_cast<uint2 *>(codes + s * D + lane * 8) =
            make_uint2(codes_of(x[i].x) | codes_of(x[i].y) << 16, codes_of(x[i].z) | codes_of(x[i].w) << 16);
      }
    };
    const bool pow2 = (__float_as_uint(sc) & 0x7FFFFFu) == 0;
    const float inv = 1.0f / sc;
    if (pow2 && !BF16 && inv <= 32768.0f && inv >= 6.103515625e-05f) {
      const __half2 f = __float2half2_rn(inv);
      store([&](uint32_t w) {
        const __half2 y = __hmul2(*reinterpret_cast<const __half2 *>(&w), f);
        uint16_t r;
        asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t *>(&y)));
        return (uint32_t)r;
      });
    } else if (pow2) {
      store([&](uint32_t w) {
        const float2 f = widen2<BF16>(w);
        return to_e4m3x2(f.x * inv, f.y * inv);
      });
    } else {
      store([&](uint32_t w) {
        const float2 f = widen2<BF16>(w);
        return to_e4m3x2(f.x / sc, f.y / sc);
      });
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) x[i] = next[i];
    old_raw = old_next;
  }
}

// At most 4 passes: 32 bytes of a token's tile in a thread's registers, and as
// many of the next item's.
template <int D, bool BF16>
cudaError_t append_launch(const AppendParams &p, dim3 grid, cudaStream_t s) {
  switch (p.page_size * D) {
    case 1024: return launch_dependent(kv8_append_kernel<D, 128, 1, BF16>, grid, 128, 0, p, s);
    case 2048: return launch_dependent(kv8_append_kernel<D, 128, 2, BF16>, grid, 128, 0, p, s);
    case 4096: return launch_dependent(kv8_append_kernel<D, 128, 4, BF16>, grid, 128, 0, p, s);
    case 8192: return launch_dependent(kv8_append_kernel<D, 256, 4, BF16>, grid, 256, 0, p, s);
    case 16384: return launch_dependent(kv8_append_kernel<D, 512, 4, BF16>, grid, 512, 0, p, s);
    default: return cudaErrorInvalidValue;
  }
}

// ------------------------------------------------------------------ copy
constexpr int kCopyLayers = 64;          // layers a launch takes
// Units of 16 KB, 2 blocks of 96 KB of ring per SM: 900 pages of 64 KB in 8
// layers 156 us (6.07 TB/s), 8 pages of 128 KB in 16 layers 6.3 us. With 8 KB
// units the one issuing thread is the bound (157 to 241 us); with 32 KB 152 us,
// but 7.2 for the small case; 16-byte loads and stores by 8 blocks of 256
// threads took 169 and 6.5 us.
constexpr int kCopyChunk = 16384;        // bytes of a unit
constexpr int kCopyStages = 6;           // of a block's ring
constexpr int kCopyLag = 3;              // loads that run ahead of the stores
constexpr int kCopyBlocksPerSm = 2;

struct CopyParams {
  uint8_t *codes[kCopyLayers][2];
  float *scales[kCopyLayers][2];
  const int32_t *src, *dst;
  int64_t page_stride, scale_stride;
  int64_t units;           // n * layers * 2 * chunks
  int num_pages, layers, heads, chunks, page_bytes;
};

// One thread of warp 0 moves the codes through a ring of shared memory with
// 1-D bulk copies, in and out again; warp 1 moves the scales.
__global__ void __launch_bounds__(64) kv8_copy_kernel(const __grid_constant__ CopyParams p) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full[kCopyStages];
  __shared__ uint8_t *to[kCopyStages];  // of the loads on their way
  __shared__ uint32_t bytes[kCopyStages];
  if (threadIdx.x == 0) {
    for (int i = 0; i < kCopyStages; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  __syncthreads();
  grid_dependency_wait();
  fence_proxy_async_global();  // the bulk copies read what the launch before wrote
  grid_launch_dependents();
  const int64_t per_pair = (int64_t)p.layers * 2 * p.chunks;
  if (threadIdx.x >= 32) {
    // Scales: units of (pair, layer, K or V).
    const int lane = threadIdx.x - 32;
    for (int64_t u = blockIdx.x; u < p.units / p.chunks; u += gridDim.x) {
      const int64_t i = u / (p.layers * 2);
      const int which = (int)(u - i * (p.layers * 2));
      const int src = p.src[i], dst = p.dst[i];
      if (src < 0 || src >= p.num_pages || dst < 0 || dst >= p.num_pages) {
        if (lane == 0) record_error(kErrOutOfBounds);
        continue;
      }
      float *s = p.scales[which >> 1][which & 1];
      if (src != dst)
        for (int h = lane; h < p.heads; h += 32)
          s[(int64_t)dst * p.scale_stride + h] = s[(int64_t)src * p.scale_stride + h];
    }
    return;
  }
  if (threadIdx.x != 0) return;
  // The unit's place; its page numbers are fetched a unit ahead.
  int64_t u = blockIdx.x;
  int src = -1, dst = -1;
  if (u < p.units) {
    src = p.src[u / per_pair];
    dst = p.dst[u / per_pair];
  }
  int loaded = 0, stored = 0;
  bool ok = true;
  auto store = [&]() {
    const int st = stored % kCopyStages;
    ok = mbar_wait(&full[st], (stored / kCopyStages) & 1);
    if (!ok) return;
    bulk_store_1d(to[st], ring + st * kCopyChunk, bytes[st]);
    bulk_commit_group();
    ++stored;
  };
  for (; ok && u < p.units;) {
    const int64_t r = u % per_pair;
    const int which = (int)(r / p.chunks), chunk = (int)(r % p.chunks);
    const bool good = src >= 0 && src < p.num_pages && dst >= 0 && dst < p.num_pages && src != dst;
    uint8_t *base = p.codes[which >> 1][which & 1] + (int64_t)chunk * kCopyChunk;
    uint8_t *from = base + (int64_t)src * p.page_stride, *dest = base + (int64_t)dst * p.page_stride;
    u += gridDim.x;
    if (u < p.units) {
      src = p.src[u / per_pair];
      dst = p.dst[u / per_pair];
    }
    if (!good) continue;  // out of range (the scales' warp reports it), or onto itself
    if (loaded >= kCopyLag) store();
    if (!ok) break;
    // The stage's last store, kCopyStages loads ago, has been read.
    bulk_wait_group_read<kCopyStages - kCopyLag>();
    const int st = loaded % kCopyStages;
    bytes[st] = min(kCopyChunk, p.page_bytes - chunk * kCopyChunk);
    to[st] = dest;
    mbar_arrive_expect_tx(&full[st], bytes[st]);
    bulk_load_1d(ring + st * kCopyChunk, from, bytes[st], &full[st]);
    ++loaded;
  }
  while (ok && stored < loaded) store();
  // After a wait that ran out, copies on their way get time to land.
  for (; !ok && stored < loaded; ++stored)
    mbar_wait(&full[stored % kCopyStages], (stored / kCopyStages) & 1, 1000000000ull);
  bulk_wait_group<0>();
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8AppendArgs &a, cudaStream_t stream) {
  const vc_kv8_cache &c = *a.cache;
  AppendParams p;
  p.src[0] = a.K;
  p.src[1] = a.V;
  p.src_stride[0] = a.k_stride;
  p.src_stride[1] = a.v_stride;
  p.codes[0] = static_cast<uint8_t *>(c.k);
  p.codes[1] = static_cast<uint8_t *>(c.v);
  p.scales[0] = c.k_scale;
  p.scales[1] = c.v_scale;
  p.page_stride = c.page_stride;
  p.scale_stride = c.scale_stride;
  p.table = a.table;
  p.start = a.start;
  p.cu = a.cu;
  p.lens_out = a.lens_out;
  p.num_pages = c.num_pages;
  p.page_size = c.page_size;
  p.table_width = a.table_width;
  p.max_new = a.max_new;
  p.T = a.T;
  // max_new tokens from any slot touch at most this many pages.
  const int64_t pages = ((int64_t)a.max_new - 1 + c.page_size - 1) / c.page_size + 1;
  if (pages * a.B > INT32_MAX) return cudaErrorInvalidValue;
  p.pages_per_seq = (int)pages;
  // Several items in a block hide the look-up of lengths and page, and the
  // next item's loads, behind the first one's work; more of them leave a tail
  // in which few blocks work. 37k tokens of 8 heads with 2 / 4 / 8 / 16 items
  // a block: 46.5 / 43.0 / 44.1 / 49.6 us; 32 single tokens with 1 / 2 / 4 / 8:
  // 3.7 / 3.2 / 4.0 / 6.0 us.
  const int64_t items = (int64_t)c.heads * 2;
  p.heads = c.heads;
  p.per_block = pages * a.B * items >= (int64_t)sm_count_current() * 32 ? 4 : 2;
  const dim3 grid((unsigned)(pages * a.B), (unsigned)((items + p.per_block - 1) / p.per_block));
  const bool bf16 = a.dtype == VC_DTYPE_BF16;
  if (c.head_dim == 64)
    return bf16 ? append_launch<64, true>(p, grid, stream) : append_launch<64, false>(p, grid, stream);
  return bf16 ? append_launch<128, true>(p, grid, stream) : append_launch<128, false>(p, grid, stream);
}

cudaError_t launch_kv8_copy(const vc_kv8_cache *layers, int n_layers, const int32_t *src,
                            const int32_t *dst, int n, cudaStream_t stream) {
  for (int l0 = 0; l0 < n_layers; l0 += kCopyLayers) {
    CopyParams p;
    p.layers = n_layers - l0 < kCopyLayers ? n_layers - l0 : kCopyLayers;
    for (int l = 0; l < p.layers; ++l) {
      const vc_kv8_cache &c = layers[l0 + l];
      p.codes[l][0] = static_cast<uint8_t *>(c.k);
      p.codes[l][1] = static_cast<uint8_t *>(c.v);
      p.scales[l][0] = c.k_scale;
      p.scales[l][1] = c.v_scale;
    }
    const vc_kv8_cache &c = layers[0];
    p.src = src;
    p.dst = dst;
    p.page_stride = c.page_stride;
    p.scale_stride = c.scale_stride;
    p.num_pages = c.num_pages;
    p.heads = c.heads;
    p.page_bytes = c.heads * c.page_size * c.head_dim;
    p.chunks = (p.page_bytes + kCopyChunk - 1) / kCopyChunk;
    p.units = (int64_t)n * p.layers * 2 * p.chunks;
    const int64_t most = (int64_t)sm_count_current() * kCopyBlocksPerSm;
    const unsigned grid = (unsigned)(p.units < most ? p.units : most);
    constexpr int bytes = kCopyStages * kCopyChunk;
    static uint64_t configured = 0;  // devices whose smem attribute is set
    static std::mutex mu;
    int dev = 0;
    cudaGetDevice(&dev);
    {
      std::lock_guard<std::mutex> lk(mu);
      if (dev >= 64 || !(configured & (1ull << dev))) {
        cudaError_t e = cudaFuncSetAttribute(kv8_copy_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured |= (1ull << dev);
      }
    }
    cudaError_t e = launch_dependent(kv8_copy_kernel, dim3(grid), 64, bytes, p, stream);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace vcb

VCB_DEFINE_ERROR_ACCESSOR(kv8_pages_error)
