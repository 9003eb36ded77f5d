// kv8_pages.cu - writing and moving the pages of the 8-bit paged K/V cache.
//
// A page holds page_size tokens of every K/V head, [heads][page_size][d] e4m3
// codes, with one fp32 scale per head, for K and V apart: x = code * scale.
//
// kv8_append_kernel: new 16-bit K/V tokens into the pages behind each
// sequence's end. One block per (page touched, head, K or V): it loads the
// page's new tokens once into registers, takes their largest magnitude,
// raises the page's scale to it where needed (tokens already in the page are
// then re-expressed at the new scale), rounds and stores. 2 bytes are read
// and 1 written per element.
//
// kv8_copy_kernel: whole pages src[i] -> dst[i], codes and scales, in every
// layer with one launch; 16-byte copies, bound by HBM.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "internal.h"
#include "kv8_index.h"
#include "ptx.cuh"

namespace vcb {
namespace {

constexpr int kAppendThreads = 128;

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
};

// D / 8 threads per token (8 elements each), PASSES * 128 * 8 = page_size * D.
template <int D, int PASSES, bool BF16>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const AppendParams p) {
  constexpr int kLanes = D / 8;                    // threads per token
  constexpr int kRows = kAppendThreads / kLanes;   // tokens per pass
  const int b = blockIdx.x / p.pages_per_seq;
  const int pi = blockIdx.x % p.pages_per_seq;
  const int head = blockIdx.y;
  const int kv = blockIdx.z;
  const int P = p.page_size;

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
  const bool first_block = pi == 0 && head == 0 && kv == 0 && threadIdx.x == 0;
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
  uint8_t *codes = p.codes[kv] + (int64_t)page * p.page_stride + (int64_t)head * P * D;
  float *scale = p.scales[kv] + (int64_t)page * p.scale_stride + head;
  // Token of slot s: row0 + (page_idx * P + s - pos0).
  const int64_t tok0 = row0 + page_idx * P - pos0;
  const char *src = static_cast<const char *>(p.src[kv]);
  const int lane = threadIdx.x % kLanes;
  const int row = threadIdx.x / kLanes;
  const float old_raw = s0 > 0 ? *scale : 0.0f;

  uint4 x[PASSES];
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int s = i * kRows + row;
    x[i] = make_uint4(0, 0, 0, 0);
    if (s >= s0 && s < s1)
      x[i] = *reinterpret_cast<const uint4 *>(
          src + ((tok0 + s) * p.src_stride[kv] + (int64_t)head * D + lane * 8) * 2);
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = widen2<BF16>(w[j]);
      const float a = fabsf(f.x), c = fabsf(f.y);
      // fmaxf passes NaN over; an infinity saturates instead of setting the scale.
      if (a < INFINITY) amax = fmaxf(amax, a);
      if (c < INFINITY) amax = fmaxf(amax, c);
    }
  }
  __shared__ float warp_max[kAppendThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = amax;
  __syncthreads();  // also: every thread has read the old scale
#pragma unroll
  for (int i = 0; i < kAppendThreads / 32; ++i) amax = fmaxf(amax, warp_max[i]);

  const float old = old_raw > 0.0f && old_raw < INFINITY ? old_raw : 0.0f;
  const float sc = fmaxf(e4m3_block_scale(amax), old);
  if (threadIdx.x == 0) *scale = sc;
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
  // correctly rounded quotient.
  const bool pow2 = (__float_as_uint(sc) & 0x7FFFFFu) == 0;
  const float inv = 1.0f / sc;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int s = i * kRows + row;
    if (s < s0 || s >= s1) continue;
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = widen2<BF16>(w[j]);
      c[j] = pow2 ? to_e4m3x2(f.x * inv, f.y * inv) : to_e4m3x2(f.x / sc, f.y / sc);
    }
    *reinterpret_cast<uint2 *>(codes + s * D + lane * 8) =
        make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
  }
}

template <int D, int PASSES>
void append_launch(const AppendParams &p, dim3 grid, bool bf16, cudaStream_t s) {
  if (bf16)
    kv8_append_kernel<D, PASSES, true><<<grid, kAppendThreads, 0, s>>>(p);
  else
    kv8_append_kernel<D, PASSES, false><<<grid, kAppendThreads, 0, s>>>(p);
}

// ------------------------------------------------------------------ copy
constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 4;                                   // 16-byte loads in flight a thread
constexpr int kCopyChunk = kCopyThreads * kCopyVecs * 16;      // bytes a block moves at a time
constexpr int kCopyLayers = 64;                                // layers a launch takes

struct CopyParams {
  uint8_t *codes[kCopyLayers][2];
  float *scales[kCopyLayers][2];
  const int32_t *src, *dst;
  int64_t page_stride, scale_stride;
  int64_t units;           // n * layers * 2 * chunks
  int num_pages, layers, heads, chunks, page_bytes;
};

__global__ void __launch_bounds__(kCopyThreads) kv8_copy_kernel(const __grid_constant__ CopyParams p) {
  for (int64_t u = blockIdx.x; u < p.units; u += gridDim.x) {
    const int chunk = (int)(u % p.chunks);
    int64_t r = u / p.chunks;
    const int kv = (int)(r & 1);
    r >>= 1;
    const int layer = (int)(r % p.layers);
    const int64_t i = r / p.layers;
    const int src = p.src[i], dst = p.dst[i];
    if (src < 0 || src >= p.num_pages || dst < 0 || dst >= p.num_pages) {
      if (threadIdx.x == 0) record_error(kErrOutOfBounds);
      continue;
    }
    if (src == dst) continue;
    const uint8_t *from = p.codes[layer][kv] + (int64_t)src * p.page_stride;
    uint8_t *to = p.codes[layer][kv] + (int64_t)dst * p.page_stride;
    uint4 v[kCopyVecs];
    const int base = chunk * kCopyChunk + threadIdx.x * 16;
#pragma unroll
    for (int j = 0; j < kCopyVecs; ++j) {
      const int at = base + j * kCopyThreads * 16;
      if (at < p.page_bytes) v[j] = __ldcs(reinterpret_cast<const uint4 *>(from + at));
    }
#pragma unroll
    for (int j = 0; j < kCopyVecs; ++j) {
      const int at = base + j * kCopyThreads * 16;
      if (at < p.page_bytes) __stcs(reinterpret_cast<uint4 *>(to + at), v[j]);
    }
    if (chunk == 0)
      for (int h = threadIdx.x; h < p.heads; h += kCopyThreads)
        p.scales[layer][kv][(int64_t)dst * p.scale_stride + h] =
            p.scales[layer][kv][(int64_t)src * p.scale_stride + h];
  }
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
  const dim3 grid((unsigned)(pages * a.B), c.heads, 2);
  const bool bf16 = a.dtype == VC_DTYPE_BF16;
  const int passes = c.page_size * c.head_dim / (kAppendThreads * 8);
  if (c.head_dim == 64) {
    switch (passes) {
      case 1: append_launch<64, 1>(p, grid, bf16, stream); break;
      case 2: append_launch<64, 2>(p, grid, bf16, stream); break;
      case 4: append_launch<64, 4>(p, grid, bf16, stream); break;
      case 8: append_launch<64, 8>(p, grid, bf16, stream); break;
      default: return cudaErrorInvalidValue;
    }
  } else {
    switch (passes) {
      case 2: append_launch<128, 2>(p, grid, bf16, stream); break;
      case 4: append_launch<128, 4>(p, grid, bf16, stream); break;
      case 8: append_launch<128, 8>(p, grid, bf16, stream); break;
      case 16: append_launch<128, 16>(p, grid, bf16, stream); break;
      default: return cudaErrorInvalidValue;
    }
  }
  return cudaGetLastError();
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
    const int64_t most = (int64_t)sm_count_current() * 8;
    const unsigned grid = (unsigned)(p.units < most ? p.units : most);
    kv8_copy_kernel<<<grid, kCopyThreads, 0, stream>>>(p);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace vcb

VCB_DEFINE_ERROR_ACCESSOR(kv8_pages_error)
