// kv8_attn.cu - attention of single tokens over the 8-bit paged K/V cache.
//
// One query token per sequence, at position lens[b] - 1:
//   O[b, h] = sum_j p_j v_j,  p = softmax_2(scale_log2 * q . k_j),
// over the keys j < lens[b] with j >= lens[b] - window or j < sinks, where
// k_j = k_scale * code of the page that holds j (v_j alike).
//
// One warp per (sequence, query head): a lane holds d / 32 elements of q and
// of the accumulator, and the keys pass one by one with the running maximum
// and sum of the softmax.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "internal.h"
#include "kv8_index.h"
#include "ptx.cuh"

namespace vcb {
namespace {

template <bool BF16>
__device__ __forceinline__ float load16(const void *p, int64_t i) {
  if constexpr (BF16)
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
  else
    return __half2float(static_cast<const __half *>(p)[i]);
}
template <bool BF16>
__device__ __forceinline__ void store16(void *p, int64_t i, float v) {
  if constexpr (BF16)
    static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16(v);
  else
    static_cast<__half *>(p)[i] = __float2half(v);
}
__device__ __forceinline__ float from_e4m3(uint8_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)c));
  return __half2float(__ushort_as_half((unsigned short)(h & 0xFFFFu)));
}

struct AttnParams {
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  int64_t page_stride, scale_stride, q_stride, o_stride;
  const void *Q;
  void *O;
  const int32_t *table, *lens;
  int num_pages, page_size, heads, Hq, table_width, window, sinks;
  float scale_log2;
};

template <int D, bool BF16>
__global__ void __launch_bounds__(32) kv8_attn_kernel(const AttnParams p) {
  const int b = blockIdx.y, h = blockIdx.x, kvh = h / (p.Hq / p.heads);
  const int lane = threadIdx.x;
  constexpr int E = D / 32;
  float q[E], acc[E];
  for (int e = 0; e < E; ++e) {
    q[e] = load16<BF16>(p.Q, b * p.q_stride + (int64_t)h * D + e * 32 + lane) * p.scale_log2;
    acc[e] = 0.0f;
  }
  int64_t len = p.lens[b];
  if (len < 0 || len > (int64_t)p.table_width * p.page_size) {
    if (lane == 0) record_error(kErrOutOfBounds);
    len = len < 0 ? 0 : (int64_t)p.table_width * p.page_size;
  }
  const VisibleKeys vis = visible_keys((int)len, p.window, p.sinks);
  float m = -INFINITY, l = 0.0f;
  for (int j = 0; j < vis.len; ++j) {
    if (!key_visible(vis, j)) continue;
    const int page = p.table[(int64_t)b * p.table_width + j / p.page_size];
    if (page < 0 || page >= p.num_pages) {
      if (lane == 0) record_error(kErrOutOfBounds);
      continue;
    }
    const int64_t at = page * p.page_stride + ((int64_t)kvh * p.page_size + j % p.page_size) * D;
    const int64_t sc = page * p.scale_stride + kvh;
    float s = 0.0f;
    for (int e = 0; e < E; ++e) s += q[e] * from_e4m3(p.k[at + e * 32 + lane]);
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= p.k_scale[sc];
    const float m2 = fmaxf(m, s), alpha = exp2f(m - m2), w = exp2f(s - m2);
    l = l * alpha + w;
    const float wv = w * p.v_scale[sc];
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * alpha + wv * from_e4m3(p.v[at + e * 32 + lane]);
    m = m2;
  }
  for (int e = 0; e < E; ++e)
    store16<BF16>(p.O, b * p.o_stride + (int64_t)h * D + e * 32 + lane, l != 0.0f ? acc[e] / l : 0.0f);
}

}  // namespace

size_t kv8_attn_workspace_bytes(const vc_kv8_cache &, int, int) { return 256; }

cudaError_t launch_kv8_attn(const Kv8AttnArgs &a, cudaStream_t stream) {
  const vc_kv8_cache &c = *a.cache;
  const AttnParams p{static_cast<const uint8_t *>(c.k), static_cast<const uint8_t *>(c.v),
                     c.k_scale, c.v_scale, c.page_stride, c.scale_stride, a.q_stride, a.o_stride,
                     a.Q, a.O, a.table, a.lens, c.num_pages, c.page_size, c.heads, a.Hq,
                     a.table_width, a.window, a.sinks, a.scale_log2};
  const dim3 grid(a.Hq, a.B);
  const bool bf16 = a.dtype == VC_DTYPE_BF16;
  if (c.head_dim == 64)
    bf16 ? kv8_attn_kernel<64, true><<<grid, 32, 0, stream>>>(p)
         : kv8_attn_kernel<64, false><<<grid, 32, 0, stream>>>(p);
  else
    bf16 ? kv8_attn_kernel<128, true><<<grid, 32, 0, stream>>>(p)
         : kv8_attn_kernel<128, false><<<grid, 32, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace vcb

VCB_DEFINE_ERROR_ACCESSOR(kv8_attn_error)
