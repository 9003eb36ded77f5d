// flash_window.cu - causal attention of prompts through a sliding window,
// with a few first tokens that stay visible (sinks), K/V heads shared by
// groups of query heads, fp16 or bf16.
//
// Query row i of a sequence stands at position t = i + Nk - Nq:
//   O[b, h, i] = sum_j p_j V[b, h / G, j],  p = softmax_2(scale_log2 q . k_j),
// over j <= t with t - j < window or j < sinks, and j < lens[b].
//
// One warp per query row, keys one by one in fp32.
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

template <int D, bool BF16>
__global__ void __launch_bounds__(128) flash_window_kernel(const FlashWindowArgs a) {
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int b = blockIdx.y / a.Hq, h = blockIdx.y % a.Hq, kvh = h / (a.Hq / a.Hkv);
  if (i >= a.Nq) return;
  const int t = i + a.Nk - a.Nq;
  const int n = a.lens ? a.lens[b] : a.Nk;
  if (t >= n && a.lens) return;
  constexpr int E = D / 32;
  float q[E], acc[E];
  for (int e = 0; e < E; ++e) {
    q[e] = load16<BF16>(a.Q, b * a.sq[0] + h * a.sq[1] + i * a.sq[2] + e * 32 + lane) * a.scale_log2;
    acc[e] = 0.0f;
  }
  const VisibleKeys vis = visible_keys(t + 1, a.window, a.sinks);
  float m = -INFINITY, l = 0.0f;
  for (int j = 0; j < vis.len; ++j) {
    if (!key_visible(vis, j)) continue;
    float s = 0.0f;
    for (int e = 0; e < E; ++e)
      s += q[e] * load16<BF16>(a.K, b * a.sk[0] + kvh * a.sk[1] + j * a.sk[2] + e * 32 + lane);
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float m2 = fmaxf(m, s), alpha = exp2f(m - m2), w = exp2f(s - m2);
    l = l * alpha + w;
    for (int e = 0; e < E; ++e)
      acc[e] = acc[e] * alpha +
               w * load16<BF16>(a.V, b * a.sv[0] + kvh * a.sv[1] + j * a.sv[2] + e * 32 + lane);
    m = m2;
  }
  for (int e = 0; e < E; ++e)
    store16<BF16>(a.O, b * a.so[0] + h * a.so[1] + i * a.so[2] + e * 32 + lane,
                  l != 0.0f ? acc[e] / l : 0.0f);
}

}  // namespace

cudaError_t launch_flash_window(const FlashWindowArgs &a, cudaStream_t stream) {
  const dim3 grid((a.Nq + 3) / 4, a.B * a.Hq);
  const bool bf16 = a.dtype == VC_DTYPE_BF16;
  if (a.d == 64)
    bf16 ? flash_window_kernel<64, true><<<grid, 128, 0, stream>>>(a)
         : flash_window_kernel<64, false><<<grid, 128, 0, stream>>>(a);
  else
    bf16 ? flash_window_kernel<128, true><<<grid, 128, 0, stream>>>(a)
         : flash_window_kernel<128, false><<<grid, 128, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace vcb

VCB_DEFINE_ERROR_ACCESSOR(flash_window_error)
