// flash_window.cu - causal attention of prompts through a sliding window,
// with a few first tokens that stay visible (sinks), K/V heads shared by
// groups of query heads, on sm_100a tensor cores: fp16 or bf16 Q/K/V/O, fp32
// scores, softmax statistics and accumulator.
//
// Query row i of a sequence stands at position t = i + Nk - Nq:
//   O[b, h, i] = sum_j p_j V[b, h / G, j],  p = softmax_2(scale_log2 q . k_j),
// over j <= t with t - j < window or j < sinks, and j < lens[b].
//
// Bound: the tensor cores, 4 d operations per visible (row, key) pair.
//
// The pipeline is the one of the plain forward (flash_fwd_tcgen05.cu): one CTA
// per SM, two tiles of 128 query rows, 128-key tiles of K and V through a ring
// of two stages of (V(u - 1), K(u)), one thread that issues the MMAs
//   S_w = Q_w K^T (shared memory), O_w += P_w V (P_w in TMEM),
// so that the softmax of one tile runs under the MMAs of the other, P handed
// over in two halves, O rescaled when the maximum grows by more than 2^8.
//
// What differs is which tiles meet. The row tiles of all query heads of a K/V
// head, (rows 0..127 of its G heads, rows 128..255, ...), are paired in that
// order, so that both tiles of a CTA mostly have the same rows, and with them
// the same keys, and every K/V tile that is loaded serves two heads. A CTA
// walks the union of its two tiles' key tiles - those of the sinks, then from
// the window's lower edge to the diagonal - and each row tile skips the ones
// it does not see. Only tiles on an edge are masked.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <mutex>

#include "internal.h"
#include "ptx.cuh"

namespace vcb {
namespace {

constexpr int BQ = 128;    // query rows per tile (two tiles per CTA)
constexpr int BKV = 128;   // keys per tile
constexpr int kStages = 2;
constexpr int kThreads = 384;  // 12 warps of 168 registers, split 232 (softmax) / 40 (the rest)
constexpr int kWgThreads = 128;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kBoxBytes = 128 * 128;  // 128 rows x 64 16-bit elements
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr int kHandoffs = 2;               // parts in which P reaches the MMAs
constexpr int kChunksPerHandoff = (BKV / 32) / kHandoffs;
// K/V slices per ordering group (heaviest CTAs of every slice of a group first).
constexpr int kOrderGroup = 8;

struct __align__(8) WindowBarriers {
  uint64_t q_full;
  uint64_t kv_full[kStages];
  uint64_t kv_empty[kStages];
  uint64_t v_clean;  // V rows behind the sequence's end are zeroed
  uint64_t s_full[2];
  uint64_t p_full[2][kHandoffs];
  uint64_t o_full[2];
  uint32_t tmem_base;
};

template <int HD>
struct WindowSmem {
  static constexpr uint32_t kTile = (HD / 64) * kBoxBytes;  // one Q, K or V tile
  static constexpr uint32_t kRing = 2 * kTile;              // behind the two Q tiles
  static constexpr uint32_t kBars = kRing + kStages * 2 * kTile;
  static constexpr size_t kUsed = 1024 + kBars + sizeof(WindowBarriers);
  // At least 120 KiB so that a second CTA never shares the SM: each CTA
  // allocates all 512 TMEM columns.
  static constexpr size_t kBytes = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
};

struct WindowParams {
  CUtensorMap q, k, v, o;  // (d, tokens, heads, batch)
  const int32_t *lens;
  uint16_t *O;
  int64_t so[3];
  int Hq, Hkv, Nq, Nk, window, sinks;
  float scale_log2;
};

// Key tiles of a tile of query rows: t < hi with t >= lo or t < sink.
struct KeyTiles {
  int sink, lo, hi;
  __device__ __forceinline__ bool has(int t) const { return t < hi && (t >= lo || t < sink); }
  __device__ __forceinline__ int count() const { return hi - lo + min(sink, lo); }
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
  } else {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
  }
}

template <int HD, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
flash_window_kernel(const __grid_constant__ WindowParams p) {
  using L = WindowSmem<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  WindowBarriers *bars = reinterpret_cast<WindowBarriers *>(smem + L::kBars);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // ---- which row tiles: groups of K/V slices, the last rows (with the most
  // keys) of every slice of a group first.
  int pair, slice;
  {
    const int64_t lin = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int g = (int)(lin / ((int64_t)kOrderGroup * gridDim.x));
    const int first = g * kOrderGroup;
    const int gsz = min(kOrderGroup, (int)gridDim.y - first);
    const int r = (int)(lin - (int64_t)g * kOrderGroup * gridDim.x);
    pair = gridDim.x - 1 - r / gsz;
    slice = first + r % gsz;
  }
  const int group = p.Hq / p.Hkv;
  const int b = slice / p.Hkv, kvh = slice % p.Hkv;
  const int shift = p.Nk - p.Nq;  // position of row 0
  const int n = p.lens ? min(max(p.lens[b], 0), p.Nk) : p.Nk;
  const int units = (p.Nq + BQ - 1) / BQ * group;
  int row0[2], head[2];
  KeyTiles kt[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int unit = 2 * pair + w;
    row0[w] = unit / group * BQ;
    head[w] = kvh * group + unit % group;
    // Positions of the rows that are computed: the last one has the most keys.
    const int t_first = max(row0[w] + shift, 0);
    const int t_last = min(min(row0[w] + BQ, p.Nq) - 1 + shift, n - 1);
    kt[w] = {0, 0, 0};
    if (unit < units && t_last >= t_first) {
      kt[w].hi = t_last / BKV + 1;
      if (p.window > 0) {
        kt[w].lo = max(t_first - p.window + 1, 0) / BKV;
        kt[w].sink = (int)min(((int64_t)p.sinks + BKV - 1) / BKV, (int64_t)kt[w].lo);
      }
    }
  }
  const int count0 = kt[0].count(), count1 = kt[1].count();
  // The union of both: tiles [0, sink), then [lo, hi).
  const int lo = count0 && count1 ? min(kt[0].lo, kt[1].lo) : count0 ? kt[0].lo : kt[1].lo;
  const int hi = max(kt[0].hi, kt[1].hi);
  const int sink = min(max(kt[0].sink, kt[1].sink), lo);
  const int total = hi - lo + sink;
  auto tile_of = [&](int u) { return u < sink ? u : lo + (u - sink); };
  // V's rows behind the end of a padded sequence are zeroed in its last tile:
  // their weights are 0, but 0 times what they hold may not be.
  const bool clean = n < p.Nk && hi > 0 && hi * BKV > n;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->kv_full[s], 1);
      mbar_init(&bars->kv_empty[s], 1);
    }
    mbar_init(&bars->v_clean, 1);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&bars->s_full[w], 1);
      for (int h = 0; h < kHandoffs; ++h)
        mbar_init(&bars->p_full[w][h], kWgThreads / 32);  // one per warp
      mbar_init(&bars->o_full[w], 1);
    }
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  // 256 x 232 + 128 x 40 = 384 x 168 registers.
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // -------------------------------------------------- softmax, warps 0..7
    const int w = warp >> 2;              // which query tile
    const int quad = warp & 3;            // TMEM lane quadrant
    const int row = quad * 32 + lane;     // row within the tile == TMEM lane
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t s_col = tmem + lane_off + w * 128;
    const uint32_t o_col = tmem + lane_off + 256 + w * 128;
    const KeyTiles mine = w ? kt[1] : kt[0];
    const int my_count = w ? count1 : count0;
    const int my_row0 = w ? row0[1] : row0[0], my_head = w ? head[1] : head[0];
    const int t_first = my_row0 + shift, t = t_first + row;  // positions
    float m_run = -INFINITY;  // running max of scale_log2 * s
    float l_run = 0.0f;
    bool ok = true;
    int j = 0;                // key tiles so far
    for (int u = 0; u < total; ++u) {
      const int tile = tile_of(u);
      if (!mine.has(tile)) continue;
      if (!mbar_wait(&bars->s_full[w], j & 1)) ok = false;
      // Warp-uniform status: the TMEM accesses below are warp-collective.
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      const int key0 = tile * BKV;
      // The whole S row in registers with one wait.
      uint32_t s[BKV / 32][32];
      if constexpr (BF16) {
#pragma unroll
        for (int c = 0; c < BKV / 32; ++c) tmem_ld32(s_col + c * 32, s[c]);
      } else {
        tmem_ld128(s_col, *reinterpret_cast<uint32_t(*)[128]>(&s[0][0]));
      }
      tmem_ld_wait();
      // Keys key0 + x of this row: hidden from x = end on, and below `begin`
      // where they are no sinks (x >= keep).
      if (key0 + BKV - 1 > t_first) {
        const int end = t - key0 + 1;
#pragma unroll
        for (int c = 0; c < BKV / 32; ++c)
#pragma unroll
          for (int x = 0; x < 32; ++x)
            if (c * 32 + x >= end) s[c][x] = __float_as_uint(-INFINITY);
      }
      if (p.window > 0 && t_first + BQ - 1 - key0 >= p.window && key0 + BKV > p.sinks) {
        const int begin = t - p.window + 1 - key0, keep = p.sinks - key0;
#pragma unroll
        for (int c = 0; c < BKV / 32; ++c)
#pragma unroll
          for (int x = 0; x < 32; ++x)
            if (c * 32 + x < begin && c * 32 + x >= keep) s[c][x] = __float_as_uint(-INFINITY);
      }
      // Row max: three-input max into 4 independent partial maxima.
      float mxp[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < BKV / 32; ++c)
#pragma unroll
        for (int x = 0; x < 32; x += 2)
          mxp[(x >> 1) & 3] = fmax3(mxp[(x >> 1) & 3], __uint_as_float(s[c][x]),
                                    __uint_as_float(s[c][x + 1]));
      const float mx = fmax3(fmaxf(mxp[0], mxp[1]), mxp[2], mxp[3]);
      const float m_cand = fmaxf(m_run, mx * p.scale_log2);
      const bool grow = m_cand > m_run + kRescaleThreshold;  // true where the first keys appear
      // Warp-uniform decision (TMEM loads and stores are warp-collective).
      const bool rescale = __any_sync(0xffffffffu, grow);
      float alpha = 1.0f;
      if (rescale) {
        // A row may still have seen no key (then it stays at minus infinity).
        if (m_cand != -INFINITY) alpha = ex2_approx(m_run - m_cand);
        l_run *= alpha;
        m_run = m_cand;
      }
      const float m_use = (m_run == -INFINITY) ? 0.0f : m_run;
      const bool rescale_o = rescale && j > 0;  // warp-uniform
      int handed = 0;                           // parts of P handed over
      // P = exp2(scale_log2 * s - m) -> 16-bit pairs over S columns.
      float lsp[4] = {0.f, 0.f, 0.f, 0.f};
      const float neg_m = -m_use, scale = p.scale_log2;
#pragma unroll
      for (int c = 0; c < BKV / 32; ++c) {
        uint32_t pr[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          float x0, x1;
          fma2(x0, x1, __uint_as_float(s[c][2 * x]), __uint_as_float(s[c][2 * x + 1]), scale, scale,
               neg_m, neg_m);
          // Masked scores are -inf: the exponential returns exactly 0.
          const float p0 = ex2_approx(x0);
          const float p1 = ex2_approx(x1);
          pr[x] = pack2<BF16>(p0, p1);
          // bf16: the row sum adds the rounded values, so numerator and
          // denominator use the same weights (with one dominant key the
          // unrounded sum would leave that key's 2^-9 rounding in O).
          const int a = 2 * (x & 1);
          if constexpr (BF16)
            add_bf16x2_to_f32(lsp[a], lsp[a + 1], pr[x]);
          else
            add2(lsp[a], lsp[a + 1], lsp[a], lsp[a + 1], p0, p1);
        }
        tmem_st16(s_col + c * 16, pr);
        if (rescale_o && c == 1) {
          // S_w complete implies that O_w's products so far are: O_w is stable,
          // and the next wait for the hand-offs below.
#pragma unroll
          for (int oc = 0; oc < HD / 32; ++oc) {
            uint32_t o[32];
            tmem_ld32(o_col + oc * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
            tmem_st32(o_col + oc * 32, o);
          }
        }
        // Hand over every part whose P is complete (with an O rescale
        // pending, not before it is done).
        if ((c + 1) % kChunksPerHandoff == 0 && (!rescale_o || c >= 1)) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          const int upto = c / kChunksPerHandoff;
          if (lane == 0)
            for (int h = handed; h <= upto; ++h) mbar_arrive(&bars->p_full[w][h]);
          handed = upto + 1;
        }
      }
      l_run += (lsp[0] + lsp[1]) + (lsp[2] + lsp[3]);
      ++j;
      if (!ok) break;
    }
    // Epilogue: O / l -> 16-bit. Rows of the sequence (t < n); a row without a
    // key is zero.
    const bool exists = 2 * pair + w < units;
    const bool mine_row = my_row0 + row < p.Nq && (!p.lens || t < n);
    const float inv_l = l_run != 0.0f ? 1.0f / l_run : 0.0f;
    const bool whole = !p.lens || t_first + BQ <= n;  // of the tile, but for rows past Nq
    uint16_t *out = p.O + b * p.so[0] + my_head * p.so[1] + (int64_t)(my_row0 + row) * p.so[2];
    if (exists && my_count == 0) {
      if (mine_row && t < 0)
        for (int c = 0; c < HD / 8; ++c) reinterpret_cast<uint4 *>(out)[c] = make_uint4(0, 0, 0, 0);
    } else if (__all_sync(0xffffffffu, ok && exists && mbar_wait(&bars->o_full[w], 0))) {
      tc_fence_after();
      uint8_t *stage = smem + w * L::kTile;  // over this tile's Q
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(o_col + c * 32, o);
        tmem_ld_wait();
        uint8_t *rowp = stage + (c / 2) * kBoxBytes + row * 128;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4 v;
          v.x = pack2<BF16>(__uint_as_float(o[8 * q + 0]) * inv_l, __uint_as_float(o[8 * q + 1]) * inv_l);
          v.y = pack2<BF16>(__uint_as_float(o[8 * q + 2]) * inv_l, __uint_as_float(o[8 * q + 3]) * inv_l);
          v.z = pack2<BF16>(__uint_as_float(o[8 * q + 4]) * inv_l, __uint_as_float(o[8 * q + 5]) * inv_l);
          v.w = pack2<BF16>(__uint_as_float(o[8 * q + 6]) * inv_l, __uint_as_float(o[8 * q + 7]) * inv_l);
          if (whole) {
            const int chunk = (c % 2) * 4 + q;
            *reinterpret_cast<uint4 *>(rowp + ((chunk ^ (row & 7)) * 16)) = v;
          } else if (mine_row) {
            reinterpret_cast<uint4 *>(out)[c * 4 + q] = v;
          }
        }
      }
      if (whole) {
        fence_proxy_async_smem();
        named_bar_sync(1 + w, kWgThreads);
        if (quad == 0 && lane == 0) {
#pragma unroll
          for (int c = 0; c < HD / 64; ++c)
            tma_store_4d(&p.o, stage + c * kBoxBytes, c * 64, my_row0, my_head, b);
          bulk_commit_group();
          bulk_wait_group<0>();
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
  if (warp == 8) {
    int issued = 0;
    if (lane == 0 && total > 0) {
      // ------------------------------------------------ TMA producer
      tma_prefetch_desc(&p.q);
      tma_prefetch_desc(&p.k);
      tma_prefetch_desc(&p.v);
      mbar_arrive_expect_tx(&bars->q_full, ((count0 > 0) + (count1 > 0)) * L::kTile);
#pragma unroll
      for (int w = 0; w < 2; ++w)
        if (w ? count1 > 0 : count0 > 0) {
#pragma unroll
          for (int c = 0; c < HD / 64; ++c)
            tma_load_4d(smem + w * L::kTile + c * kBoxBytes, &p.q, c * 64, row0[w], head[w], b,
                        &bars->q_full);
        }
      // Stage s = 0..total: V(s - 1) in its first tile slot (from s = 1), K(s)
      // in its second (up to s = total - 1).
      for (int s = 0; s <= total; ++s) {
        const int st = s % kStages;
        if (!mbar_wait(&bars->kv_empty[st], ((s / kStages) & 1) ^ 1)) break;
        mbar_arrive_expect_tx(&bars->kv_full[st], ((s >= 1) + (s < total)) * L::kTile);
        uint8_t *slot = smem + L::kRing + st * 2 * L::kTile;
        const int kv = tile_of(s - 1) * BKV, kk = tile_of(s) * BKV;
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) {
          if (s >= 1)
            tma_load_4d(slot + c * kBoxBytes, &p.v, c * 64, kv, kvh, b, &bars->kv_full[st]);
          if (s < total)
            tma_load_4d(slot + L::kTile + c * kBoxBytes, &p.k, c * 64, kk, kvh, b,
                        &bars->kv_full[st]);
        }
        ++issued;
      }
    }
    issued = __shfl_sync(0xffffffffu, issued, 0);
    if (clean && issued == total + 1) {
      // The last V tile, in stage `total`.
      const int st = total % kStages;
      bool ok = mbar_wait(&bars->kv_full[st], (total / kStages) & 1);
      uint8_t *v = smem + L::kRing + st * 2 * L::kTile;
      const int first = n - (hi - 1) * BKV;  // a 128-byte row per token and box
      if (ok)
        for (int i = lane; i < (BKV - first) * 8; i += 32)
#pragma unroll
          for (int c = 0; c < HD / 64; ++c)
            *reinterpret_cast<uint4 *>(v + c * kBoxBytes + first * 128 + i * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->v_clean);
    }
    if (lane == 0 && total > 0) {
      // No copy is in flight when the CTA ends.
      mbar_wait(&bars->q_full, 0, 1000000000ull);
      const int last = issued < kStages ? issued : kStages;
      for (int i = 0; i < last; ++i) {
        const int s = issued - 1 - i;
        mbar_wait(&bars->kv_full[s % kStages], (s / kStages) & 1, 1000000000ull);
      }
    }
  } else if (warp == 9) {
    if (lane == 0 && total > 0) {
      // ------------------------------------------------ MMA issuer
      const uint32_t idesc_s = idesc_f16_f32(BQ, BKV, BF16, false, false);
      const uint32_t idesc_o = idesc_f16_f32(BQ, HD, BF16, false, true);
      // Descriptors are built once; a byte offset within the shared window is
      // an add of (offset >> 4) to the descriptor's address field.
      const uint64_t dq = smem_desc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t dk = smem_desc_sw128(smem_u32(smem + L::kRing), 16, 1024);
      const uint64_t dv = smem_desc_sw128(smem_u32(smem + L::kRing), kBoxBytes, 1024);
      const uint32_t dq_hi = (uint32_t)(dq >> 32), dk_hi = (uint32_t)(dk >> 32), dv_hi = (uint32_t)(dv >> 32);
      // K(s) and V(s - 1) of stage s: second and first tile slot.
      auto issue_s = [&](int w, int s) {
        const uint32_t q_lo = (uint32_t)dq + w * (L::kTile >> 4);
        const uint32_t k_lo = (uint32_t)dk + ((((s % kStages) * 2 + 1) * L::kTile) >> 4);
        const uint32_t d_tmem = tmem + w * 128;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          const uint32_t off = (ks / 4) * (kBoxBytes >> 4) + (ks % 4) * (32 >> 4);
          mma_f16_ss_lohi(d_tmem, q_lo + off, dq_hi, k_lo + off, dk_hi, idesc_s, ks > 0 ? 1u : 0u);
        }
        mma_commit(&bars->s_full[w]);
      };
      int done[2] = {0, 0};  // PV products of each row tile so far
      auto issue_pv = [&](int w, int s) {
        const uint32_t v_lo = (uint32_t)dv + ((((s % kStages) * 2) * L::kTile) >> 4);
        const uint32_t o_tmem = tmem + 256 + w * 128, p_tmem = tmem + w * 128;
        constexpr int kSteps = (BKV / 16) / kHandoffs;  // K = 16 MMAs per part
#pragma unroll
        for (int h = 0; h < kHandoffs; ++h) {
          if (!mbar_wait(&bars->p_full[w][h], done[w] & 1)) return false;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < kSteps; ++kk) {
            const int ks = h * kSteps + kk;
            mma_f16_ts_lohi(o_tmem, p_tmem + ks * 8, v_lo + ks * ((16 * 128) >> 4), dv_hi, idesc_o,
                            (done[w] > 0 || ks > 0) ? 1u : 0u);
          }
        }
        // Only the epilogue waits for O: one commit after the tile's last PV.
        if (++done[w] == (w ? count1 : count0)) mma_commit(&bars->o_full[w]);
        return true;
      };
      auto wait_stage = [&](int s) {
        const bool ok = mbar_wait(&bars->kv_full[s % kStages], (s / kStages) & 1);
        tc_fence_after();
        return ok;
      };
      bool ok = mbar_wait(&bars->q_full, 0) && wait_stage(0);
      if (ok) {
        if (kt[0].has(tile_of(0))) issue_s(0, 0);
        if (kt[1].has(tile_of(0))) issue_s(1, 0);
        mma_commit(&bars->kv_empty[0]);
      }
      // Step u: stage u + 1 brings V(u) and K(u + 1); one commit after the
      // step's last MMA releases it.
      for (int u = 0; ok && u < total; ++u) {
        const int s = u + 1;
        if (!wait_stage(s)) break;
        if (clean && s == total && !mbar_wait(&bars->v_clean, 0)) break;
        const int t = tile_of(u), t_next = tile_of(s);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (kt[w].has(t)) ok = ok && issue_pv(w, s);
          if (ok && s < total && kt[w].has(t_next)) issue_s(w, s);
        }
        if (ok) mma_commit(&bars->kv_empty[s % kStages]);
      }
    }
  }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, kTmemCols);
}

// ------------------------------------------------------------ host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                  const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// (d, tokens, heads, batch) at element strides s (batch, head, token).
bool make_map(CUtensorMap *map, bool bf16, const void *base, int B, int H, int N, int d,
              const int64_t *s) {
  auto encode = reinterpret_cast<EncodeTiledFn>(tensor_map_encoder());
  if (!encode) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)N, (cuuint64_t)H, (cuuint64_t)B};
  const cuuint64_t strides[3] = {(cuuint64_t)s[2] * 2, (cuuint64_t)s[1] * 2, (cuuint64_t)s[0] * 2};
  const cuuint32_t box[4] = {64, 128, 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, bool BF16>
cudaError_t launch_typed(const WindowParams &p, dim3 grid, cudaStream_t stream) {
  static uint64_t configured = 0;  // devices whose smem attribute is set
  static std::mutex mu;
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (dev >= 64 || !(configured & (1ull << dev))) {
      cudaError_t e = cudaFuncSetAttribute(flash_window_kernel<HD, BF16>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)WindowSmem<HD>::kBytes);
      if (e != cudaSuccess) return e;
      if (dev < 64) configured |= (1ull << dev);
    }
  }
  flash_window_kernel<HD, BF16><<<grid, kThreads, WindowSmem<HD>::kBytes, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_flash_window(const FlashWindowArgs &a, cudaStream_t stream) {
  const bool bf16 = a.dtype == VC_DTYPE_BF16;
  WindowParams p;
  if (!make_map(&p.q, bf16, a.Q, a.B, a.Hq, a.Nq, a.d, a.sq) ||
      !make_map(&p.k, bf16, a.K, a.B, a.Hkv, a.Nk, a.d, a.sk) ||
      !make_map(&p.v, bf16, a.V, a.B, a.Hkv, a.Nk, a.d, a.sv) ||
      !make_map(&p.o, bf16, a.O, a.B, a.Hq, a.Nq, a.d, a.so))
    return cudaErrorInvalidValue;
  p.lens = a.lens;
  p.O = static_cast<uint16_t *>(a.O);
  for (int i = 0; i < 3; ++i) p.so[i] = a.so[i];
  p.Hq = a.Hq;
  p.Hkv = a.Hkv;
  p.Nq = a.Nq;
  p.Nk = a.Nk;
  p.window = a.window;
  p.sinks = a.sinks;
  p.scale_log2 = a.scale_log2;
  const int64_t units = ((int64_t)a.Nq + BQ - 1) / BQ * (a.Hq / a.Hkv);
  if (units > INT32_MAX / 2) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)((units + 1) / 2), a.B * a.Hkv);
  if (a.d == 64)
    return bf16 ? launch_typed<64, true>(p, grid, stream) : launch_typed<64, false>(p, grid, stream);
  return bf16 ? launch_typed<128, true>(p, grid, stream) : launch_typed<128, false>(p, grid, stream);
}

}  // namespace vcb

VCB_DEFINE_ERROR_ACCESSOR(flash_window_error)
