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
// Measured (bf16, 32 heads over 8 K/V heads of 128, short runs at 1.9 GHz): 8192
// tokens through a window of 2048 246 us, 980 TFLOP/s of visible work; the last
// 2048 of 6144 through 4096 268 us, 1030 TFLOP/s (0.62 of the dense peak); on
// another GPU 271 and 291 us. A step of 128 keys
// for both row tiles takes ~3600 cycles, of which the MMAs are 2048; the issuing
// warp spends ~2500 (75 to 80 cycles an MMA) and waits ~900 for P.
//
// The pipeline is the one of the plain forward (flash_fwd_tcgen05.cu): one CTA
// per SM, two tiles of 128 query rows, 128-key tiles of K and V through a ring
// of two stages of (V(u - 1), K(u)), one thread that issues the MMAs
//   S_w = Q_w K^T (shared memory), O_w += P_w V (P_w in TMEM),
// so that the softmax of one tile runs under the MMAs of the other, P handed
// over in two parts, O rescaled when the maximum grows by more than 2^8.
//
// The CTAs are persistent: each takes its next pair of row tiles from the
// grid's queue (cluster launch control), and the steps of one pair follow on
// those of the last: the stage of a pair's last V brings the next pair's first
// K, and its first S products are issued between the last PV products, so that
// they run under the last softmax and the epilogue (set-up, fill and epilogue
// of a fresh CTA took 7 us, of 21 to 69 in all). A scheduler warp takes the
// pairs and writes what the other warps need into shared memory. The whole
// issuing warp runs its loop, on values that are broadcast, so that descriptors
// stay in uniform registers (one lane on values out of shared memory took 3540
// cycles a step to issue instead of 2500), and the registers are split between
// the roles (168 for all cost 11 % of the time in spills).
//
// What differs is which tiles meet. The row tiles of all query heads of a K/V
// head, (rows 0..127 of its G heads, rows 128..255, ...), are paired in that
// order, so that both tiles of a CTA mostly have the same rows, and with them
// the same keys, and every K/V tile that is loaded serves two heads. A CTA
// walks the union of its two tiles' key tiles - those of the sinks, then from
// the window's lower edge to the diagonal - and each row tile skips the ones
// it does not see. Only tiles on an edge are masked.
//
// Few row tiles (SPLIT): a step takes as long with one tile as with two, because
// a tile's scores, softmax and products follow one another. So a CTA takes one
// row tile and each half of it takes half of its keys, with its own S, O, maximum
// and sum; at the end the first half's warps read both O from TMEM.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <mutex>

#include "dependent_launch.cuh"
#include "internal.h"
#include "ptx.cuh"

namespace vcb {
namespace {

constexpr int BQ = 128;    // query rows per tile (two tiles per CTA)
constexpr int BKV = 128;   // keys per tile
constexpr int kStages = 2;
constexpr int kThreads = 384;  // 12 warps of 168 registers, split 216 (softmax) / 72 (the rest)
constexpr int kWgThreads = 128;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kBoxBytes = 128 * 128;  // 128 rows x 64 16-bit elements
constexpr float kRescaleThreshold = 8.0f;  // log2 units
// P reaches the MMAs in two parts: 96 keys, whose products run under the
// exponentials of the last 32, and those, whose products are all that the next
// scores wait for (64 + 64 took 2 to 3 % longer, four parts of 32 7 %).
constexpr int kFirstKeys = 96;
// K/V slices per ordering group (heaviest CTAs of every slice of a group first).
constexpr int kOrderGroup = 8;

// Key tiles of a tile of query rows: t < hi with t >= lo or t < sink.
struct KeyTiles {
  int sink, lo, hi;
  __device__ __forceinline__ bool has(int t) const { return t < hi && (t >= lo || t < sink); }
  __device__ __forceinline__ int count() const { return hi - lo + min(sink, lo); }
};

// A pair of row tiles of the query heads that share a K/V head, and the key
// tiles of their union: [0, sink), then [lo, hi). Or (SPLIT) one row tile, whose
// key tiles the two halves of the CTA share: they take them in turns, one the
// lower half of the list, the other, which has the last turn, the upper.
struct Work {
  int valid;                   // 0: the queue is empty
  int b, kvh, n;               // n: tokens of the sequence
  int row0[2], head[2], count[2], exists[2];
  KeyTiles kt[2];
  int lo, hi, sink, total;
  int clean;                   // V's rows from n on are zeroed in the last tile
  int chained;                 // K(0) shares the stage of the last pair's last V (pairs only)
  int stage0, n_live, n_clean; // stage of K(0); pairs with keys, cleaned tiles before this one
};
// Key tile of step u of a list [0, sink), [lo, ...) of `total`.
template <bool SPLIT>
__device__ __forceinline__ int tile_of(int u, int total, int sink, int lo) {
  const int i = !SPLIT ? u : (u >> 1) + ((u ^ (total - 1)) & 1 ? 0 : total >> 1);
  return i < sink ? i : lo + (i - sink);
}

struct __align__(16) WindowBarriers {
  uint4 answer;  // of the grid's queue
  Work work[2];
  uint64_t answer_full;
  uint64_t work_full[2], work_empty[2];
  uint64_t q_full, q_empty;
  uint64_t kv_full[kStages];
  uint64_t kv_empty[kStages];
  uint64_t v_dirty, v_clean;  // the last V tile of a padded sequence is there; is zeroed
  uint64_t s_full[2];
  uint64_t p_full[2][2];
  uint64_t o_full[2], o_empty[2];
  uint64_t stats_full[4], stats_empty[4];  // of the quadrants of a split row tile
  float2 stats[BQ];                        // maxima and sums of its second half
  uint32_t tmem_base;
};

template <int HD>
struct WindowSmem {
  static constexpr uint32_t kTile = (HD / 64) * kBoxBytes;  // one Q, K or V tile
  static constexpr uint32_t kRing = 2 * kTile;              // behind the two Q tiles
  static constexpr uint32_t kOut = kRing + kStages * 2 * kTile;  // 4 KiB a softmax warp
  static constexpr uint32_t kBars = kOut + 8 * 4096;
  static constexpr size_t kUsed = 1024 + kBars + sizeof(WindowBarriers);
  // At least 120 KiB so that a second CTA never shares the SM: each CTA
  // allocates all 512 TMEM columns.
  static constexpr size_t kBytes = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
  static_assert(kBytes <= 227 * 1024, "shared memory of a block");
};

struct WindowParams {
  CUtensorMap q, k, v;  // (d, tokens, heads, batch)
  const int32_t *lens;
  uint16_t *O;
  int64_t so[3];
  int Hq, Hkv, Nq, Nk, window, sinks;
  int items, slices;  // pairs (split: row tiles) of a slice (a sequence's K/V head); slices
  float scale_log2;
  uint64_t pair_wait_ns;  // limit of the waits that a whole pair may take
};

// Order of the grid: groups of K/V slices, the last rows (with the most keys)
// of every slice of a group first.
template <bool SPLIT>
__device__ __forceinline__ void work_of(const WindowParams &p, int item, Work &k) {
  const int per = kOrderGroup * p.items;
  const int g = item / per, first = g * kOrderGroup;
  const int gsz = min(kOrderGroup, p.slices - first);
  const int r = item - g * per;
  const int pair = p.items - 1 - r / gsz, slice = first + r % gsz;
  const int group = p.Hq / p.Hkv;
  const int shift = p.Nk - p.Nq;  // position of row 0
  const int b = slice / p.Hkv, kvh = slice - b * p.Hkv;
  const int n = p.lens ? min(max(p.lens[b], 0), p.Nk) : p.Nk;
  const int units = (p.Nq + BQ - 1) / BQ * group;
  KeyTiles kt[2];
  int count[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int unit = SPLIT ? pair : 2 * pair + w;
    const int row0 = unit / group * BQ;
    // Positions of the rows that are computed: the last one has the most keys.
    const int t_first = max(row0 + shift, 0);
    const int t_last = min(min(row0 + BQ, p.Nq) - 1 + shift, n - 1);
    kt[w] = {0, 0, 0};
    const bool exists = unit < units;
    if (exists && t_last >= t_first) {
      kt[w].hi = t_last / BKV + 1;
      if (p.window > 0) {
        kt[w].lo = max(t_first - p.window + 1, 0) / BKV;
        kt[w].sink = (int)min(((int64_t)p.sinks + BKV - 1) / BKV, (int64_t)kt[w].lo);
      }
    }
    count[w] = kt[w].count();
    k.row0[w] = row0;
    k.head[w] = kvh * group + unit % group;
    k.exists[w] = exists && !(SPLIT && w);
    k.count[w] = !SPLIT ? count[w] : w ? count[w] / 2 : (count[w] + 1) / 2;
    k.kt[w] = kt[w];
  }
  const int lo = count[0] && count[1] ? min(kt[0].lo, kt[1].lo) : count[0] ? kt[0].lo : kt[1].lo;
  const int hi = max(kt[0].hi, kt[1].hi);
  const int sink = min(max(kt[0].sink, kt[1].sink), lo);
  k.b = b;
  k.kvh = kvh;
  k.n = n;
  k.lo = lo;
  k.hi = hi;
  k.sink = sink;
  k.total = hi - lo + sink;
  // V's rows behind the end of a padded sequence are zeroed in its last tile:
  // their weights are 0, but 0 times what they hold may not be.
  k.clean = n < p.Nk && hi > 0 && hi * BKV > n;
}

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

template <int HD, bool BF16, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
flash_window_kernel(const __grid_constant__ WindowParams p) {
  using L = WindowSmem<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  WindowBarriers *bars = reinterpret_cast<WindowBarriers *>(smem + L::kBars);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars->work_full[s], 1);
      mbar_init(&bars->work_empty[s], 11);  // one per warp that reads it
    }
    mbar_init(&bars->answer_full, 1);
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->q_empty, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->kv_full[s], 1);
      mbar_init(&bars->kv_empty[s], 1);
    }
    mbar_init(&bars->v_dirty, 1);
    mbar_init(&bars->v_clean, 1);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&bars->s_full[w], 1);
      for (int h = 0; h < 2; ++h)
        mbar_init(&bars->p_full[w][h], kWgThreads / 32);  // one per warp
      mbar_init(&bars->o_full[w], 1);
      mbar_init(&bars->o_empty[w], kWgThreads / 32);
    }
    fence_barrier_init();
  }
  if (threadIdx.x == 32)
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bars->stats_full[i], 1);
      mbar_init(&bars->stats_empty[i], 1);
    }
  if (warp == 9) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  grid_dependency_wait();
  fence_proxy_async_global();  // TMA reads what the launch before wrote
  grid_launch_dependents();

  // The pairs, for every warp but the scheduler: `work` waits for pair `round`
  // (false at the end of the queue, and on an error: then the others' waits
  // run out too), `done` gives its slot back.
  int round = 0;
  auto wait_work = [&](int r) {
    return __all_sync(0xffffffffu, mbar_wait(&bars->work_full[r & 1], (r >> 1) & 1));
  };
  auto done = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->work_empty[round & 1]);
    ++round;
  };

  // 256 x 216 + 128 x 72 = 384 x 168 registers.
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // -------------------------------------------------- softmax, warps 0..7
    const int w = warp >> 2;              // which query tile
    const int quad = warp & 3;            // TMEM lane quadrant
    const int row = quad * 32 + lane;     // row within the tile == TMEM lane
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t s_col = tmem + lane_off + w * 128;
    const uint32_t o_col = tmem + lane_off + 256 + w * 128;
    const uint32_t stage = smem_u32(smem + L::kOut) + warp * 4096;
    int n_s = 0, n_o = 0;  // S tiles and O tiles so far
    int n_o1 = 0, n_split = 0;  // O tiles of the second half, exchanges of statistics
    bool ok = true;
    for (; wait_work(round) && bars->work[round & 1].valid; done()) {
      const Work &k = bars->work[round & 1];
      const KeyTiles mine = k.kt[w];
      const int count = k.count[w], row0 = k.row0[w], head = k.head[w];
      const int total = k.total, lo = k.lo, sink = k.sink, n = k.n;
      const bool both = SPLIT && total > 1;  // a split tile of which both halves have keys
      const int t_first = row0 + p.Nk - p.Nq, t = t_first + row;  // positions
      float m_run = -INFINITY;  // running max of scale_log2 * s
      float l_run = 0.0f;
      bool first = true;
      for (int u = SPLIT ? w : 0; u < total; u += 1 + SPLIT) {
        const int tile = tile_of<SPLIT>(u, total, sink, lo);
        if (!mine.has(tile)) continue;
        if (!mbar_wait(&bars->s_full[w], n_s & 1)) ok = false;
        ++n_s;
        // Warp-uniform status: the TMEM accesses below are warp-collective.
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        const int key0 = tile * BKV;
        // The whole S row in registers with one wait.
        uint32_t s[BKV / 32][32];
        tmem_ld128(s_col, *reinterpret_cast<uint32_t(*)[128]>(&s[0][0]));
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
        const bool rescale_o = rescale && !first;  // warp-uniform
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
          if ((c + 1) * 32 >= kFirstKeys) {  // a part is complete
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->p_full[w][(c + 1) * 32 > kFirstKeys]);
          }
        }
        l_run += (lsp[0] + lsp[1]) + (lsp[2] + lsp[3]);
        first = false;
        if (!ok) break;
      }
      // O / l -> 16-bit. The warp's rows of the sequence (t < n); a row without a
      // key is zero.
      const int rows_of_warp = min(p.Nq - row0, n - t_first) - quad * 32;
      uint16_t *out = p.O + k.b * p.so[0] + head * p.so[1] + (int64_t)(row0 + quad * 32) * p.so[2];
      if (count == 0) {
        if (k.exists[w] && lane < rows_of_warp && t < 0)
          for (int c = 0; c < HD / 8; ++c)
            reinterpret_cast<uint4 *>(out + lane * p.so[2])[c] = make_uint4(0, 0, 0, 0);
      } else if (both && w == 1) {
        // The other half's warps write the rows.
        ++n_o;
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars->stats_empty[quad], (n_split & 1) ^ 1));
        if (!ok) break;
        bars->stats[row] = make_float2(m_run, l_run);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->stats_full[quad]);
        ++n_split;
      } else {
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars->o_full[w], n_o & 1));
        ++n_o;
        if (!ok) break;
        float f0 = 1.0f, f1 = 1.0f;  // factors of the halves
        if (both) {
          ok = __all_sync(0xffffffffu, mbar_wait(&bars->stats_full[quad], n_split & 1) &&
                                           mbar_wait(&bars->o_full[1], n_o1 & 1));
          ++n_split;
          if (!ok) break;
          const float2 other = bars->stats[row];
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->stats_empty[quad]);
          // A side without a visible key holds zeros (or NaN, which stays).
          const float m = fmaxf(m_run, other.x);
          if (m_run != -INFINITY) f0 = ex2_approx(m_run - m);
          if (other.x != -INFINITY) f1 = ex2_approx(other.x - m);
          l_run = l_run * f0 + other.y * f1;
        }
        tc_fence_after();
        const float inv_l = l_run != 0.0f ? 1.0f / l_run : 0.0f;
        uint32_t o[HD / 32][32];
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) tmem_ld32(o_col + c * 32, o[c]);
        tmem_ld_wait();
        if (both) {
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o1[32];
            tmem_ld32(o_col + 128 + c * 32, o1);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 32; ++x)
              o[c][x] = __float_as_uint(__uint_as_float(o[c][x]) * f0 + __uint_as_float(o1[x]) * f1);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {  // the next pair's products may begin
          mbar_arrive(&bars->o_empty[w]);
          if (both) mbar_arrive(&bars->o_empty[1]);
        }
        // A thread has a row; through shared memory (16-byte chunks placed by
        // their row, so that both sides meet all banks) the warp writes 128 bytes
        // of four rows at a time (32 bytes of 32 rows at a time: 1 to 3 % slower).
#pragma unroll
        for (int half = 0; half < HD / 64; ++half) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint32_t *f = &o[half * 2 + c / 4][c % 4 * 8];
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[i] = pack2<BF16>(__uint_as_float(f[2 * i]) * inv_l, __uint_as_float(f[2 * i + 1]) * inv_l);
            sts128(stage + lane * 128 + ((c ^ (lane & 7)) << 4), make_uint4(v[0], v[1], v[2], v[3]));
          }
          __syncwarp();
          uint4 v[8];  // rows lane / 8, 4 + lane / 8, ...
          const int rr = lane >> 3, c = lane & 7;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[i] = lds128(stage + (i * 4 + rr) * 128 + ((c ^ ((i * 4 + rr) & 7)) << 4));
          uint16_t *to = out + rr * p.so[2] + half * 64 + c * 8;
#pragma unroll
          for (int i = 0; i < 8; ++i, to += 4 * p.so[2])
            if (i * 4 + rr < rows_of_warp) *reinterpret_cast<uint4 *>(to) = v[i];
          __syncwarp();  // read before it is written again
        }
      }
      n_o1 += k.count[1] > 0;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 10) {
      // ------------------------------------------------ scheduler
      if (lane == 0) {
        int x = blockIdx.x;
        int stage = 0, n_live = 0, n_clean = 0;
        bool live = false;  // the last pair had keys
        for (int r = 0;; ++r) {
          if (!mbar_wait_idle(&bars->work_empty[r & 1], ((r >> 1) & 1) ^ 1, p.pair_wait_ns)) break;
          Work &k = bars->work[r & 1];
          bool have = true;
          if (r > 0) {
            mbar_arrive_expect_tx(&bars->answer_full, 16);
            steal_cta(&bars->answer, &bars->answer_full);
            have = mbar_wait(&bars->answer_full, (r - 1) & 1) &&
                   stolen_cta(smem_u32(&bars->answer), x);
            fence_proxy_async_smem();  // read before the queue writes there again
          }
          k.valid = have;
          if (have) {
            work_of<SPLIT>(p, x, k);
            k.chained = !SPLIT && live && k.total > 0;
            live = k.total > 0;
            if (live) {
              // Its K(0) joins the last pair's last V, or begins a stage.
              k.stage0 = k.chained ? stage - 1 : stage;
              k.n_live = n_live++;
              k.n_clean = n_clean;
              n_clean += k.clean;
              stage = k.stage0 + k.total + 1 + SPLIT;
            }
          } else {
            k.chained = 0;
          }
          mbar_arrive(&bars->work_full[r & 1]);
          if (!have) break;
        }
      }
    } else if (warp == 8) {
      // ------------------------------------------------ TMA producer
      if (lane == 0) {
        tma_prefetch_desc(&p.q);
        tma_prefetch_desc(&p.k);
        tma_prefetch_desc(&p.v);
      }
      bool ok = true;
      // One stage: V of key tile tv of `kv`, K of key tile tk of `kk` (either may be absent).
      auto load_stage = [&](int s, const Work *kv, int tv, const Work *kk, int tk) {
        const int st = s % kStages;
        if (!mbar_wait(&bars->kv_empty[st], ((s / kStages) & 1) ^ 1)) return false;
        mbar_arrive_expect_tx(&bars->kv_full[st], ((kv != nullptr) + (kk != nullptr)) * L::kTile);
        uint8_t *slot = smem + L::kRing + st * 2 * L::kTile;
        if (kv) {
#pragma unroll
          for (int c = 0; c < HD / 64; ++c)
            tma_load_4d(slot + c * kBoxBytes, &p.v, c * 64, tv * BKV, kv->kvh, kv->b, &bars->kv_full[st]);
        }
        if (kk) {
#pragma unroll
          for (int c = 0; c < HD / 64; ++c)
            tma_load_4d(slot + L::kTile + c * kBoxBytes, &p.k, c * 64, tk * BKV, kk->kvh, kk->b,
                        &bars->kv_full[st]);
        }
        return true;
      };
      auto tile = [](const Work &k, int u) { return tile_of<SPLIT>(u, k.total, k.sink, k.lo); };
      for (; ok && wait_work(round) && bars->work[round & 1].valid; done()) {
        const Work &k = bars->work[round & 1], &next = bars->work[(round + 1) & 1];
        if (k.total == 0) continue;
        constexpr int ahead = 1 + SPLIT;  // steps that K is ahead of V
        if (lane == 0) {
          if (!k.chained) ok = load_stage(k.stage0, nullptr, 0, &k, tile(k, 0));
          ok = ok && mbar_wait(&bars->q_empty, (k.n_live & 1) ^ 1);
          if (ok) {
            mbar_arrive_expect_tx(&bars->q_full, ((k.count[0] > 0) + (k.count[1] > 0)) * L::kTile);
#pragma unroll
            for (int w = 0; w < 2; ++w)
              if (k.count[w] > 0) {
#pragma unroll
                for (int c = 0; c < HD / 64; ++c)
                  tma_load_4d(smem + w * L::kTile + c * kBoxBytes, &p.q, c * 64, k.row0[w], k.head[w],
                              k.b, &bars->q_full);
              }
          }
          for (int u = 1 - ahead; ok && u + 1 < k.total; ++u)
            ok = load_stage(k.stage0 + u + ahead, u >= 0 ? &k : nullptr, tile(k, u),
                            u + ahead < k.total ? &k : nullptr, tile(k, u + ahead));
        }
        ok = __shfl_sync(0xffffffffu, ok, 0) && wait_work(round + 1);
        if (ok && lane == 0) {
          const bool chain = next.valid && next.chained;
          ok = load_stage(k.stage0 + k.total - 1 + ahead, &k, tile(k, k.total - 1), chain ? &next : nullptr,
                          chain ? tile(next, 0) : 0);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
      }
      // No copy is in flight when the CTA ends: the consumers have waited for
      // every one, but for those behind an error, which get time to land.
      if (!ok && lane == 0)
        for (int i = 0; i < 2; ++i) {
          mbar_wait(&bars->q_full, i, 100000000ull);
          for (int st = 0; st < kStages; ++st) mbar_wait(&bars->kv_full[st], i, 100000000ull);
        }
    } else if (warp == 11) {
      // ------------------------------------------------ V behind a sequence's end
      auto idle_work = [&]() {
        return __all_sync(0xffffffffu, mbar_wait_idle(&bars->work_full[round & 1], (round >> 1) & 1,
                                                      p.pair_wait_ns)) &&
               bars->work[round & 1].valid;
      };
      for (bool ok = true; ok && idle_work(); done()) {
        const Work &k = bars->work[round & 1];
        if (!k.clean) continue;
        // The issuer has seen the stage arrive; it stays until the issuer goes on
        // (a stage's own barrier may be phases behind when this warp comes here).
        const int s = k.stage0 + k.total + SPLIT, st = s % kStages;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->v_dirty, k.n_clean & 1, p.pair_wait_ns) &&
                                         mbar_wait(&bars->kv_full[st], (s / kStages) & 1));
        if (!ok) break;
        // 128-byte rows of tokens in each box.
        uint8_t *v = smem + L::kRing + st * 2 * L::kTile;
        const int from = k.n - (k.hi - 1) * BKV;
        for (int i = lane; i < (BKV - from) * 8; i += 32)
#pragma unroll
          for (int c = 0; c < HD / 64; ++c)
            *reinterpret_cast<uint4 *>(v + c * kBoxBytes + from * 128 + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->v_clean);
      }
    } else {
      // ------------------------------------------------ MMA issuer, warp 9
      // The whole warp runs the loop and one elected lane issues: what comes out
      // of shared memory is broadcast, so that all of it is known to be alike in
      // every lane and descriptors stay in uniform registers.
      auto uni = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
      const uint32_t idesc_s = idesc_f16_f32(BQ, BKV, BF16, false, false);
      const uint32_t idesc_o = idesc_f16_f32(BQ, HD, BF16, false, true);
      // Descriptors are built once; a byte offset within the shared window is
      // an add of (offset >> 4) to the descriptor's address field.
      const uint64_t dq = smem_desc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t dv = smem_desc_sw128(smem_u32(smem + L::kRing), kBoxBytes, 1024);
      const uint32_t dq_lo = (uint32_t)dq, dq_hi = (uint32_t)(dq >> 32);
      const uint32_t dv_lo = (uint32_t)dv, dv_hi = (uint32_t)(dv >> 32);
      static_assert(L::kRing == 2 * L::kTile, "Q0, Q1, then stages of V, K: one descriptor serves Q and K");
      const uint32_t tm = uni(tmem);
      // A wait that runs out is noted, and ends the loop at the end of its step
      // (one vote a step, not one a wait).
      bool fine = true;
      auto wait = [&](uint64_t *bar, int parity) { fine = mbar_wait(bar, parity) && fine; };
      int n_p[2] = {0, 0}, n_o[2] = {0, 0};  // P tiles and O tiles so far
      bool ok = true;
      for (; ok && wait_work(round) && uni(bars->work[round & 1].valid); done()) {
        const Work &k = bars->work[round & 1], &next = bars->work[(round + 1) & 1];
        const int total = uni(k.total);
        if (total == 0) continue;
        KeyTiles kt[2];
        int left[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          kt[w] = {uni(k.kt[w].sink), uni(k.kt[w].lo), uni(k.kt[w].hi)};
          left[w] = uni(k.count[w]);
        }
        const int lo = uni(k.lo), sink = uni(k.sink), stage0 = uni(k.stage0);
        bool begun[2] = {false, false};
        int u = uni(k.chained) ? 0 : -1 - SPLIT;
        if (u < 0) wait(&bars->q_full, uni(k.n_live) & 1);
        // Step u in stage s = stage0 + u + 1: the products of V(u), and the scores
        // of K(u + 1), which after the last step is the next pair's first. u = -1:
        // scores only. (A split tile's steps belong to its halves in turns, and K
        // is two steps ahead: u begins at -2.)
#pragma unroll 1
        for (; ok && u < total; ++u) {
          const bool last = u + 1 == total;
          const int tile = tile_of<false>(u, total, sink, lo), after = tile_of<false>(u + 1, total, sink, lo);
          bool pv[2], sc[2];  // products and scores to issue
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            pv[w] = u >= 0 && (SPLIT ? (u & 1) == w : kt[w].has(tile));
            sc[w] = SPLIT ? (u & 1) == w && u + 2 < total : kt[w].has(after);
          }
          bool chain = false, q_free = u + 2 + SPLIT == total;
          if (last) {
            ok = wait_work(round + 1);
            if (!ok) break;
            chain = uni(next.valid && next.chained);
            q_free = chain && uni(next.total) == 1;
            const int t0 = tile_of<false>(0, next.total, next.sink, next.lo);
            sc[0] = uni(chain && next.kt[0].has(t0));
            sc[1] = uni(chain && next.kt[1].has(t0));
          }
          const int s = stage0 + u + 1 + SPLIT, st = s % kStages;
          const uint32_t v_lo = dv_lo + (2 * st * L::kTile >> 4), k_lo = dq_lo + ((3 + 2 * st) * L::kTile >> 4);
          wait(&bars->kv_full[st], (s / kStages) & 1);
          if (last && uni(k.clean)) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->v_dirty);
            __syncwarp();
            wait(&bars->v_clean, uni(k.n_clean) & 1);
          }
          tc_fence_after();
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            if (pv[w]) {
              const uint32_t o_tmem = tm + 256 + w * 128, p_tmem = tm + w * 128;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                wait(&bars->p_full[w][h], n_p[w] & 1);
                // The last pair's O has been read.
                if (h == 0 && !begun[w]) wait(&bars->o_empty[w], (n_o[w] & 1) ^ 1);
                tc_fence_after();
#pragma unroll
                for (int ks = h ? kFirstKeys / 16 : 0; ks < (h ? BKV : kFirstKeys) / 16; ++ks) {  // K = 16 MMAs
                  mma_f16_ts_lohi_warp(o_tmem, p_tmem + ks * 8, v_lo + ks * ((16 * 128) >> 4), dv_hi,
                                       idesc_o, (begun[w] || ks > 0) ? 1u : 0u);
                }
              }
              ++n_p[w];
              begun[w] = true;
              // Only the epilogue waits for O: one commit after the tile's last PV.
              if (--left[w] == 0) {
                mma_commit_warp(smem_u32(&bars->o_full[w]));
                ++n_o[w];
              }
            }
            if (w == 0 && chain) wait(&bars->q_full, uni(next.n_live) & 1);
            if (sc[w]) {
#pragma unroll
              for (int ks = 0; ks < HD / 16; ++ks) {
                const uint32_t off = (ks / 4) * (kBoxBytes >> 4) + (ks % 4) * (32 >> 4);
                mma_f16_ss_lohi_warp(tm + w * 128, dq_lo + w * (L::kTile >> 4) + off, dq_hi, k_lo + off,
                                     dq_hi, idesc_s, ks > 0 ? 1u : 0u);
              }
              mma_commit_warp(smem_u32(&bars->s_full[w]));
            }
          }
          // Behind the last S of a pair, Q's tiles come free.
          if (q_free) mma_commit_warp(smem_u32(&bars->q_empty));
          mma_commit_warp(smem_u32(&bars->kv_empty[st]));
          ok = __all_sync(0xffffffffu, fine);
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

template <int HD, bool BF16, bool SPLIT>
cudaError_t launch_typed(const WindowParams &p, int grid, cudaStream_t stream) {
  static uint64_t configured = 0;  // devices whose smem attribute is set
  static std::mutex mu;
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (dev >= 64 || !(configured & (1ull << dev))) {
      cudaError_t e = cudaFuncSetAttribute(flash_window_kernel<HD, BF16, SPLIT>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)WindowSmem<HD>::kBytes);
      if (e != cudaSuccess) return e;
      if (dev < 64) configured |= (1ull << dev);
    }
  }
  return launch_dependent(flash_window_kernel<HD, BF16, SPLIT>, dim3((unsigned)grid), kThreads,
                          (int)WindowSmem<HD>::kBytes, p, stream);
}

template <int HD, bool BF16>
cudaError_t launch_any(const WindowParams &p, int grid, bool split, cudaStream_t stream) {
  return split ? launch_typed<HD, BF16, true>(p, grid, stream) : launch_typed<HD, BF16, false>(p, grid, stream);
}

}  // namespace

cudaError_t launch_flash_window(const FlashWindowArgs &a, cudaStream_t stream) {
  const bool bf16 = a.dtype == VC_DTYPE_BF16;
  WindowParams p;
  if (!make_map(&p.q, bf16, a.Q, a.B, a.Hq, a.Nq, a.d, a.sq) ||
      !make_map(&p.k, bf16, a.K, a.B, a.Hkv, a.Nk, a.d, a.sk) ||
      !make_map(&p.v, bf16, a.V, a.B, a.Hkv, a.Nk, a.d, a.sv))
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
  p.pair_wait_ns = window_pair_wait_ns(a.Nk);
  const int64_t units = ((int64_t)a.Nq + BQ - 1) / BQ * (a.Hq / a.Hkv);
  if (units * a.B * a.Hkv > INT32_MAX / kOrderGroup) return cudaErrorInvalidValue;
  p.slices = a.B * a.Hkv;
  // Two row tiles a CTA share the loads and fill the tensor cores' gaps. While
  // every row tile can have an SM of its own, two halves of its keys do: 8 heads
  // x 512 tokens 10.6 us (with one row tile a CTA, whose steps follow one another,
  // 11.4), x 1024 14.7 (17.6), x 2048 22.9 (29.4), 2 x 8192 of d 64 57.5 (85).
  // With many more row tiles than SMs it is the other way round (32 x 2048, 512
  // tiles: 57 us split, 51 in pairs; 256: 36.1 and 34.8). In between it depends on
  // the window: 160 tiles 27.5 split, 34.4 in pairs without one, 19.1 and 17.5
  // through 512 keys; 192 32.5 and 34.3; 224 34.9 and 34.4, 23.8 and 18.9.
  const bool split = units * p.slices <= sm_count_current();
  p.items = (int)(split ? units : (units + 1) / 2);
  const int grid = p.items * p.slices;
  if (a.d == 64)
    return bf16 ? launch_any<64, true>(p, grid, split, stream) : launch_any<64, false>(p, grid, split, stream);
  return bf16 ? launch_any<128, true>(p, grid, split, stream) : launch_any<128, false>(p, grid, split, stream);
}

}  // namespace vcb

VCB_DEFINE_ERROR_ACCESSOR(flash_window_error)
