// kv8_attn.cu - attention of single tokens over the 8-bit paged K/V cache.
//
// One query token per sequence, at position lens[b] - 1:
//   O[b, h] = sum_j p_j v_j,  p = softmax_2(scale_log2 * q . k_j),
// over the keys j < lens[b] with j >= lens[b] - window or j < sinks, where
// k_j = k_scale * code of the page that holds j (v_j alike).
//
// Bound: HBM, 2 d bytes per visible key and K/V head, each read once; the
// query heads that share a K/V head are the columns of one matrix product.
//
// Split. The visible keys of every (sequence, K/V head, group of up to 8 NT
// query heads) - an item - are cut into tiles of 64 keys, and all tiles of the
// batch, in order, into equal contiguous ranges, one per block of a grid that
// fills the GPU once: ragged batches load every SM alike whatever the lengths
// are, which only the device knows. An item that lies within one block is
// written at once; one that spans blocks is joined from partial results in
// the workspace by the block that finishes last, in block order (so the
// result does not depend on which that is), over groups of blocks first when
// they are many.
//
// A warp takes 16 of a tile's 64 keys, through a ring of its own: 16-byte
// asynchronous copies of the keys' codes (rows that the mask hides are
// zero-filled and not read, so what they hold does not matter) and of the
// page's two scales; warps of a block meet only where an item ends. Per 16
// keys, with m16n8k16 fp16 products and fp32 accumulators:
//   S^T = K Q^T   A = the codes as fp16 (exact), rows keys; B = q. The order of
//                 d within the product is free, so that a thread's operands are
//                 16 contiguous bytes of a row.
//   P^T           8 x 8 transposes (movmatrix) of the fp16 weights.
//   O^T += V^T P^T   A = pairs of keys' codes interleaved by byte permutes.
// bf16 queries are scaled by a power of two per row into fp16's range (exact
// but for elements 2^-28 below the row's largest). The value scale of a page
// enters the weights: p' = 2^(s + log2 v_scale - m), m the running maximum of
// s + log2 v_scale, so that the weights stay within fp16 whatever the scales
// are, while the sum of the softmax takes 2^(s - m). The maximum follows
// lazily: it moves when a value exceeds it by more than 2^8.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <mutex>

#include "internal.h"
#include "kv8_index.h"
#include "ptx.cuh"

namespace vcb {
namespace {

constexpr int kTile = 64;      // keys per tile
constexpr int kWarps = 4;      // 16 keys each
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 3;     // ring of a warp
constexpr int kMaxHeads = 16;  // query heads of an item
constexpr float kLazy = 8.0f;  // log2 units

// Workspace: partial results, two per block (the item that its range starts
// in and the one that it ends in), then the counters, at offsets that depend
// on the device alone, so that calls of any shape share a workspace.
constexpr size_t kSlotFloats = kMaxHeads * (128 + 2);
struct Counters {
  unsigned group[2];  // of the group that starts with this block, by slot
  unsigned item;      // of the item that starts in this block
};
constexpr int blocks_per_sm(int NT) { return NT == 1 ? 3 : 2; }
int grid_blocks(int NT) { return sm_count_current() * blocks_per_sm(NT); }

struct AttnParams {
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  int64_t page_stride, scale_stride, q_stride, o_stride;
  const void *Q;
  void *O;
  const int32_t *table, *lens;
  float *slots;
  Counters *counters;
  int B, num_pages, page_shift, heads, group, groups, table_width, window, sinks;
  float scale_log2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
// Two e4m3 codes (low 16 bits of `c`, or its high ones) as fp16, exactly.
__device__ __forceinline__ uint32_t half2_lo(uint32_t c) {
  uint32_t h;
  asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(h) : "r"(c));
  return h;
}
__device__ __forceinline__ uint32_t half2_hi(uint32_t c) {
  uint32_t h;
  asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, u;\n\t}" : "=r"(h) : "r"(c));
  return h;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&h);
}

// Where a tile of the batch's list lies.
struct Cursor {
  int b, item, tile;  // item: K/V head * groups + group of query heads
  VisibleKeys vis;
  VisibleTiles tiles;
};

__device__ __forceinline__ int clamped_len(const AttnParams &p, int b) {
  const int len = p.lens[b], most = p.table_width << p.page_shift;
  return len < 0 ? 0 : len > most ? most : len;
}
__device__ __forceinline__ void set_sequence(Cursor &c, const AttnParams &p, int b) {
  c.b = b;
  c.vis = visible_keys(clamped_len(p, b), p.window, p.sinks);
  c.tiles = visible_tiles(c.vis, kTile);
}
__device__ __forceinline__ void next_item(Cursor &c, const AttnParams &p) {
  c.tile = 0;
  if (++c.item < p.heads * p.groups) return;
  c.item = 0;
  // A sequence with tiles follows wherever the caller has tiles left (the
  // bound holds the walk within `lens` even if that changes underneath).
  c.tiles.count = 0;
  while (c.tiles.count == 0 && c.b + 1 < p.B) set_sequence(c, p, c.b + 1);
}

template <int D>
struct Smem {
  static constexpr int kStageBytes = 2 * 16 * D + 16;  // K rows, V rows, scales, mask
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kRow = D + 4;  // floats of a head's row in the merge
  template <int NT>
  static constexpr int bytes() {
    return kRing + kWarps * 8 * NT * (kRow + 2) * 4;
  }
};

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(NT)) kv8_attn_kernel(const AttnParams p) {
  using S = Smem<D>;
  constexpr int NH = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int sh_scan[kWarps], sh_found[2];
  __shared__ unsigned sh_last;
  float *merge_o = reinterpret_cast<float *>(smem + S::kRing);    // [warp][NH][kRow]
  float *merge_m = merge_o + kWarps * NH * S::kRow;               // [warp][NH]
  float *merge_l = merge_m + kWarps * NH;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = lane >> 2, t = lane & 3;
  const int items = p.heads * p.groups;

  // ---- this block's range of tiles
  auto tiles_of = [&](int b) {
    return visible_tiles(visible_keys(clamped_len(p, b), p.window, p.sinks), kTile).count;
  };
  auto block_scan = [&](int x, int &before) {  // inclusive sum over the block, and its total
    int s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    __syncthreads();
    if (lane == 31) sh_scan[warp] = s;
    __syncthreads();
    int total = 0, mine = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) mine += sh_scan[w];
      total += sh_scan[w];
    }
    before = mine + s - x;
    return total;
  };
  const int mine = tid < p.B ? tiles_of(tid) : 0;
  int seq_tiles = mine, before;
  for (int b = tid + kThreads; b < p.B; b += kThreads) seq_tiles += tiles_of(b);
  const int all = block_scan(seq_tiles, before);
  const int64_t total = (int64_t)all * items;
  const int blocks = (int)(total < gridDim.x ? total : gridDim.x);

  // Sequences without a token: zero rows.
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    const int len = p.lens[b];
    if (tid == 0 && (len < 0 || len > p.table_width << p.page_shift)) record_error(kErrOutOfBounds);
    if (len > 0) continue;
    uint4 *row = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.O) + b * p.o_stride);
    for (int i = tid; i < p.heads * p.group * D / 8; i += kThreads) row[i] = make_uint4(0, 0, 0, 0);
  }
  if ((int)blockIdx.x >= blocks) return;
  const int64_t t0 = split_start(total, blocks, blockIdx.x);
  const int64_t t1 = split_start(total, blocks, blockIdx.x + 1);
  if (tid == 0) sh_found[0] = -1;
  __syncthreads();
  auto found = [&](int b, int n, int64_t first) {
    if (t0 < first || t0 >= first + (int64_t)n * items) return;
    sh_found[0] = b;
    sh_found[1] = (int)(t0 - first);
  };
  if (p.B <= kThreads) {
    found(tid, mine, (int64_t)before * items);
  } else {
    int64_t base = 0;  // tiles before the chunk of sequences, times items
    for (int b0 = 0; b0 < p.B && base <= t0; b0 += kThreads) {
      const int n = b0 + tid < p.B ? tiles_of(b0 + tid) : 0;
      const int chunk = block_scan(n, before);
      found(b0 + tid, n, base + (int64_t)before * items);
      base += (int64_t)chunk * items;
    }
  }
  __syncthreads();
  if (sh_found[0] < 0) return;
  Cursor cur;
  set_sequence(cur, p, sh_found[0]);
  cur.item = sh_found[1] / cur.tiles.count;
  cur.tile = sh_found[1] % cur.tiles.count;

  // ---- the warp's ring
  uint8_t *ring = smem + warp * kStages * S::kStageBytes;
  Cursor pre = cur;
  int64_t pre_t = t0;
  auto first_key = [&](const Cursor &c) { return tile_key(c.tiles, c.tile, kTile) + warp * 16; };
  auto any_visible = [&](const Cursor &c, int k0) {
    return k0 < c.vis.len && (k0 + 15 >= c.vis.lo || k0 < c.vis.sink);
  };
  // Pages of 32 tiles of the item from `pages_at` on, one per lane.
  int pages = -1, pages_at = 0;
  auto look_up = [&]() {
    pages_at = pre.tile;
    const int i = pre.tile + lane;
    if (i >= pre.tiles.count) return;
    const int k0 = tile_key(pre.tiles, i, kTile) + warp * 16;
    if (any_visible(pre, k0)) pages = __ldg(p.table + (int64_t)pre.b * p.table_width + (k0 >> p.page_shift));
  };
  auto issue = [&](int stage) {
    if (pre_t < t1) {
      uint8_t *at = ring + stage * S::kStageBytes;
      const int k0 = first_key(pre);
      uint32_t mask = 0;
      if (any_visible(pre, k0)) {
        const int page = __shfl_sync(0xffffffffu, pages, pre.tile - pages_at);
        const bool bad = page < 0 || page >= p.num_pages;
        if (bad && lane == 0) record_error(kErrOutOfBounds);
        mask = __ballot_sync(0xffffffffu, !bad && lane < 16 && key_visible(pre.vis, k0 + lane));
        if (!bad) {
          const int head = pre.item / p.groups;
          const int64_t off = page * p.page_stride +
                              (((int64_t)head << p.page_shift) + (k0 & ((1 << p.page_shift) - 1))) * D;
          constexpr int kChunks = D / 16;  // of a row
#pragma unroll
          for (int i = 0; i < kChunks / 2; ++i) {
            const int row = (i * 32 + lane) / kChunks, ch = lane % kChunks;
            const uint32_t bytes = mask >> row & 1 ? 16 : 0;
            const int64_t src = off + row * D + ch * 16;
            const int swk = D == 128 ? (row & 1) << 2 : 0;
            const int swv = D == 128 ? ((row >> 1) & 3) << 1 : (row >> 1) & 3;
            cp_async16(smem_u32(at + row * D + (ch ^ swk) * 16), p.k + src, bytes);
            cp_async16(smem_u32(at + 16 * D + row * D + (ch ^ swv) * 16), p.v + src, bytes);
          }
          if (lane < 2)
            cp_async4(smem_u32(at + 32 * D + lane * 4),
                      (lane ? p.v_scale : p.k_scale) + page * p.scale_stride + head, 4);
        }
      }
      if (lane == 0) *reinterpret_cast<uint32_t *>(at + 32 * D + 8) = mask;
      ++pre_t;
      const bool turn = ++pre.tile == pre.tiles.count;
      if (turn && pre_t < t1) next_item(pre, p);
      if (turn || pre.tile - pages_at == 32) look_up();
    }
    cp_async_commit();
  };
  look_up();
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(s);

  int stage = 0;
  for (int64_t at_tile = t0; at_tile < t1;) {
    // ---- one item: its queries
    const int head = cur.item / p.groups, grp = cur.item % p.groups;
    const int h0 = head * p.group + grp * NH;  // first query head
    const int nh = min(NH, p.group - grp * NH);
    uint32_t q[NT][D / 16][2];
    float mult[NT][2];  // of the scores of this thread's two columns
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool have = nt * 8 + r < nh;
      const uint16_t *src = static_cast<const uint16_t *>(p.Q) + cur.b * p.q_stride +
                            (int64_t)(h0 + nt * 8 + (have ? r : 0)) * D + t * 16;
      float inv = 1.0f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ks += 2) {
        const uint4 w = have ? *reinterpret_cast<const uint4 *>(src + (ks / 4) * 64 + (ks % 4) * 4)
                             : make_uint4(0, 0, 0, 0);
        q[nt][ks][0] = w.x;
        q[nt][ks][1] = w.y;
        q[nt][ks + 1][0] = w.z;
        q[nt][ks + 1][1] = w.w;
      }
      if constexpr (BF16) {
        uint32_t top = 0;  // largest magnitude's bits
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            top = max(top, q[nt][ks][j] & 0x7FFFu);
            top = max(top, q[nt][ks][j] >> 16 & 0x7FFFu);
          }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^e brings the largest to [2^14, 2^15); inf and NaN stay what they are.
        int e = 14 + 127 - (int)(top >> 7);
        e = top == 0 || top >= 0x7F80u ? 0 : e > 120 ? 120 : e;
        const float mul = __uint_as_float((uint32_t)(e + 127) << 23);
        inv = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            q[nt][ks][j] = pack_half2(__uint_as_float(q[nt][ks][j] << 16) * mul,
                                      __uint_as_float(q[nt][ks][j] & 0xFFFF0000u) * mul);
      }
      mult[nt][0] = __shfl_sync(0xffffffffu, inv, t * 8) * p.scale_log2;
      mult[nt][1] = __shfl_sync(0xffffffffu, inv, t * 8 + 4) * p.scale_log2;
    }
    float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
    }

    // ---- its tiles
    const int64_t left = t1 - at_tile;
    const int n = (int)(left < cur.tiles.count - cur.tile ? left : cur.tiles.count - cur.tile);
    if (n <= 0) break;
    for (int i = 0; i < n; ++i) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      issue(stage == 0 ? kStages - 1 : stage - 1);
      const uint32_t at = smem_u32(ring + stage * S::kStageBytes);
      stage = stage + 1 == kStages ? 0 : stage + 1;
      const uint4 meta = lds128(at + 32 * D);
      const uint32_t mask = meta.z;
      if (mask == 0) continue;  // uniform over the warp
      const float ks = __uint_as_float(meta.x), vs = __uint_as_float(meta.y);

      float s[NT][4], s2[NT][4];  // even and odd steps of d: two shorter chains of products
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[nt][x] = s2[nt][x] = 0.0f;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const int sw = D == 128 ? (r & 1) << 2 : 0;  // rows r and r + 8 alike
        const uint4 lo = lds128(at + r * D + ((4 * c + t) ^ sw) * 16);
        const uint4 hi = lds128(at + (r + 8) * D + ((4 * c + t) ^ sw) * 16);
        const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a0 = half2_lo(wl[j]), a1 = half2_lo(wh[j]), a2 = half2_hi(wl[j]),
                         a3 = half2_hi(wh[j]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816(j & 1 ? s2[nt] : s[nt], a0, a1, a2, a3, q[nt][4 * c + j][0], q[nt][4 * c + j][1]);
        }
      }
      // Scores in log2 units; hidden keys -inf.
      const bool on0 = mask >> r & 1, on1 = mask >> (r + 8) & 1;
      // log2 of the value scale: for the maximum kept from minus infinity, for
      // the weights not (a zero scale takes its values out).
      const float lv = vs > 0.0f ? fmaxf(lg2_approx(vs), -110.0f) : -110.0f;
      const float lvp = vs > 0.0f ? lv : -INFINITY;
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          s[nt][x] = on0 ? (s[nt][x] + s2[nt][x]) * (mult[nt][x] * ks) : -INFINITY;
          s[nt][2 + x] = on1 ? (s[nt][2 + x] + s2[nt][2 + x]) * (mult[nt][x] * ks) : -INFINITY;
          grow |= fmaxf(s[nt][x], s[nt][2 + x]) + lv > m[nt][x] + kLazy;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float mx = fmaxf(s[nt][x], s[nt][2 + x]) + lv;
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mx = fmaxf(mx, m[nt][x]);
            const float alpha = mx == -INFINITY ? 1.0f : ex2_approx(m[nt][x] - mx);
            m[nt][x] = mx;
            l[nt][x] *= alpha;
#pragma unroll
            for (int i2 = 0; i2 < D / 16; ++i2) {
              o[nt][i2][x] *= alpha;
              o[nt][i2][2 + x] *= alpha;
            }
          }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float mm = m[nt][x] == -INFINITY ? 0.0f : m[nt][x];
          w[x] = ex2_approx(s[nt][x] + (lvp - mm));
          w[2 + x] = ex2_approx(s[nt][2 + x] + (lvp - mm));
          l[nt][x] += ex2_approx(s[nt][x] - mm) + ex2_approx(s[nt][2 + x] - mm);
        }
        pb[nt][0] = transpose8x8(pack_half2(w[0], w[1]));
        pb[nt][1] = transpose8x8(pack_half2(w[2], w[3]));
      }
      // Values: this thread's keys 2t, 2t + 1, 2t + 8, 2t + 9, D / 8 codes from d = r D / 8 on.
      uint32_t v[4][D / 32];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int key = 2 * t + (k & 1) + (k >> 1) * 8;
        if constexpr (D == 128) {
          const uint4 w = lds128(at + 16 * D + key * D + ((r ^ (t << 1)) * 16));
          v[k][0] = w.x;
          v[k][1] = w.y;
          v[k][2] = w.z;
          v[k][3] = w.w;
        } else {
          const uint2 w = lds64(at + 16 * D + key * D + ((r >> 1) ^ t) * 16 + (r & 1) * 8);
          v[k][0] = w.x;
          v[k][1] = w.y;
        }
      }
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t sel = half ? 0x7362 : 0x5140;
          const uint32_t ab = __byte_perm(v[0][j], v[1][j], sel), cd = __byte_perm(v[2][j], v[3][j], sel);
          const uint32_t a0 = half2_lo(ab), a1 = half2_hi(ab), a2 = half2_lo(cd), a3 = half2_hi(cd);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816(o[nt][2 * j + half], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
        }
    }

    // ---- the warps' results joined
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float sum = l[nt][x];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int col = nt * 8 + 2 * t + x;
        if (r == 0) {
          merge_m[warp * NH + col] = m[nt][x];
          merge_l[warp * NH + col] = sum;
        }
        // d = r D / 8 + 2 i, + 1 of fragment i.
        float *to = merge_o + (warp * NH + col) * S::kRow + r * (D / 8);
#pragma unroll
        for (int i = 0; i < D / 16; i += 2)
          *reinterpret_cast<float4 *>(to + 2 * i) =
              make_float4(o[nt][i][x], o[nt][i][2 + x], o[nt][i + 1][x], o[nt][i + 1][2 + x]);
      }
    __syncthreads();
    const int64_t item0 = at_tile - cur.tile, item1 = item0 + cur.tiles.count;
    const bool whole = item0 >= t0 && item1 <= t1;
    const int slot_of_mine = item0 <= t0 ? 0 : 1;
    // A thread holds d = 4 x .. 4 x + 3 of one head at a time.
    auto write_out = [&](int h, int d, const float4 &v, float sum) {
      if (h >= nh) return;
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
      uint2 w;
      if constexpr (BF16) {
        __nv_bfloat162 a = __floats2bfloat162_rn(v.x * inv, v.y * inv), b = __floats2bfloat162_rn(v.z * inv, v.w * inv);
        w = make_uint2(*reinterpret_cast<uint32_t *>(&a), *reinterpret_cast<uint32_t *>(&b));
      } else {
        w = make_uint2(pack_half2(v.x * inv, v.y * inv), pack_half2(v.z * inv, v.w * inv));
      }
      *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.O) + cur.b * p.o_stride + (int64_t)(h0 + h) * D + d) = w;
    };
    float *const my_slot = p.slots + ((size_t)blockIdx.x * 2 + slot_of_mine) * kSlotFloats;
    for (int e = tid; e < NH * D / 4; e += kThreads) {
      const int h = e / (D / 4), d = e % (D / 4) * 4;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, merge_m[w * NH + h]);
      float sum = 0.0f;
      float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = merge_m[w * NH + h];
        const float f = mw == -INFINITY ? 0.0f : ex2_approx(mw - mm);
        const float4 x = *reinterpret_cast<const float4 *>(merge_o + (w * NH + h) * S::kRow + d);
        // A warp without a visible key has nothing to add (0, not 0 * NaN: its sum is 0 too).
        acc.x += f * x.x;
        acc.y += f * x.y;
        acc.z += f * x.z;
        acc.w += f * x.w;
        sum += mw == -INFINITY ? merge_l[w * NH + h] : f * merge_l[w * NH + h];
      }
      if (whole) {
        write_out(h, d, acc, sum);
      } else {
        __stcg(reinterpret_cast<float4 *>(my_slot + h * D + d), acc);
        if (d == 0) {
          __stcg(my_slot + NH * D + 2 * h, mm);
          __stcg(my_slot + NH * D + 2 * h + 1, sum);
        }
      }
    }
    if (!whole) {
      // ---- blocks first .. last hold parts of this item
      const int first = split_owner(total, blocks, item0), last = split_owner(total, blocks, item1 - 1);
      const int parts = last - first + 1;
      // Up to 8 parts are joined at once; more in groups of about their root.
      int size = parts;
      if (parts > 8)
        for (size = 3; size * size < parts;) ++size;
      const int groups = (parts + size - 1) / size;
      // A part's slot: 1 where the item starts within the block's range.
      const int first_slot = split_start(total, blocks, first) < item0 ? 1 : 0;
      auto slot_of = [&](int part) { return (size_t)(first + part) * 2 + (part ? 0 : first_slot); };
      // Joins the n parts a, a + step, ... into the output, or into part a's slot.
      auto join = [&](int a, int n, int step, bool to_out) {
        __threadfence();
        float *w = merge_o;  // [n][NH] weights, then [NH] sums
        for (int e = tid; e < n * NH; e += kThreads) {
          const float *from = p.slots + slot_of(a + e / NH * step) * kSlotFloats + NH * D;
          w[e] = __ldcg(from + 2 * (e % NH));
          w[(n + 1) * NH + e] = __ldcg(from + 2 * (e % NH) + 1);
        }
        __syncthreads();
        if (tid < NH) {
          float mm = -INFINITY, sum = 0.0f;
          for (int i = 0; i < n; ++i) mm = fmaxf(mm, w[i * NH + tid]);
          for (int i = 0; i < n; ++i) {
            const float mi = w[i * NH + tid];
            // Of a part without a visible key: 0 and 0, or NaN.
            const float f = mi == -INFINITY ? 1.0f : ex2_approx(mi - mm);
            w[i * NH + tid] = f;
            sum += f * w[(n + 1 + i) * NH + tid];
          }
          w[n * NH + tid] = sum;
          merge_m[tid] = mm;
        }
        __syncthreads();
        constexpr int kVecs = NH * D / 4 / kThreads;
        float4 acc[kVecs];
#pragma unroll
        for (int x = 0; x < kVecs; ++x) acc[x] = make_float4(0, 0, 0, 0);
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
          const float *from = p.slots + slot_of(a + i * step) * kSlotFloats;
#pragma unroll
          for (int x = 0; x < kVecs; ++x) {
            const int e = tid + x * kThreads;
            const float f = w[i * NH + e / (D / 4)];
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(from) + e);
            acc[x] = make_float4(acc[x].x + f * v.x, acc[x].y + f * v.y, acc[x].z + f * v.z,
                                 acc[x].w + f * v.w);
          }
        }
        if (!to_out) __syncthreads();  // every thread has read part a's slot
        float *to = p.slots + slot_of(a) * kSlotFloats;
#pragma unroll
        for (int x = 0; x < kVecs; ++x) {
          const int e = tid + x * kThreads, h = e / (D / 4);
          if (to_out)
            write_out(h, e % (D / 4) * 4, acc[x], w[n * NH + h]);
          else
            __stcg(reinterpret_cast<float4 *>(to) + e, acc[x]);
        }
        if (!to_out && tid < NH) {
          __stcg(to + NH * D + 2 * tid, merge_m[tid]);
          __stcg(to + NH * D + 2 * tid + 1, w[n * NH + tid]);
        }
      };
      // Counts this block in; true for the one that completes `of`.
      auto arrive = [&](unsigned *counter, int of) {
        __threadfence();
        __syncthreads();
        if (tid == 0) {
          const unsigned before2 = atomicAdd(counter, 1u);
          sh_last = before2 + 1 == (unsigned)of;
          if (sh_last) *counter = 0;  // ready for the next call
        }
        __syncthreads();
        return sh_last != 0;
      };
      const int part = (int)blockIdx.x - first, g = part / size;
      const int ga = g * size, gb = min(ga + size, parts);
      const size_t lead = slot_of(ga);
      if (arrive(&p.counters[lead >> 1].group[lead & 1], gb - ga)) {
        join(ga, gb - ga, 1, groups == 1);
        if (groups > 1 && arrive(&p.counters[first].item, groups)) join(0, groups, size, true);
      }
    }
    __syncthreads();  // the merge buffer is free again
    at_tile += n;
    cur.tile += n;
    if (at_tile < t1) next_item(cur, p);
  }
  cp_async_wait<0>();
}

template <int D, int NT, bool BF16>
cudaError_t launch_typed(const AttnParams &p, cudaStream_t stream) {
  constexpr int bytes = Smem<D>::template bytes<NT>();
  static uint64_t configured = 0;  // devices whose smem attribute is set
  static std::mutex mu;
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (dev >= 64 || !(configured & (1ull << dev))) {
      cudaError_t e = cudaFuncSetAttribute(kv8_attn_kernel<D, NT, BF16>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      if (e != cudaSuccess) return e;
      if (dev < 64) configured |= (1ull << dev);
    }
  }
  kv8_attn_kernel<D, NT, BF16><<<grid_blocks(NT), kThreads, bytes, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

size_t kv8_attn_workspace_bytes(const vc_kv8_cache &, int, int) {
  const size_t blocks = grid_blocks(1);
  return blocks * (2 * kSlotFloats * sizeof(float) + sizeof(Counters));
}

cudaError_t launch_kv8_attn(const Kv8AttnArgs &a, cudaStream_t stream) {
  const vc_kv8_cache &c = *a.cache;
  const int group = a.Hq / c.heads;
  const int NT = group <= 8 ? 1 : 2;
  const int groups = (group + 8 * NT - 1) / (8 * NT);
  int shift = 4;
  while (1 << shift < c.page_size) ++shift;
  // Tiles are counted in 32 bits.
  const int64_t tiles = (((int64_t)a.table_width << shift) + kTile - 1) / kTile + 1;
  if (tiles * a.B > INT32_MAX || tiles * c.heads * groups > INT32_MAX) return cudaErrorInvalidValue;
  float *slots = static_cast<float *>(a.workspace);
  const AttnParams p{static_cast<const uint8_t *>(c.k), static_cast<const uint8_t *>(c.v),
                     c.k_scale, c.v_scale, c.page_stride, c.scale_stride, a.q_stride, a.o_stride,
                     a.Q, a.O, a.table, a.lens, slots,
                     reinterpret_cast<Counters *>(slots + (size_t)grid_blocks(1) * 2 * kSlotFloats),
                     a.B, c.num_pages, shift, c.heads, group, groups, a.table_width, a.window,
                     a.sinks, a.scale_log2};
  const bool bf16 = a.dtype == VC_DTYPE_BF16;
  if (c.head_dim == 64) {
    if (NT == 1) return bf16 ? launch_typed<64, 1, true>(p, stream) : launch_typed<64, 1, false>(p, stream);
    return bf16 ? launch_typed<64, 2, true>(p, stream) : launch_typed<64, 2, false>(p, stream);
  }
  if (NT == 1) return bf16 ? launch_typed<128, 1, true>(p, stream) : launch_typed<128, 1, false>(p, stream);
  return bf16 ? launch_typed<128, 2, true>(p, stream) : launch_typed<128, 2, false>(p, stream);
}

}  // namespace vcb

VCB_DEFINE_ERROR_ACCESSOR(kv8_attn_error)
