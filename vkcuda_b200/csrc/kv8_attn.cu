// kv8_attn.cu - attention of single tokens over the 8-bit paged K/V cache.
//
// One query token per sequence, at position lens[b] - 1:
//   O[b, h] = sum_j p_j v_j,  p = softmax_2(scale_log2 * q . k_j),
// over the keys j < lens[b] with j >= lens[b] - window or j < sinks, where
// k_j = k_scale * code of the page that holds j (v_j alike).
//
// Bound: HBM, 2 d bytes per visible key and K/V head, each read once; the
// query heads that share a K/V head are the columns of one matrix product.
// Measured (head dim 128, 8 K/V heads of 4 query heads): 32 sequences of up to
// 16384 tokens 104 us, 5.9 TB/s, 0.90 of the copy rate; 64 of up to 16384
// (4 K/V heads) through a window of 4096 52 us, 5.0 TB/s. Of a call's time about
// 9 us do not shrink with the work: lengths, page numbers, scales and the first
// codes come one after the other (5 us), and at the end the warps' and the
// blocks' results are joined (4 us).
//
// Split. The visible keys of every (sequence, K/V head, group of up to 8 NT
// query heads) - an item - are cut into tiles of 128 keys, and all tiles of the
// batch, in order, into equal contiguous ranges, one per block of a grid that
// fills the GPU once: ragged batches load every SM alike whatever the lengths
// are, which only the device knows. An item that lies within one block is
// written at once; one that spans blocks is joined from partial results in
// the workspace by the block that finishes last, in block order (so the
// result does not depend on which that is).
//
// A warp takes 32 of a tile's 128 keys, through a ring of its own that TMA
// fills: boxes of 16 or 32 rows of the page's codes, swizzled so that the
// reads below meet no bank twice. Warps of a block meet only where an item
// ends: there each joins a quarter of the results, while the next item's queries
// are on their way (two warps, then one, and the queries after that: 256 sequences
// of up to 500 tokens took 63.6 us instead of 55.0; that is 57 on another GPU, and
// 59 with the sum's own maximum). Rows that the mask hides arrive too; their scores
// become minus infinity and their values zero, whatever they hold. Per 16 keys, with
// m16n8k16 fp16 products and fp32 accumulators:
//   S^T = K Q^T   A = the codes as fp16 (exact), rows keys; B = q. The order of
//                 d within the product is free, so that a thread's operands are
//                 16 contiguous bytes of a row; so is the order of the keys.
//   P^T           8 x 8 transposes (movmatrix) of the fp16 weights.
//   O^T += V^T P^T   A = pairs of keys' codes interleaved by byte permutes.
// bf16 queries are scaled by a power of two per row into fp16's range (exact
// but for elements 2^-28 below the row's largest). The value scale of a page
// enters the weights: p' = 2^(s + log2 v_scale - m), m the running maximum of
// s + log2 v_scale, so that the weights stay within fp16 whatever the scales
// are. What a weight below 2^-25 of the largest would add, less than 2^-16 of a
// unit of the codes that have the largest, is left out (their half step is 2^-10
// at least). The sum of the softmax has a maximum of its own, that of s: relative
// to m its terms would lie between 2^-119 and 2^110, and the factor between two
// such sums is not an fp32 number. Both maxima follow lazily: they move when a
// value exceeds its own by more than 2^8. Where the warps' results are joined,
// products and sums come to one reference, see there.
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

constexpr int kTile = 128;     // keys per tile
constexpr int kWarps = 4;      // 32 keys each
constexpr int kThreads = kWarps * 32;
// Two blocks with 16 KB of ring per warp: 32 sequences of up to 16384 tokens
// 105 us, one of 32000 17.6 us, 64 of up to 700 25.4 us (104, 19 and 23 to 25 since).
// Three: 109, 20.6 (more parts to join) and 23.3 us; one block of 8 warps: 109,
// 14.5 and 31.8 us.
constexpr int kBlocksPerSm = 2;
constexpr int kMaxHeads = 16;  // query heads of an item
constexpr float kLazy = 8.0f;  // log2 units
constexpr float kLargest = 3.402823466e38f;  // of fp32

// Workspace: partial results, two per block (the item that its range starts
// in and the one that it ends in), then the counters, at offsets that depend
// on the device alone, so that calls of any shape share a workspace.
constexpr size_t kSlotFloats = kMaxHeads * (128 + 2);
struct Counters {
  unsigned group[2];  // of the group that starts with this block, by slot
  unsigned item;      // of the item that starts in this block
};
int grid_blocks() { return sm_count_current() * kBlocksPerSm; }

struct AttnParams {
  CUtensorMap k, v;  // (d, heads * page_size, pages)
  const float *k_scale, *v_scale;
  int64_t scale_stride, q_stride, o_stride;
  const void *Q;
  void *O;
  const int32_t *table, *lens;
  float *slots;
  Counters *counters;
  int B, num_pages, page_shift, heads, group, groups, table_width, window, sinks;
  float scale_log2;
};

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

template <int D, int NT>
struct Smem {
  static constexpr int kHalf = 16 * D;       // 16 keys' codes of K or V
  static constexpr int kStage = 4 * kHalf;   // K, K, V, V
  static constexpr int kStages = 16384 / kStage;  // ring of a warp
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kMetas = kRing;       // of every stage
  static constexpr int kBars = kMetas + kWarps * kStages * 32;
  static constexpr int kMerge = kBars + ((kWarps * kStages * 8 + 15) & ~15);
  static constexpr int kMergeWarp = 32 * (D * NT / 4 + 6 * NT);  // floats a warp hands over
  static constexpr int kBytes = kMerge + kWarps * kMergeWarp * 4 + 1024;  // the ring 1024-byte aligned
};
struct alignas(16) Meta {
  float k_scale[2], v_scale[2];  // of the halves
  uint32_t mask;                 // visible keys
};
static_assert(sizeof(Meta) == 32, "two 16-byte words a stage");

// Fragment i of a thread of the O^T product: d = r D / 8 + 2 i and + 1, columns
// (query heads) 2t and 2t + 1 of nt (x, z: the first column; y, w: the second),
// divided by the columns' sums into the output rows (of nh heads from `out` on).
template <int D, bool BF16>
__device__ __forceinline__ void write_fragment(uint16_t *out, int nh, int lane, int nt, int i,
                                               const float4 &v, float sum0, float sum1) {
  const int r = lane >> 2, t = lane & 3;
  uint16_t *row = out + (nt * 8 + 2 * t) * D + r * (D / 8) + 2 * i;
  // No visible key: zeros.
  const float i0 = sum0 != 0.0f ? 1.0f / sum0 : 0.0f, i1 = sum1 != 0.0f ? 1.0f / sum1 : 0.0f;
  uint32_t a, c;
  if constexpr (BF16) {
    __nv_bfloat162 x = __floats2bfloat162_rn(v.x * i0, v.z * i0), y = __floats2bfloat162_rn(v.y * i1, v.w * i1);
    a = *reinterpret_cast<uint32_t *>(&x);
    c = *reinterpret_cast<uint32_t *>(&y);
  } else {
    a = pack_half2(v.x * i0, v.z * i0);
    c = pack_half2(v.y * i1, v.w * i1);
  }
  if (nt * 8 + 2 * t < nh) *reinterpret_cast<uint32_t *>(row) = a;
  if (nt * 8 + 2 * t + 1 < nh) *reinterpret_cast<uint32_t *>(row + D) = c;
}

// Slot of part i of an item whose part 0 lies in block `first`: every later
// part begins its block's range (slot 0).
__device__ __forceinline__ size_t part_slot(int first, int first_slot, int i) {
  return (size_t)(first + i) * 2 + (i ? 0 : first_slot);
}

// Factor that takes what is relative to the maximum `from` to `to`. A side without a
// visible key holds zeros (or NaN, which stays).
__device__ __forceinline__ float rescale(float from, float to) {
  return from == -INFINITY ? 1.0f : ex2_approx(from - to);
}

// Joins the n parts a, a + step, ... of an item into the output rows, or (out
// null) into part a's slot; the loads of 4 parts are in flight while 4 are added. Not inlined: its
// registers are not the main loop's.
template <int D, int NT, bool BF16>
__device__ __noinline__ void join_parts(float *slots, int first, int first_slot, int a, int n,
                                        int step, uint16_t *out, int nh) {
  constexpr int kFrags = D / 16 * NT, kVecs = kFrags * 32 / kThreads;
  constexpr int kBatch = 4;
  const int tid = threadIdx.x, lane = tid & 31, t = lane & 3;
  float4 acc[kVecs];
  float mx[NT][2], sum[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    mx[nt][0] = mx[nt][1] = -INFINITY;
    sum[nt][0] = sum[nt][1] = 0.0f;
  }
#pragma unroll
  for (int x = 0; x < kVecs; ++x) acc[x] = make_float4(0, 0, 0, 0);
  float4 v[kBatch][kVecs], ml[kBatch][NT], v2[kBatch][kVecs], ml2[kBatch][NT];
  auto load = [&](int i0, float4 (&v)[kBatch][kVecs], float4 (&ml)[kBatch][NT]) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      // Behind the last part: that one again, with weight 0.
      const int part = a + min(i0 + i, n - 1) * step;
      const float4 *from = reinterpret_cast<const float4 *>(slots + part_slot(first, first_slot, part) * kSlotFloats);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) ml[i][nt] = __ldcg(from + kFrags * 32 + nt * 4 + t);
#pragma unroll
      for (int x = 0; x < kVecs; ++x) v[i][x] = __ldcg(from + tid + x * kThreads);
    }
  };
  load(0, v, ml);
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += kBatch) {
    if (i0 + kBatch < n) load(i0 + kBatch, v2, ml2);  // while this batch is added up
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float old0 = mx[nt][0], old1 = mx[nt][1];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        mx[nt][0] = fmaxf(mx[nt][0], ml[i][nt].x);
        mx[nt][1] = fmaxf(mx[nt][1], ml[i][nt].z);
      }
      // A side without a visible key holds zeros (or NaN, which stays).
      const float g0 = old0 == -INFINITY ? 1.0f : ex2_approx(old0 - mx[nt][0]);
      const float g1 = old1 == -INFINITY ? 1.0f : ex2_approx(old1 - mx[nt][1]);
      sum[nt][0] *= g0;
      sum[nt][1] *= g1;
#pragma unroll
      for (int x = 0; x < kVecs; ++x)
        if (x * kThreads / (D / 16 * 32) == nt)
          acc[x] = make_float4(acc[x].x * g0, acc[x].y * g1, acc[x].z * g0, acc[x].w * g1);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (i0 + i >= n) break;
        const float f0 = ml[i][nt].x == -INFINITY ? 1.0f : ex2_approx(ml[i][nt].x - mx[nt][0]);
        const float f1 = ml[i][nt].z == -INFINITY ? 1.0f : ex2_approx(ml[i][nt].z - mx[nt][1]);
        sum[nt][0] += f0 * ml[i][nt].y;
        sum[nt][1] += f1 * ml[i][nt].w;
#pragma unroll
        for (int x = 0; x < kVecs; ++x)
          if (x * kThreads / (D / 16 * 32) == nt)
            acc[x] = make_float4(acc[x].x + f0 * v[i][x].x, acc[x].y + f1 * v[i][x].y,
                                 acc[x].z + f0 * v[i][x].z, acc[x].w + f1 * v[i][x].w);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) ml[i][nt] = ml2[i][nt];
#pragma unroll
      for (int x = 0; x < kVecs; ++x) v[i][x] = v2[i][x];
    }
  }
  if (!out) __syncthreads();  // every thread has read part a's slot
  float4 *to = reinterpret_cast<float4 *>(slots + part_slot(first, first_slot, a) * kSlotFloats);
#pragma unroll
  for (int x = 0; x < kVecs; ++x) {
    const int e = tid + x * kThreads, nt = x * kThreads / (D / 16 * 32);
    if (out)
      write_fragment<D, BF16>(out, nh, lane, nt, e / 32 % (D / 16), acc[x], sum[nt][0], sum[nt][1]);
    else
      __stcg(to + e, acc[x]);
  }
  if (!out && tid < 4) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      __stcg(to + kFrags * 32 + nt * 4 + t, make_float4(mx[nt][0], sum[nt][0], mx[nt][1], sum[nt][1]));
  }
}

// How the parts of an item are joined: blocks first, first + 1, ... hold them,
// part 0 in slot 1 of its block where the item starts within the block's range.
// Up to 16 parts are joined at once; more in groups of about their root, each by
// the block of the group that arrives last, and the groups' results by the last
// of those.
struct Join {
  int first, first_slot, size, groups;
  int from, count;  // this block's group
  size_t lead;      // slot of its first part
};
// A block's part of an item [item0, item1) that other blocks have parts of.
struct Part {
  Join join;
  uint16_t *out;    // the item's output rows; null: there is no part
  int nh;
  unsigned before;  // parts of the group that had arrived before it
};
__device__ __forceinline__ Join join_of(const TileSplit &split, int64_t item0, int64_t item1) {
  Join j;
  j.first = split.owner(item0);
  const int parts = split.owner(item1 - 1) - j.first + 1;
  j.first_slot = split.start(j.first) < item0 ? 1 : 0;
  j.size = parts;
  if (parts > 16)
    for (j.size = 3; j.size * j.size < parts;) ++j.size;
  j.groups = (parts + j.size - 1) / j.size;
  j.from = ((int)blockIdx.x - j.first) / j.size * j.size;
  j.count = min(j.size, parts - j.from);
  j.lead = part_slot(j.first, j.first_slot, j.from);
  return j;
}
__device__ __forceinline__ unsigned arrive(unsigned *counter) {
  unsigned before;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  return before;
}

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
kv8_attn_kernel(const __grid_constant__ AttnParams p) {
  using S = Smem<D, NT>;
  constexpr int NH = 8 * NT, kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *const smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ Part sh_parts[2];  // of items that began, or end, in other blocks
  __shared__ bool sh_last;
  float *const merge = reinterpret_cast<float *>(smem + S::kMerge);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = lane >> 2, t = lane & 3;
  uint64_t *const full = reinterpret_cast<uint64_t *>(smem + S::kBars) + warp * kStages;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  if (tid == 0) {
    sh_parts[0].out = sh_parts[1].out = nullptr;
    tma_prefetch_desc(&p.k);
    tma_prefetch_desc(&p.v);
  }
  __syncwarp();
  const int items = p.heads * p.groups;

  grid_dependency_wait();
  fence_proxy_async_global();  // TMA reads what the launch before wrote
  grid_launch_dependents();

  // ---- this block's range of tiles
  auto tiles_of = [&](int b) {
    return visible_tiles(visible_keys(clamped_len(p, b), p.window, p.sinks), kTile).count;
  };
  // Every warp finds it for itself, 32 sequences at a time.
  const int n0 = lane < p.B ? tiles_of(lane) : 0;
  int seq_tiles = n0;
  for (int b = lane + 32; b < p.B; b += 32) seq_tiles += tiles_of(b);
  const int64_t total = (int64_t)__reduce_add_sync(0xffffffffu, seq_tiles) * items;
  const TileSplit split(total > 0 ? total : 1, gridDim.x);

  // Sequences without a token: zero rows.
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    const int len = p.lens[b];
    if (tid == 0 && (len < 0 || len > p.table_width << p.page_shift)) record_error(kErrOutOfBounds);
    if (len > 0) continue;
    uint4 *row = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.O) + b * p.o_stride);
    for (int i = tid; i < p.heads * p.group * D / 8; i += kThreads) row[i] = make_uint4(0, 0, 0, 0);
  }
  if (total == 0 || (int)blockIdx.x >= split.blocks) return;
  const int64_t t0 = split.start(blockIdx.x), t1 = split.start(blockIdx.x + 1);
  Cursor cur;
  cur.b = -1;
  int64_t base = 0;  // tiles before these 32 sequences
  for (int b0 = 0; b0 < p.B && cur.b < 0; b0 += 32) {
    const int n = b0 == 0 ? n0 : b0 + lane < p.B ? tiles_of(b0 + lane) : 0;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const int64_t begin = base + (int64_t)(upto - n) * items;
    const unsigned hit = __ballot_sync(0xffffffffu, t0 >= begin && t0 < begin + (int64_t)n * items);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int off = __shfl_sync(0xffffffffu, (int)(t0 - begin), src);
      set_sequence(cur, p, b0 + src);
      const int count = __shfl_sync(0xffffffffu, n, src);
      cur.item = off / count;
      cur.tile = off - cur.item * count;
    }
    base += (int64_t)__shfl_sync(0xffffffffu, upto, 31) * items;
  }
  if (cur.b < 0) return;  // (lengths that change underneath)

  // ---- the warp's ring
  uint8_t *const ring = smem + warp * kStages * S::kStage;
  Meta *const metas = reinterpret_cast<Meta *>(smem + S::kMetas + warp * kStages * 32);
  const bool two = p.page_shift == 4;  // pages of 16 tokens: two per step
  Cursor pre = cur;
  int64_t pre_t = t0;
  // Pages of the item's tiles from `pages_at` on, one tile per lane, and their
  // scales; a lane issues the copies of its own tile.
  int pages[2] = {-1, -1}, pages_at = 0;
  float scales[4];
  auto look_up = [&]() {
    pages_at = pre.tile;
    const int i = pre.tile + lane;
    pages[0] = pages[1] = -1;
    scales[0] = scales[1] = scales[2] = scales[3] = 0.0f;
    if (i >= pre.tiles.count || pre_t + lane >= t1) return;
    const int k0 = tile_key(pre.tiles, i, kTile) + warp * 32;
    const int32_t *row = p.table + (int64_t)pre.b * p.table_width;
    const int head = pre.item / p.groups;
    const uint32_t mask = visible_mask(pre.vis, k0);
    bool bad = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (!(mask >> 16 * h & 0xffffu)) continue;
      pages[h] = row[(k0 + 16 * h) >> p.page_shift];
      if (pages[h] < 0 || pages[h] >= p.num_pages) {
        pages[h] = -1;
        bad = true;
      } else {
        scales[h] = p.k_scale[pages[h] * p.scale_stride + head];
        scales[2 + h] = p.v_scale[pages[h] * p.scale_stride + head];
      }
    }
    if (bad) record_error(kErrOutOfBounds);
  };
  // One step's copies into a stage. The scales, which come a lookup later, go
  // to `publish`, which also says how much the stage waits for.
  auto copy = [&](int stage) {
    uint32_t bytes = 0;
    if (lane == pre.tile - pages_at) {
      const int k0 = tile_key(pre.tiles, pre.tile, kTile) + warp * 32;
      uint8_t *at = ring + stage * S::kStage;
      const int row = ((pre.item / p.groups) << p.page_shift) + (k0 & ((1 << p.page_shift) - 1));
      if (two) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (pages[h] >= 0) {
            tma_load_3d(at + h * S::kHalf, &p.k, 0, row, pages[h], &full[stage]);
            tma_load_3d(at + (2 + h) * S::kHalf, &p.v, 0, row, pages[h], &full[stage]);
            bytes += 2 * S::kHalf;
          }
      } else {
        const int page = max(pages[0], pages[1]);
        if (page >= 0) {
          tma_load_3d(at, &p.k, 0, row, page, &full[stage]);
          tma_load_3d(at + 2 * S::kHalf, &p.v, 0, row, page, &full[stage]);
          bytes = S::kStage;
        }
      }
    }
    return bytes;
  };
  auto publish = [&](int stage, int tile, uint32_t bytes) {
    if (lane != tile - pages_at) return;
    const int k0 = tile_key(pre.tiles, tile, kTile) + warp * 32;
    uint32_t mask = visible_mask(pre.vis, k0);
    if (pages[0] < 0) mask &= 0xffff0000u;
    if (pages[1] < 0) mask &= 0x0000ffffu;
    Meta &m = metas[stage];
    m.k_scale[0] = scales[0];
    m.k_scale[1] = scales[1];
    m.v_scale[0] = scales[2];
    m.v_scale[1] = scales[3];
    m.mask = mask;
    mbar_arrive_expect_tx(&full[stage], bytes);
  };
  auto advance = [&]() {
    ++pre_t;
    const bool turn = ++pre.tile == pre.tiles.count;
    if (turn && pre_t < t1) next_item(pre, p);
    if (turn || pre.tile - pages_at == 32) look_up();
  };
  auto issue = [&](int stage) {
    if (pre_t >= t1) return;
    const uint32_t bytes = copy(stage);
    publish(stage, pre.tile, bytes);
    advance();
  };
  __syncwarp();
  look_up();
#pragma unroll 1
  for (int s = 0; s < kStages; ++s) issue(s);
  uint32_t phase = 0;
  bool ok = true;

  // Queries of an item, as they are.
  uint32_t q[NT][D / 16][2];
  auto load_q = [&](const Cursor &c) {
    const int h0 = c.item / p.groups * p.group + c.item % p.groups * NH;
    const int nh = min(NH, p.group - c.item % p.groups * NH);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool have = nt * 8 + r < nh;
      const uint16_t *src = static_cast<const uint16_t *>(p.Q) + c.b * p.q_stride +
                            (int64_t)(h0 + nt * 8 + (have ? r : 0)) * D + t * 16;
#pragma unroll
      for (int ks = 0; ks < D / 16; ks += 2) {
        const uint4 w = have ? *reinterpret_cast<const uint4 *>(src + (ks / 4) * 64 + (ks % 4) * 4)
                             : make_uint4(0, 0, 0, 0);
        q[nt][ks][0] = w.x;
        q[nt][ks][1] = w.y;
        q[nt][ks + 1][0] = w.z;
        q[nt][ks + 1][1] = w.w;
      }
    }
  };
  load_q(cur);
  int stage = 0;
  for (int64_t at_tile = t0; at_tile < t1;) {
    // ---- one item: its queries
    const int grp = cur.item % p.groups;
    const int h0 = cur.item / p.groups * p.group + grp * NH;  // first query head
    const int nh = min(NH, p.group - grp * NH);
    float mult[NT][2];  // of the scores of this thread's two columns
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float inv = 1.0f;
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
    float o[NT][D / 16][4], m[NT][2], peak[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = peak[nt][0] = peak[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
    }

    // ---- its tiles
    const int64_t left = t1 - at_tile;
    const int n = (int)(left < cur.tiles.count - cur.tile ? left : cur.tiles.count - cur.tile);
    if (n <= 0) break;
    for (int i = 0; i < n; ++i) {
      if (!ok) break;
      ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase));
      if (!ok) break;
      const uint32_t at = smem_u32(ring + stage * S::kStage);
      const uint4 sc = lds128(smem_u32(&metas[stage]));
      const uint32_t mask = metas[stage].mask;
      const int mine = stage;
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
      if (mask == 0) {  // uniform over the warp
        __syncwarp();
        issue(mine);
        continue;
      }
      const float ks[2] = {__uint_as_float(sc.x), __uint_as_float(sc.y)};
      const float vs[2] = {__uint_as_float(sc.z), __uint_as_float(sc.w)};

      // Row x of the product is key x of the half in an order in which the 8
      // lanes that a shared-memory read serves at once meet different banks:
      // even rows 2i take key 2i, odd rows 2i + 1 key (2i ^ 4) + 1.
      const int key_r = r & 1 ? ((r - 1) ^ 4) + 1 : r;
      float s[2][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[h][nt][x] = 0.0f;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const int ch = (4 * c + t) ^ (D == 128 ? key_r & 7 : (key_r >> 1) & 3);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t from = at + h * S::kHalf + key_r * D + ch * 16;
          const uint4 lo = lds128(from), hi = lds128(from + 8 * D);
          const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a0 = half2_lo(wl[j]), a1 = half2_lo(wh[j]), a2 = half2_hi(wl[j]),
                           a3 = half2_hi(wh[j]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816(s[h][nt], a0, a1, a2, a3, q[nt][4 * c + j][0], q[nt][4 * c + j][1]);
          }
        }
      }
      // Scores in log2 units; hidden keys -inf. A factor past fp32's range meets
      // products that are zero (scores are finite), which stay zero.
      auto factor = [](float back, float scale) {
        const float f = back * scale;
        return f > kLargest ? kLargest : f;
      };
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[h][nt][x] *= factor(mult[nt][x & 1], ks[h]);
      if (mask != 0xffffffffu) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (!(mask >> (16 * h + key_r + (x >> 1) * 8) & 1)) s[h][nt][x] = -INFINITY;
      }
      // log2 of the value scales: for the maximum kept from minus infinity, for
      // the weights not (a zero scale takes its values out).
      float lv[2], lvp[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        lv[h] = vs[h] > 0.0f ? fmaxf(lg2_approx(vs[h]), -110.0f) : -110.0f;
        lvp[h] = vs[h] > 0.0f ? lv[h] : -INFINITY;
      }
      float top[NT][2], high[NT][2];
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float a = fmaxf(s[0][nt][x], s[0][nt][2 + x]), b = fmaxf(s[1][nt][x], s[1][nt][2 + x]);
          top[nt][x] = fmaxf(a + lv[0], b + lv[1]);
          high[nt][x] = fmaxf(a, b);
          grow |= top[nt][x] > m[nt][x] + kLazy || high[nt][x] > peak[nt][x] + kLazy;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float mx = top[nt][x], pk = high[nt][x];
#pragma unroll
            for (int lanes = 4; lanes < 32; lanes *= 2) {
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, lanes));
              pk = fmaxf(pk, __shfl_xor_sync(0xffffffffu, pk, lanes));
            }
            mx = fmaxf(mx, m[nt][x]);
            pk = fmaxf(pk, peak[nt][x]);
            const float alpha = rescale(m[nt][x], mx);
            l[nt][x] *= rescale(peak[nt][x], pk);
            m[nt][x] = mx;
            peak[nt][x] = pk;
#pragma unroll
            for (int i2 = 0; i2 < D / 16; ++i2) {
              o[nt][i2][x] *= alpha;
              o[nt][i2][2 + x] *= alpha;
            }
          }
      }
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float mm[2] = {m[nt][0] == -INFINITY ? 0.0f : m[nt][0],
                             m[nt][1] == -INFINITY ? 0.0f : m[nt][1]};
        const float pp[2] = {peak[nt][0] == -INFINITY ? 0.0f : peak[nt][0],
                             peak[nt][1] == -INFINITY ? 0.0f : peak[nt][1]};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float w[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            // One difference for both, so that what the sum of a large score and a
            // scale is rounded by does not come between them.
            const float below = s[h][nt][x] - pp[x & 1];
            w[x] = ex2_approx(below + (pp[x & 1] - mm[x & 1] + lvp[h]));
            l[nt][x & 1] += ex2_approx(below);
          }
          pb[h][nt][0] = transpose8x8(pack_half2(w[0], w[1]));
          pb[h][nt][1] = transpose8x8(pack_half2(w[2], w[3]));
        }
      }
      // Values: rows 2t, 2t + 1, 2t + 8, 2t + 9, D / 8 codes from d = r D / 8 on.
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t v[4][D / 32];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int key = (k & 1 ? ((2 * t) ^ 4) + 1 : 2 * t) + (k >> 1) * 8;
          const uint32_t row = at + (2 + h) * S::kHalf + key * D;
          if constexpr (D == 128) {
            const uint4 w = lds128(row + ((r ^ (key & 7)) * 16));
            v[k][0] = w.x;
            v[k][1] = w.y;
            v[k][2] = w.z;
            v[k][3] = w.w;
          } else {
            const uint2 w = lds64(row + (((r >> 1) ^ ((key >> 1) & 3)) * 16) + (r & 1) * 8);
            v[k][0] = w.x;
            v[k][1] = w.y;
          }
          if (mask != 0xffffffffu && !(mask >> (16 * h + key) & 1)) {
#pragma unroll
            for (int j = 0; j < D / 32; ++j) v[k][j] = 0;
          }
        }
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t sel = u ? 0x7362 : 0x5140;
            const uint32_t ab = __byte_perm(v[0][j], v[1][j], sel), cd = __byte_perm(v[2][j], v[3][j], sel);
            const uint32_t a0 = half2_lo(ab), a1 = half2_hi(ab), a2 = half2_lo(cd), a3 = half2_hi(cd);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816(o[nt][2 * j + u], a0, a1, a2, a3, pb[h][nt][0], pb[h][nt][1]);
          }
      }
      __syncwarp();
      issue(mine);
    }

    // ---- the next item's queries are on their way while this one is joined
    const int64_t item0 = at_tile - cur.tile, item1 = item0 + cur.tiles.count;
    const bool whole = item0 >= t0 && item1 <= t1;
    const int slot_of_mine = item0 <= t0 ? 0 : 1;
    uint16_t *const out = static_cast<uint16_t *>(p.O) + cur.b * p.o_stride + (int64_t)h0 * D;
    at_tile += n;
    cur.tile += n;
    if (at_tile < t1) {
      next_item(cur, p);
      load_q(cur);
    }

    // ---- the warps' results joined, through shared memory: each warp takes a
    // quarter of the fragments, from the same lanes of all warps in order. The
    // joint reference of products and sums is the largest score, so that the sum
    // is at least 2^-8, or 2^48 above it where the values are large: sums of up to
    // 2^31 keys times 2^8 then leave the products (output times sum) within fp32.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], 4);
        l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], 8);
        l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], 16);
      }
    constexpr int kFrags = D / 16 * NT;  // float4 of O per thread
    float4 *const mine = reinterpret_cast<float4 *>(merge + warp * S::kMergeWarp) + lane;
    auto peaks_of = [&](int w) {  // behind the warp's fragments, maxima and sums
      return reinterpret_cast<float2 *>(merge + w * S::kMergeWarp + (kFrags + NT) * 32 * 4) + lane;
    };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        mine[(nt * (D / 16) + i) * 32] = make_float4(o[nt][i][0], o[nt][i][1], o[nt][i][2], o[nt][i][3]);
      mine[(kFrags + nt) * 32] = make_float4(m[nt][0], m[nt][1], l[nt][0], l[nt][1]);
      peaks_of(warp)[nt * 32] = make_float2(peak[nt][0], peak[nt][1]);
    }
    __syncthreads();
    {
      constexpr int kShare = kFrags / kWarps;
      const int nt = warp * kShare / (D / 16);  // of all of them
      const float4 *const from = reinterpret_cast<const float4 *>(merge) + lane;
      constexpr int kStep = S::kMergeWarp / 4;
      float4 ml[kWarps];
      float2 pk[kWarps];
      float mx[2] = {-INFINITY, -INFINITY}, ref[2] = {-INFINITY, -INFINITY};
      float sum[2] = {0.0f, 0.0f}, f[kWarps][2];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        ml[w] = from[w * kStep + (kFrags + nt) * 32];
        pk[w] = peaks_of(w)[nt * 32];
        mx[0] = fmaxf(mx[0], ml[w].x);
        mx[1] = fmaxf(mx[1], ml[w].y);
        ref[0] = fmaxf(ref[0], pk[w].x);
        ref[1] = fmaxf(ref[1], pk[w].y);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (mx[x] - ref[x] > 60.0f) ref[x] += 48.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        f[w][0] = rescale(ml[w].x, ref[0]);
        f[w][1] = rescale(ml[w].y, ref[1]);
        sum[0] += ml[w].z * rescale(pk[w].x, ref[0]);
        sum[1] += ml[w].w * rescale(pk[w].y, ref[1]);
      }
      float4 *const my_slot =
          reinterpret_cast<float4 *>(p.slots + ((size_t)blockIdx.x * 2 + slot_of_mine) * kSlotFloats);
#pragma unroll
      for (int j = 0; j < kShare; ++j) {
        const int at = warp * kShare + j;
        float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 y = from[w * kStep + at * 32];
          v.x += y.x * f[w][0];
          v.y += y.y * f[w][1];
          v.z += y.z * f[w][0];
          v.w += y.w * f[w][1];
        }
        if (whole)
          write_fragment<D, BF16>(out, nh, lane, nt, at % (D / 16), v, sum[0], sum[1]);
        else
          __stcg(my_slot + at * 32 + lane, v);
      }
      // The references and sums of a slot: [column] pairs behind its fragments.
      if (!whole && r == 0 && warp * kShare % (D / 16) == 0) {
        float2 *to = reinterpret_cast<float2 *>(my_slot + kFrags * 32) + nt * 8 + 2 * t;
        __stcg(to, make_float2(ref[0], sum[0]));
        __stcg(to + 1, make_float2(ref[1], sum[1]));
      }
    }
    __syncthreads();  // the merge buffer is free again, the block's stores come before the arrival
    // A part is counted in at once, but its join, where it falls to this block,
    // waits for the block's own work, which may be what others wait for.
    if (!whole && tid == 0) {
      Part &part = sh_parts[at_tile < t1 ? 0 : 1];
      part.join = join_of(split, item0, item1);
      part.out = out;
      part.nh = nh;
      part.before = arrive(&p.counters[part.join.lead >> 1].group[part.join.lead & 1]);
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    const Part part = sh_parts[i];
    const Join &j = part.join;
    if (!part.out || part.before + 1 != (unsigned)j.count) continue;  // another block is the last
    if (tid == 0) p.counters[j.lead >> 1].group[j.lead & 1] = 0;      // ready for the next call
    __threadfence();
    join_parts<D, NT, BF16>(p.slots, j.first, j.first_slot, j.from, j.count, 1,
                            j.groups == 1 ? part.out : nullptr, part.nh);
    if (j.groups == 1) continue;
    __syncthreads();
    if (tid == 0) {
      sh_last = arrive(&p.counters[j.first].item) + 1 == (unsigned)j.groups;
      if (sh_last) p.counters[j.first].item = 0;
    }
    __syncthreads();
    if (sh_last)
      join_parts<D, NT, BF16>(p.slots, j.first, j.first_slot, 0, j.groups, j.size, part.out, part.nh);
  }
  // Only a wait that ran out leaves copies behind: they get time to land.
  for (int i = 0; !ok && i < kStages; ++i) {
    mbar_wait(&full[stage], phase, 1000000000ull);
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
}

template <int D, int NT, bool BF16>
cudaError_t launch_typed(const AttnParams &p, cudaStream_t stream) {
  constexpr int bytes = Smem<D, NT>::kBytes;
  static_assert(kBlocksPerSm * (bytes + 1024) <= 228 * 1024, "blocks per SM");
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
  return launch_dependent(kv8_attn_kernel<D, NT, BF16>, dim3(grid_blocks()), kThreads, bytes, p, stream);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                  const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Codes of K or V as (d, heads * page_size, pages), boxes of up to 32 tokens of a page.
bool make_map(CUtensorMap *map, const vc_kv8_cache &c, void *codes) {
  auto encode = reinterpret_cast<EncodeTiledFn>(tensor_map_encoder());
  if (!encode) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.heads * c.page_size,
                              (cuuint64_t)c.num_pages};
  const cuuint64_t strides[2] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_stride};
  const cuuint32_t box[3] = {(cuuint32_t)c.head_dim, c.page_size < 32 ? 16u : 32u, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, codes, dims, strides, box, estr,
                CU_TENSOR_MAP_INTERLEAVE_NONE,
                c.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

size_t kv8_attn_workspace_bytes(const vc_kv8_cache &, int, int) {
  const size_t blocks = grid_blocks();
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
  AttnParams p{{}, {}, c.k_scale, c.v_scale, c.scale_stride, a.q_stride, a.o_stride,
               a.Q, a.O, a.table, a.lens, slots,
               reinterpret_cast<Counters *>(slots + (size_t)grid_blocks() * 2 * kSlotFloats),
               a.B, c.num_pages, shift, c.heads, group, groups, a.table_width, a.window,
               a.sinks, a.scale_log2};
  if (!make_map(&p.k, c, c.k) || !make_map(&p.v, c, c.v)) return cudaErrorInvalidValue;
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
