// What the kernels of the paged attention share (paged_decode.cu over 16-bit pools, paged_decode8.cu over 8-bit ones): how the
// sequences' tiles are dealt over the blocks, and the joining of what they leave.
//
// The work items (sequence, key head, chunk of up to 8 NT query heads), each a run of tiles of TILE tokens behind kItemCost
// units for its start and end, are laid end to end and every block takes an equal share of the units, whatever the
// sequences' lengths. An item that lies in one block is finished there; one that is cut leaves a partial
// (max, sum, 32-bit accumulators) per block, which a second kernel joins. That kernel has no room on an SM beside the first
// one's blocks, so all that it does is paid: the block that starts an item tells it which blocks hold the rest. (Found from the
// lengths instead, 64 sequences of up to 8190 tokens, 40/8 heads: 44.0 us for 41.5 in 16 bits, 39.8 for 38.5 in 8. A grid of the
// kernel's blocks, each joining the item that it cut: the same there, but 58.9 us for 51.4 over 12 long items.)
#pragma once
#include "common.cuh"
#include "launch.h"
#include "paged.h"

namespace vmb {
namespace {

constexpr int kWarps = 4;
constexpr int kItemCost = 2;  // what an item costs beside its tiles, in tiles
constexpr int kMinTiles = 4;  // a block's least share: below it the join costs more than the split gains

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// What a sequence's new token sees, with a window: the first `sink_tiles` tiles, then those from `base`
// on (a multiple of a warp's rows, so that a box stays inside a page); sink_tiles and base are 0 where the two meet. Without a window
// all of it: tiles from 0 on.
struct Span {
  int sink_tiles, base, tiles;
};
template <bool WIN, int TILE>
__device__ __forceinline__ Span span_of(const PagedParams& p, int len) {
  Span s{0, 0, 0};
  if (WIN) {
    s.sink_tiles = (min(p.sinks, len) + TILE - 1) / TILE;
    s.base = max(len - p.window, 0) & ~(TILE / kWarps - 1);
    if (s.base <= s.sink_tiles * TILE && s.sink_tiles > 0) s.sink_tiles = s.base = 0;
  }
  s.tiles = len > 0 ? s.sink_tiles + (len - s.base + TILE - 1) / TILE : 1;
  return s;
}
template <bool WIN, int TILE>
__device__ __forceinline__ int tiles_of(const PagedParams& p, int len) { return span_of<WIN, TILE>(p, len).tiles; }
__device__ __forceinline__ int seq_len(const PagedParams& p, int b) {
  return max(0, min(p.lengths[b], p.max_len));
}

// The flat order of units: sequences, then items (key head, head chunk) of a sequence, then kItemCost units
// and the item's tiles.
template <bool WIN, int TILE>
__device__ __forceinline__ int units_of(const PagedParams& p, int len) { return kItemCost + tiles_of<WIN, TILE>(p, len); }
// Units of one item of every sequence, summed (warp-collective).
template <bool WIN, int TILE>
__device__ __forceinline__ long long total_units(const PagedParams& p, int lane) {
  long long sum = 0;
  for (int b = lane; b < p.batch; b += 32) sum += units_of<WIN, TILE>(p, seq_len(p, b));
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  return sum;
}
// Blocks that take part: every one has at least kMinTiles units.
__device__ __forceinline__ long long parts_of(const PagedParams& p, long long total) {
  const long long most = (total + kMinTiles - 1) / kMinTiles;
  return most < p.blocks ? most : p.blocks;
}

// A walk over a block's tiles: `left` units from the tile it stands at to the end of the block's share.
struct Cursor {
  int seq, item, tile, tiles, len;
  int left;
  int sink_tiles, base;  // with a window
  template <bool WIN, int TILE>
  __device__ __forceinline__ void enter(const PagedParams& p) {  // the sequence `seq`
    len = seq_len(p, seq);
    const Span s = span_of<WIN, TILE>(p, len);
    tiles = s.tiles;
    if (WIN) sink_tiles = s.sink_tiles, base = s.base;
  }
  // first token of the tile
  template <bool WIN, int TILE>
  __device__ __forceinline__ int token() const {
    return !WIN || tile < sink_tiles ? tile * TILE : base + (tile - sink_tiles) * TILE;
  }
};
// The first tile at or behind unit `at` (warp-collective).
template <bool WIN, int TILE>
__device__ __forceinline__ void seek(const PagedParams& p, long long at, int left, int lane, Cursor& c) {
  long long before = 0;
  c = Cursor{0, 0, 0, 1, 0, 0, 0, 0};
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + lane;
    const int t = b < p.batch ? units_of<WIN, TILE>(p, seq_len(p, b)) : 0;
    int incl = t;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, s);
      if (lane >= s) incl += y;
    }
    const unsigned m = __ballot_sync(0xffffffffu, at < (before + incl) * p.items);
    if (m) {
      const int l = __ffs(m) - 1, units = __shfl_sync(0xffffffffu, t, l);
      const long long rel = at - (before + __shfl_sync(0xffffffffu, incl - t, l)) * p.items;
      const int in = (int)(rel % units) - kItemCost;  // negative: the item's own cost comes first
      c.seq = b0 + l;
      c.item = (int)(rel / units);
      c.enter<WIN, TILE>(p);
      c.tile = in > 0 ? in : 0;
      c.left = left + (in < 0 ? in : 0);
      return;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
}
template <bool WIN, int TILE>
__device__ __forceinline__ void advance(const PagedParams& p, Cursor& c) {
  --c.left;
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  c.left -= kItemCost;
  if (++c.item < p.items) return;
  c.item = 0;
  if (++c.seq < p.batch) c.enter<WIN, TILE>(p);
}

// A block of 512 threads joins `rows` heads of an item from the blocks [c0, c1]: DP / 4 lanes hold a row's columns, four each; the
// threads' groups of lanes are dealt over the heads (group g has head r of those from g0 on), and a head's groups over the parts.
template <typename T, int DP, int NT>
__device__ __forceinline__ void join_parts(const PagedParams& p, int seq, int h, int g0, int r, int rows, int c0, int c1) {
  constexpr int HEADS = 8 * NT, LANES = DP / 4, GROUPS = 512 / LANES;
  __shared__ float4 sum_o[GROUPS][LANES];
  __shared__ float2 sum_ml[GROUPS];
  const int grp = threadIdx.x / LANES, d4 = threadIdx.x % LANES, per = GROUPS / rows;
  const int64_t head = (int64_t)h * p.group + g0 + r;
  // block c0 holds the item's start (its second slot), the others continue it (their first)
  auto at = [&](int c) { return ((int64_t)c * 2 + (c == c0 ? 1 : 0)) * HEADS + r; };
  float m = -1e30f, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (grp < per * rows) {
#pragma unroll 4
    for (int c = c0 + grp / rows; c <= c1; c += per) {
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at(c) * 2);
      const float4 v = reinterpret_cast<const float4*>(p.part + at(c) * DP)[d4];
      const float mn = fmaxf(m, ml.x), fa = fast_exp2(m - mn), fb = fast_exp2(ml.x - mn);
      l = l * fa + ml.y * fb;
      o.x = o.x * fa + v.x * fb;
      o.y = o.y * fa + v.y * fb;
      o.z = o.z * fa + v.z * fb;
      o.w = o.w * fa + v.w * fb;
      m = mn;
    }
  }
  sum_o[grp][d4] = o;
  if (d4 == 0) sum_ml[grp] = make_float2(m, l);
  __syncthreads();
  if (grp >= rows) return;
  for (int i = 1; i < per; ++i) m = fmaxf(m, sum_ml[grp + i * rows].x);
  l = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < per; ++i) {
    const float f = fast_exp2(sum_ml[grp + i * rows].x - m);
    const float4 v = sum_o[grp + i * rows][d4];
    l += sum_ml[grp + i * rows].y * f;
    o.x += v.x * f;
    o.y += v.y * f;
    o.z += v.z * f;
    o.w += v.w * f;
  }
  if (4 * d4 < p.dim) {
    uint2 w;
    w.x = Elem<T>::pack(o.x / l, o.y / l);
    w.y = Elem<T>::pack(o.z / l, o.w / l);
    *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + (int64_t)seq * p.o_row + head * p.o_head + 4 * d4) = w;
  }
  if (d4 == 0 && p.lse) p.lse[(int64_t)seq * p.heads + head] = (m + log2f(l)) * kLn2;
}

// Joins the parts of one (sequence, query head), or where that would be more blocks than fit at once, of all
// heads of a (sequence, item): those without work (items in one block, most of a batch's) then cost no
// second wave.
template <typename T, int DP, int NT>
__global__ void __launch_bounds__(512) paged_join_kernel(const __grid_constant__ PagedParams p) {
  constexpr int HEADS = 8 * NT;
  const int seq = blockIdx.x / p.join_blocks, in_seq = blockIdx.x % p.join_blocks;
  const bool one = p.join_blocks == p.heads;  // a block per head
  const int item = one ? in_seq / p.group * p.chunks + in_seq % p.group / HEADS : in_seq;
  const int h = item / p.chunks, g0 = (item % p.chunks) * HEADS, rows = one ? 1 : min(HEADS, p.group - g0);
  // every block waits, those without work too: the stream's next kernel must find the first one done. (It is not let start before
  // that: its blocks would take the SMs from this one's.)
  wait_for_kernel_before();
  const int2 cut = p.cuts[(int64_t)seq * p.items + item];
  if (cut.x < 0) return;  // finished by its block
  join_parts<T, DP, NT>(p, seq, h, g0, one ? in_seq % p.group - g0 : threadIdx.x / (DP / 4) % rows, rows, cut.x, cut.y);
}

// The blocks of the item that this block has started and the end of its share cuts. `rest`: tiles of the item behind it.
__device__ __forceinline__ int2 cut_behind(long long total, long long parts, int rest) {
  const long long last = total * (blockIdx.x + 1) / parts;  // the end of the share, in units
  return make_int2(blockIdx.x, (int)(((last + rest) * parts - 1) / total));
}

}  // namespace
}  // namespace vmb
