// Attention of one new token per sequence over a paged key / value cache.
//
//   o_b,h = sum_t p_t v_t / sum_t p_t,  p_t = exp(sm_scale q_b,h . k_t - m),  t < lengths[b],
// where token t of sequence b lies in slot t % page_size of page table[b][t / page_size]; with a window (WIN) over its
// tokens t >= lengths[b] - window and t < sinks, whose tiles alone are walked.
//
// Every cached key and value is read once for up to 16 query heads that share it (larger groups go in chunks of 16), so the
// work is bound by memory: 4 D bytes and 4 D group flops a token and key head. The work items (sequence, key
// head, chunk of up to 8 NT query heads), each a run of 64-token tiles behind kItemCost units for its start
// and end, are laid end to end and every block takes an equal share of the units, whatever the
// sequences' lengths. An item that lies in one block is finished there; one that is cut leaves a partial
// (max, sum, 32-bit accumulators) per block, which a second kernel joins. Two blocks per SM, about 128 KB
// of keys and values in flight on each SM.
//
// A warp owns 16 tokens of every tile and its own ring of TMA stages, so the loop has no block-wide
// synchronisation. A stage is as few TMA boxes as the page size allows (64 columns x gcd(16, page size) rows: four
// of them at D = 128 and pages of 16), each issued by a lane that has looked up its page one stage ahead;
// with per-thread 16-byte copies the addresses cost more issue slots than the arithmetic. Matrix
// products (mma.sync, m = 16 tokens, n = 8 heads, so a group of up to 8 wastes nothing):
//   S^T = K Q^T (A from shared memory, B = Q in registers), P^T moved to operand layout by movmatrix,
//   O^T += V^T P^T (A by transposing loads).
// tcgen05 would pad a group of 8 heads to 128 rows and pass every score through TMEM; the products here
// are 16 flops a byte at most, far below what mma.sync does.
// The four warps meet at the end of an item. P is rounded to 16 bits for the product; scores,
// exponentials, sums and accumulators are 32-bit.
//
// Scores of tokens past the length are dropped; the slots of a last page that hold no token may hold
// anything, so their value rows are cleared before the product (0 x inf). Pages past the last, page ids outside
// the pool and columns past D arrive as zeros (coordinates outside the tensor map).
//
// 64 sequences of up to 8190 tokens, 40/8 heads, D = 128, pages of 16: 44 us, 4.3 TB/s; 3 of up to 262143, 16/4 heads,
// pages of 64: 93 us, 5.8 TB/s (the measured copy rate is 6.5); one of 201 tokens, 8/2 heads, D = 64: 6.5 us, replayed in a graph.
//
// 8-bit pools (E8): e4m3 values, each page and head with a scale for its keys and one for its values, a sixteenth to half of
// whose work is the same but for the operands. A 16-token row of boxes is one swizzle atom of 128 bytes a token; ldmatrix moves pairs
// of bytes, which leaves a lane with four neighbouring columns of a key (a permutation of the contraction index that the
// queries share) and, transposed, with two neighbouring columns of two tokens (a byte permutation, and rows 2 r and 2 r + 1
// of V^T where the 16-bit form has r and r + 8). e4m3 converts to fp16 exactly, so the products are fp16 for bf16 queries
// too: a row of those is scaled by the power of two that brings its largest element below 2^15, which loses nothing above
// 2^-29 of it. The key scale multiplies the score. The value scale goes into the exponent: the sum takes 2^(x - m), the
// product 2^(x + log2 scale - m'), each against its own running maximum, so that pages of any scales meet in one
// accumulator with the precision that they would have alone; the end of an item brings the accumulators from m' to m.
//
// Waits for a stage are bounded (sm100.cuh): a warp that gives up records a code, goes through the rest of its share
// without loads, waits and products, drains its copies and leaves the block's outputs invalid.
#include <algorithm>
#include <numeric>
#include <type_traits>

#include "common.cuh"
#include "launch.h"
#include "paged.h"
#include "sm100.cuh"
#include "tma_host.h"

namespace vmb {

__device__ int g_paged_err;

namespace {

using namespace sm100;

constexpr int kTile = 64;     // tokens per tile: 16 per warp
constexpr int kWarps = 4;
constexpr int kItemCost = 2;  // what an item costs beside its tiles, in tiles
constexpr int kMinTiles = 4;  // a block's least share: below it the join costs more than the split gains

template <int DP, int NT, bool E8>
struct Cfg {
  static constexpr int STAGES = E8 ? 5 : DP == 128 ? 3 : 6;
  static constexpr int ATOM = 16 * 128;             // 16 tokens x 128 bytes (64 columns, or 128 of e4m3), 128-byte swizzle
  static constexpr int NA = E8 ? 1 : DP / 64;
  static constexpr int STAGE = 2 * NA * ATOM;       // K atoms, V atoms
  static constexpr int RING = kWarps * STAGES * STAGE;
  static constexpr int SCALES = E8 ? kWarps * STAGES * 128 : 0;  // per stage 16 scales of keys, 16 of values
  static constexpr int LD = DP + 4;              // joined accumulators: 8 heads per warp at a time
  static constexpr int JOIN = kWarps * 8 * LD * 4 + kWarps * 8 * 2 * 4;  // accumulators, (max, sum)
  static constexpr int SMEM = RING + JOIN + SCALES + kWarps * STAGES * 8 + 16;  // + barriers, abort flag
  static_assert(2 * (SMEM + 1024) <= 233472, "two blocks per SM");
};

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Two e4m3 values (the low or high half of x) as two fp16, exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t x) {
  uint32_t y;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2_hi(uint32_t x) {
  uint32_t y;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(y) : "r"(x));
  return y;
}
// 4 bytes from global to shared memory, or zeros.
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}

// What a sequence's new token sees, with a window: the tiles of the first `sink_tiles` x 64 tokens, then those from `base`
// on (a multiple of 16, so that a box stays inside a page); sink_tiles and base are 0 where the two meet. Without a window
// all of it: tiles from 0 on.
struct Span {
  int sink_tiles, base, tiles;
};
template <bool WIN>
__device__ __forceinline__ Span span_of(const PagedParams& p, int len) {
  Span s{0, 0, 0};
  if (WIN) {
    s.sink_tiles = (min(p.sinks, len) + kTile - 1) / kTile;
    s.base = max(len - p.window, 0) & ~15;
    if (s.base <= s.sink_tiles * kTile && s.sink_tiles > 0) s.sink_tiles = s.base = 0;
  }
  s.tiles = len > 0 ? s.sink_tiles + (len - s.base + kTile - 1) / kTile : 1;
  return s;
}
template <bool WIN>
__device__ __forceinline__ int tiles_of(const PagedParams& p, int len) { return span_of<WIN>(p, len).tiles; }
__device__ __forceinline__ int seq_len(const PagedParams& p, int b) {
  return max(0, min(p.lengths[b], p.max_len));
}

// The flat order of units: sequences, then items (key head, head chunk) of a sequence, then kItemCost units
// and the item's tiles.
template <bool WIN>
__device__ __forceinline__ int units_of(const PagedParams& p, int len) { return kItemCost + tiles_of<WIN>(p, len); }
// Units of one item of every sequence, summed (warp-collective).
template <bool WIN>
__device__ __forceinline__ long long total_units(const PagedParams& p, int lane) {
  long long sum = 0;
  for (int b = lane; b < p.batch; b += 32) sum += units_of<WIN>(p, seq_len(p, b));
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
  template <bool WIN>
  __device__ __forceinline__ void enter(const PagedParams& p) {  // the sequence `seq`
    len = seq_len(p, seq);
    const Span s = span_of<WIN>(p, len);
    tiles = s.tiles;
    if (WIN) sink_tiles = s.sink_tiles, base = s.base;
  }
  // first token of the tile
  template <bool WIN>
  __device__ __forceinline__ int token() const {
    return !WIN || tile < sink_tiles ? tile * kTile : base + (tile - sink_tiles) * kTile;
  }
};
// The first tile at or behind unit `at` (warp-collective).
template <bool WIN>
__device__ __forceinline__ void seek(const PagedParams& p, long long at, int left, int lane, Cursor& c) {
  long long before = 0;
  c = Cursor{0, 0, 0, 1, 0, 0, 0, 0};
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + lane;
    const int t = b < p.batch ? units_of<WIN>(p, seq_len(p, b)) : 0;
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
      c.enter<WIN>(p);
      c.tile = in > 0 ? in : 0;
      c.left = left + (in < 0 ? in : 0);
      return;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
}
template <bool WIN>
__device__ __forceinline__ void advance(const PagedParams& p, Cursor& c) {
  --c.left;
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  c.left -= kItemCost;
  if (++c.item < p.items) return;
  c.item = 0;
  if (++c.seq < p.batch) c.enter<WIN>(p);
}

struct KParams {
  CUtensorMap tm_k, tm_v;  // boxes of 64 columns (e4m3: 128) x box_rows slots; coordinates (column, slot, head, page, 0)
  PagedParams p;
};

template <typename T, int DP, int NT, bool WIN, bool E8>
__global__ void __launch_bounds__(32 * kWarps, 2) paged_decode_kernel(const __grid_constant__ KParams kp) {
  using C = Cfg<DP, NT, E8>;
  using M = std::conditional_t<E8, __half, T>;  // type of the products' operands
  constexpr int KS = DP / 16;
  constexpr int HEADS = 8 * NT;
  const PagedParams& p = kp.p;
  extern __shared__ __align__(1024) uint8_t smem[];  // everything shared is in here, so that it starts on an atom
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(smem) + warp * C::STAGES * C::STAGE;
  const uint32_t scales = smem_u32(smem + C::RING + C::JOIN) + 128u * warp * C::STAGES;  // [stage][K, V][16]
  const uint32_t bar0 = smem_u32(smem + C::RING + C::JOIN + C::SCALES) + 8u * warp * C::STAGES;
  float* join = reinterpret_cast<float*>(smem + C::RING);          // [warp][8 heads][LD]
  float* join_ml = join + kWarps * 8 * C::LD;                       // [warp][8 heads][max, sum]
  volatile int* abort = reinterpret_cast<int*>(smem + C::RING + C::JOIN + C::SCALES + kWarps * C::STAGES * 8);

  let_next_kernel_start();
  if (lane == 0) {
    if (warp == 0) *abort = 0;
    for (int s = 0; s < C::STAGES; ++s) mbar_init(bar0 + 8u * s, 1);
    fence_mbar_init();
    prefetch_tmap(&kp.tm_k);
    prefetch_tmap(&kp.tm_v);
  }
  __syncthreads();
  Cursor cc;
  if (p.whole_items) {  // one block per item (short caches): no cut, no join
    cc.seq = blockIdx.x / p.items;
    cc.item = blockIdx.x % p.items;
    cc.tile = 0;
    cc.enter<WIN>(p);
    cc.left = cc.tiles;
  } else {
    const long long total = total_units<WIN>(p, lane) * p.items, parts = parts_of(p, total);
    if (blockIdx.x >= parts) return;
    const long long first = total * blockIdx.x / parts, last = total * (blockIdx.x + 1) / parts;
    seek<WIN>(p, first, (int)(last - first), lane, cc);
  }

  // whether token t takes part
  auto sees = [&](const Cursor& c, int t) { return t < c.len && (!WIN || t >= c.len - p.window || t < p.sinks); };
  // ---- loading. A stage's boxes: (row group of box_rows tokens) x (K, V) x atoms; lane i issues boxes i, i + 32.
  // 8-bit: lane i stands for the keys (i < 16) or values of token i % 16, whose scale it copies; the first of a group issues.
  const int boxes = 16 / p.box_rows * 2 * C::NA;
  Cursor lc = cc;
  if (p.hold_loads && warp == 0) lc.left = 0;
  int issued = 0;
  int page[2], slot[2];  // of this lane's boxes of the stage that is issued next
  auto look_up = [&](const Cursor& c) {
#pragma unroll
    for (int k = 0; k < (E8 ? 1 : 2); ++k) {
      const int box = lane + 32 * k;
      const int t = c.token<WIN>() + 16 * warp + (E8 ? lane & 15 : box / (2 * C::NA) * p.box_rows);
      page[k] = p.num_pages;  // outside the map: zeros
      slot[k] = 0;
      // (of a group that the window cuts all of the rows are loaded)
      bool wanted = (E8 || box < boxes) && t < c.len;
      if (WIN) wanted = wanted && (sees(c, t) || (t & ~(p.box_rows - 1)) + p.box_rows > c.len - p.window);
      if (wanted) {
        const int i = t / p.page_size;
        slot[k] = t - i * p.page_size;
        page[k] = p.table[(int64_t)c.seq * p.table_stride + i];
        if ((unsigned)page[k] >= (unsigned)p.num_pages) page[k] = p.num_pages;
      }
    }
  };
  auto issue = [&](int it) {  // stage it % STAGES <- this warp's rows of lc, then on to the next tile
    if (lc.left <= 0) return;
    const uint32_t st = ring + (it % C::STAGES) * C::STAGE, bar = bar0 + 8u * (it % C::STAGES);
    if (lane == 0) mbar_expect_tx(bar, C::STAGE);
    ++issued;
    __syncwarp();
    if constexpr (E8) {
      const int r = lane & 15;
      const bool v = lane >= 16, valid = page[0] < p.num_pages;
      const int head = lc.item / p.chunks;
      if ((r & (p.box_rows - 1)) == 0)
        tma_load(st + (v ? C::ATOM : 0) + r * 128, v ? &kp.tm_v : &kp.tm_k, 0, slot[0], BIdx(head, page[0], 0), bar);
      const float* from = v ? p.v_scale + page[0] * p.vs_page + head * p.vs_head : p.k_scale + page[0] * p.ks_page + head * p.ks_head;
      cp_async4(scales + (it % C::STAGES) * 128 + lane * 4, valid ? from : p.k_scale, valid);
    }
#pragma unroll
    for (int k = 0; k < (E8 ? 0 : 2); ++k) {
      const int box = lane + 32 * k;
      if (box < boxes) {
        const int part = box % (2 * C::NA);  // K atoms, then V atoms
        tma_load(st + part * C::ATOM + box / (2 * C::NA) * p.box_rows * 128, part < C::NA ? &kp.tm_k : &kp.tm_v,
                 64 * (part % C::NA), slot[k], BIdx(lc.item / p.chunks, page[k], 0), bar);
      }
    }
    advance<WIN>(p, lc);
    if (lc.left > 0) look_up(lc);
  };
  if (lc.left > 0) look_up(lc);
#pragma unroll
  for (int s = 0; s < C::STAGES - 1; ++s) {
    issue(s);
    if (E8) cp_async_commit();  // a group a stage, also behind the last
  }

  uint32_t qf[NT][KS][2];
  float acc[NT][KS][4], m[NT][2], l[NT][2];
  float mv[NT][2];  // 8-bit: the accumulators' reference
  float qs[NT][2];  // 8-bit: what a score is multiplied with, for heads 2 (lane % 4) and + 1
  // an item's query heads as B fragments (head = lane / 4, columns 2 (lane % 4) ...; 8-bit: columns 4 (lane % 4) ...)
  auto load_q = [&](const Cursor& c) {
    const int h = c.item / p.chunks, g0 = (c.item % p.chunks) * HEADS;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int g = g0 + 8 * nt + lane / 4;
      const T* q = static_cast<const T*>(p.q) + (int64_t)c.seq * p.q_row + (int64_t)(h * p.group + g) * p.q_head;
      if constexpr (E8) {
        float top = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int col = 16 * ks + 4 * (lane % 4);
          const uint2 x = g < p.group && col < p.dim ? *reinterpret_cast<const uint2*>(q + col) : make_uint2(0u, 0u);
          qf[nt][ks][0] = x.x;
          qf[nt][ks][1] = x.y;
          if (Elem<T>::is_bf16) {
            const float2 a = Elem<T>::unpack(x.x), b = Elem<T>::unpack(x.y);
            top = fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))), top);
          }
        }
        float factor = 1.f;
        if (Elem<T>::is_bf16) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int e = (int)(__float_as_uint(top) >> 23) - 127;  // top < 2^(e + 1); -127: none, 128: not finite
          const int up = top == 0.f || e == 128 ? 0 : min(14 - e, 126);
          factor = __uint_as_float((uint32_t)(127 - up) << 23);
          const float by = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int e2 = 0; e2 < 2; ++e2) {
              const float2 a = Elem<T>::unpack(qf[nt][ks][e2]);
              qf[nt][ks][e2] = Elem<__half>::pack(a.x * by, a.y * by);
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
          qs[nt][e] = p.scale_log2 * __shfl_sync(0xffffffffu, factor, 4 * (2 * (lane % 4) + e));
        continue;
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = 16 * ks + 8 * e + 2 * (lane % 4);
          qf[nt][ks][e] = g < p.group && col < p.dim ? *reinterpret_cast<const uint32_t*>(q + col) : 0u;
        }
    }
  };
  auto clear = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][ks][e] = 0.f;
      m[nt][0] = m[nt][1] = -1e30f;
      l[nt][0] = l[nt][1] = 0.f;
      if (E8) mv[nt][0] = mv[nt][1] = -1e30f;
    }
  };
  bool from_start = cc.tile == 0, ok = true;
  if (cc.left > 0) load_q(cc);
  clear();
  for (int it = 0; cc.left > 0; ++it) {
    if (ok && !__all_sync(0xffffffffu, mbar_wait(bar0 + 8u * (it % C::STAGES), (it / C::STAGES) & 1, abort, &g_paged_err, 1,
                                                 p.wait_limit))) {
      ok = false;  // no more loads and products, but on to the barriers that the block's warps share
      lc.left = 0;
    }
    const uint32_t ks_base = ring + (it % C::STAGES) * C::STAGE, vs_base = ks_base + C::NA * C::ATOM;
    const int t0 = cc.token<WIN>() + 16 * warp;
    const int left = ok ? cc.len - t0 : 0;  // tokens of this warp's rows
    uint32_t rows = 0;                      // with a window: those that take part, a bit each
    if (WIN && left > 0) rows = __ballot_sync(0xffffffffu, lane < 16 && sees(cc, t0 + lane));
    if (E8) {
      cp_async_wait<C::STAGES - 2>();  // this stage's scales
      __syncwarp();
    }
    if (WIN ? rows != 0 : left > 0) {
      if (WIN ? rows != 0xffffu : left < 16) {  // slots without a token that takes part: their values enter the product with weight 0
        for (int i = WIN ? lane : left * 8 * C::NA + lane; i < 16 * 8 * C::NA; i += 32) {
          const int r = i / (8 * C::NA), c = i % (8 * C::NA);
          if (WIN && ((rows >> r) & 1u)) continue;
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vs_base + (c >> 3) * C::ATOM + r * 128 + (c & 7) * 16),
                       "r"(0)
                       : "memory");
        }
        fence_proxy_async_smem();  // the next copy into this stage comes through the async proxy
        __syncwarp();
      }
      // 8-bit: scales of the rows' keys, logarithms of those of their values, and of the first row's that takes part
      float k_by[2], v_log[2], v_first = 0.f;
      if constexpr (E8) {
        float first;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(first) : "r"(scales + (it % C::STAGES) * 128 + 64 + (WIN ? __ffs(rows) - 1 : 0) * 4));
        v_first = fast_log2(first);
        const uint32_t at = scales + (it % C::STAGES) * 128 + lane / 4 * 4;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x;
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(k_by[e]) : "r"(at + 32 * e));
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at + 64 + 32 * e));
          v_log[e] = fast_log2(x);
        }
      }
      float s[NT][2][4];  // two chains of products each
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][0][e] = s[nt][1][e] = 0.f;
      if constexpr (E8) {
#pragma unroll
        for (int k2 = 0; k2 < KS / 2; ++k2) {  // 16 columns of rows 0-7, 8-15, the next 16 of them
          uint32_t x[4];
          const int r = lane & 15, c = 2 * k2 + (lane >> 4);
          ldsm_x4(ks_base + r * 128 + ((c ^ (r & 7)) << 4), x[0], x[1], x[2], x[3]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t a[4] = {e4m3x2_to_f16x2(x[2 * e]), e4m3x2_to_f16x2(x[2 * e + 1]), e4m3x2_to_f16x2_hi(x[2 * e]),
                                   e4m3x2_to_f16x2_hi(x[2 * e + 1])};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<M>(s[nt][e], a, qf[nt][2 * k2 + e][0], qf[nt][2 * k2 + e][1]);
          }
        }
      }
#pragma unroll
      for (int ks = 0; ks < (E8 ? 0 : KS); ++ks) {
        uint32_t a[4];
        const int r = lane & 15, c = (2 * ks + (lane >> 4)) & 7;
        ldsm_x4(ks_base + (ks >> 2) * C::ATOM + r * 128 + ((c ^ (r & 7)) << 4), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<T>(s[nt][ks & 1], a, qf[nt][ks][0], qf[nt][ks][1]);
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        // rows: tokens lane / 4 and + 8; columns: heads 2 (lane % 4) and + 1
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = (s[nt][0][e] + s[nt][1][e]) * (E8 ? qs[nt][e & 1] * k_by[e >> 1] : p.scale_log2);
          const int r = lane / 4 + 8 * (e >> 1);
          if (WIN ? !((rows >> r) & 1u) : r >= left) x[e] = -INFINITY;
        }
        float mx[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) {
          mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], w));
          mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], w));
        }
        float y[4], my[2];  // 8-bit: the scores that weigh the values, with their scale
        if constexpr (E8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = x[e] == -INFINITY ? x[e] : x[e] + v_log[e >> 1];
          if (p.box_rows == 16) {  // one page, one scale
            my[0] = mx[0] + v_first;
            my[1] = mx[1] + v_first;
          } else {
            my[0] = fmaxf(y[0], y[2]);
            my[1] = fmaxf(y[1], y[3]);
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) {
              my[0] = fmaxf(my[0], __shfl_xor_sync(0xffffffffu, my[0], w));
              my[1] = fmaxf(my[1], __shfl_xor_sync(0xffffffffu, my[1], w));
            }
          }
        }
        if (__any_sync(0xffffffffu, mx[0] > m[nt][0] || mx[1] > m[nt][1] ||
                                        (E8 && (my[0] > mv[nt][0] || my[1] > mv[nt][1])))) {
          float al[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mn = fmaxf(m[nt][e], mx[e]);
            al[e] = fast_exp2(m[nt][e] - mn);
            m[nt][e] = mn;
            l[nt][e] *= al[e];
            if constexpr (E8) {
              const float vn = fmaxf(mv[nt][e], my[e]);
              al[e] = fast_exp2(mv[nt][e] - vn);
              mv[nt][e] = vn;
            }
          }
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][ks][e] *= al[e & 1];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fast_exp2(x[e] - m[nt][e & 1]);
        l[nt][0] += x[0] + x[2];
        l[nt][1] += x[1] + x[3];
        if constexpr (E8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = fast_exp2(y[e] - mv[nt][e & 1]);
        }
        pb[nt][0] = movmatrix(Elem<M>::pack(x[0], x[1]));
        pb[nt][1] = movmatrix(Elem<M>::pack(x[2], x[3]));
      }
      if constexpr (E8) {
#pragma unroll
        for (int k2 = 0; k2 < KS / 2; ++k2) {  // 16 columns of tokens 0-7, 8-15, the next 16 of them
          uint32_t x[4];
          const int r = lane & 15, c = 2 * k2 + (lane >> 4);
          ldsm_x4_t(vs_base + r * 128 + ((c ^ (r & 7)) << 4), x[0], x[1], x[2], x[3]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // columns (2 r, 2 r + 1) of two tokens -> two tokens of column 2 r, two of 2 r + 1
            const uint32_t lo = __byte_perm(x[2 * e], 0, 0x3120), hi = __byte_perm(x[2 * e + 1], 0, 0x3120);
            const uint32_t a[4] = {e4m3x2_to_f16x2(lo), e4m3x2_to_f16x2_hi(lo), e4m3x2_to_f16x2(hi), e4m3x2_to_f16x2_hi(hi)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<M>(acc[nt][2 * k2 + e], a, pb[nt][0], pb[nt][1]);
          }
        }
      }
#pragma unroll
      for (int ks = 0; ks < (E8 ? 0 : KS); ++ks) {
        // V^T: rows d, columns tokens; matrices (tokens 0-7, 8-15) x (d, d + 8)
        uint32_t a[4];
        const int r = (lane & 7) + 8 * (lane >> 4), c = (2 * ks + ((lane >> 3) & 1)) & 7;
        ldsm_x4_t(vs_base + (ks >> 2) * C::ATOM + r * 128 + ((c ^ (r & 7)) << 4), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<T>(acc[nt][ks], a, pb[nt][0], pb[nt][1]);
      }
    }
    __syncwarp();  // every lane is done with the stage that the next issue refills
    issue(it + C::STAGES - 1);
    if (E8) cp_async_commit();

    const Cursor done = cc;
    advance<WIN>(p, cc);
    const bool to_end = cc.tile == 0;
    if (to_end || cc.left <= 0) {
      // ---- the four warps' parts of this item (or of this block's share of it)
      if (cc.left > 0) load_q(cc);  // of the next item, on its way meanwhile
      const int h = done.item / p.chunks, g0 = (done.item % p.chunks) * HEADS;
      const bool whole = from_start && to_end;
      const int64_t part = (int64_t)blockIdx.x * 2 + (from_start ? 1 : 0);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
          if (lane < 4) {
            join_ml[(warp * 8 + 2 * lane + e) * 2] = m[nt][e];
            join_ml[(warp * 8 + 2 * lane + e) * 2 + 1] = l[nt][e];
          }
        }
        float to_m[2] = {1.f, 1.f};
        if (E8) to_m[0] = fast_exp2(mv[nt][0] - m[nt][0]), to_m[1] = fast_exp2(mv[nt][1] - m[nt][1]);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            join[(warp * 8 + 2 * (lane % 4) + (e & 1)) * C::LD + 16 * ks + (E8 ? 2 * (lane / 4) + (e >> 1) : lane / 4 + 8 * (e >> 1))] =
                E8 ? acc[nt][ks][e] * to_m[e & 1] : acc[nt][ks][e];
        __syncthreads();
        for (int i = threadIdx.x; i < 8 * DP; i += 32 * kWarps) {
          const int r = i / DP, d = i % DP, g = g0 + 8 * nt + r;
          if (g >= p.group) break;  // rows only grow
          float mm = -1e30f, sum = 0.f, o = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, join_ml[(w * 8 + r) * 2]);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float f = fast_exp2(join_ml[(w * 8 + r) * 2] - mm);
            sum = fmaf(f, join_ml[(w * 8 + r) * 2 + 1], sum);
            o = fmaf(f, join[(w * 8 + r) * C::LD + d], o);
          }
          const int64_t head = h * p.group + g;
          if (whole) {
            if (d < p.dim) static_cast<T*>(p.o)[(int64_t)done.seq * p.o_row + head * p.o_head + d] =
                Elem<T>::from_f(sum == 0.f ? 0.f : o / sum);
            if (d == 0 && p.lse) p.lse[(int64_t)done.seq * p.heads + head] = sum == 0.f ? -INFINITY : (mm + log2f(sum)) * kLn2;
          } else {
            p.part[(part * HEADS + 8 * nt + r) * DP + d] = o;
            if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (part * HEADS + 8 * nt + r) * 2) = make_float2(mm, sum);
          }
        }
        __syncthreads();
      }
      clear();
      from_start = true;
    }
  }
  if (E8) cp_async_wait<0>();
  if (!ok) {  // a stage did not arrive in time: the copies under way must land before the block ends
    for (int i = max(issued - C::STAGES, 0); i < issued; ++i) mbar_wait_drain(bar0 + 8u * (i % C::STAGES), (i / C::STAGES) & 1);
  }
}

// Joins the parts of one (sequence, query head), or where that would be more blocks than fit at once, of all
// heads of a (sequence, item): those without work (items in one block, most of a batch's) then cost no
// second wave. DP / 4 lanes hold a row's columns, four each; the 512 threads' groups of lanes are dealt over the
// heads, and a head's groups over the parts.
template <typename T, int DP, int NT, bool WIN>
__global__ void __launch_bounds__(512) paged_join_kernel(const __grid_constant__ PagedParams p) {
  constexpr int HEADS = 8 * NT, LANES = DP / 4, GROUPS = 512 / LANES;
  __shared__ float4 sum_o[GROUPS][LANES];
  __shared__ float2 sum_ml[GROUPS];
  const int lane = threadIdx.x & 31;
  const int seq = blockIdx.x / p.join_blocks, in_seq = blockIdx.x % p.join_blocks;
  const bool one = p.join_blocks == p.heads;  // a block per head
  const int item = one ? in_seq / p.group * p.chunks + in_seq % p.group / HEADS : in_seq;
  // where the item lies among the blocks' shares (lengths are inputs: readable before the wait)
  long long total = 0, before = 0;
  for (int b = lane; b < p.batch; b += 32) {
    const int t = units_of<WIN>(p, seq_len(p, b));
    total += t;
    if (b < seq) before += t;
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, s);
    before += __shfl_xor_sync(0xffffffffu, before, s);
  }
  total *= p.items;
  const int tiles = tiles_of<WIN>(p, seq_len(p, seq));
  const long long parts = parts_of(p, total), t0 = before * p.items + (long long)item * (kItemCost + tiles) + kItemCost;
  const int c0 = (int)(((t0 + 1) * parts - 1) / total), c1 = (int)(((t0 + tiles) * parts - 1) / total);
  // every block waits, those without work too: the stream's next kernel must find the first one done
  wait_for_kernel_before();
  if (c0 == c1) return;  // finished by its block
  const int h = item / p.chunks, g0 = (item % p.chunks) * HEADS, rows = one ? 1 : min(HEADS, p.group - g0);
  const int grp = threadIdx.x / LANES, d4 = threadIdx.x % LANES, per = GROUPS / rows;
  const int r = one ? in_seq % p.group - g0 : grp % rows;
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

template <typename T, int DP, int NT, bool WIN, bool E8>
cudaError_t launch(const PagedParams& p, cudaStream_t st) {
  using C = Cfg<DP, NT, E8>;
  KParams kp{};
  kp.p = p;
  auto map = [&](CUtensorMap* m, const void* base, int64_t page, int64_t head, int64_t slot) {
    const View v{slot > 0 ? slot : p.dim, head, page, 0};
    const int64_t batch = (int64_t)p.kv_heads * p.num_pages;
    return E8 ? tma::make_map_view_e4m3(m, base, p.dim, p.page_size, batch, v, p.kv_heads, p.num_pages, p.box_rows)
              : tma::make_map_view(m, base, Elem<T>::is_bf16, p.dim, p.page_size, batch, v, p.kv_heads, p.num_pages, p.box_rows);
  };
  if (!map(&kp.tm_k, p.k, p.k_page, p.k_head, p.k_slot) || !map(&kp.tm_v, p.v, p.v_page, p.v_head, p.v_slot))
    return cudaErrorInvalidValue;
  auto kern = paged_decode_kernel<T, DP, NT, WIN, E8>;
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = allow_smem(kern, C::SMEM, ready);
  if (e != cudaSuccess) return e;
  // not launched early: the join behind it reads the lengths before it waits, and this kernel's start is what makes them final
  kern<<<(unsigned)p.blocks, 32 * kWarps, C::SMEM, st>>>(kp);
  e = cudaGetLastError();
  if (e != cudaSuccess || p.whole_items) return e;
  // the join starts while the last blocks still run and waits on the device for what they wrote
  return launch_early(paged_join_kernel<T, DP, NT, WIN>, (int64_t)p.batch * p.join_blocks, 512, 0, st, p);
}

template <typename T, bool WIN, bool E8>
cudaError_t launch_dim(const PagedParams& p, cudaStream_t st) {
  if (p.dim > 64) return p.nt == 2 ? launch<T, 128, 2, WIN, E8>(p, st) : launch<T, 128, 1, WIN, E8>(p, st);
  return p.nt == 2 ? launch<T, 64, 2, WIN, E8>(p, st) : launch<T, 64, 1, WIN, E8>(p, st);
}
template <typename T>
cudaError_t launch_kind(const PagedParams& p, cudaStream_t st) {
  if (p.k_scale) return p.window ? launch_dim<T, true, true>(p, st) : launch_dim<T, false, true>(p, st);
  return p.window ? launch_dim<T, true, false>(p, st) : launch_dim<T, false, false>(p, st);
}

}  // namespace

void paged_plan(PagedParams& p) {
  p.group = p.heads / p.kv_heads;
  p.nt = p.group > 8 ? 2 : 1;  // 8 or 16 query heads share a pass over their keys
  p.chunks = (p.group + 8 * p.nt - 1) / (8 * p.nt);
  p.items = p.kv_heads * p.chunks;
  p.join_blocks = (int64_t)p.batch * p.heads <= 4 * 148 ? p.heads : p.items;  // four blocks of 512 threads an SM
  p.box_rows = std::gcd(16, p.page_size);
  int64_t tiles = ((int64_t)p.max_len + kTile - 1) / kTile;  // most that an item can have
  if (p.window) tiles = std::min(tiles, ((int64_t)p.sinks + kTile - 1) / kTile + ((int64_t)p.window + 15 + kTile - 1) / kTile);
  p.whole_items = tiles <= kMinTiles;
  p.blocks = p.whole_items ? (int64_t)p.batch * p.items : 2 * 148;
}

int64_t paged_workspace(const PagedParams& p) {
  if (p.whole_items) return 0;
  const int64_t rows = p.blocks * 2 * 8 * p.nt;
  return rows * (p.dim > 64 ? 128 : 64) * 4 + rows * 2 * 4;
}

cudaError_t paged_decode(PagedParams p, void* workspace, bool bf16, cudaStream_t st) {
  p.part = static_cast<float*>(workspace);
  p.part_ml = p.part + p.blocks * 2 * 8 * p.nt * (p.dim > 64 ? 128 : 64);
  return bf16 ? launch_kind<__nv_bfloat16>(p, st) : launch_kind<__half>(p, st);
}

cudaError_t paged_status(cudaStream_t st, int* out) {
  int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(out, g_paged_err, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && *out) e = cudaMemcpyToSymbolAsync(g_paged_err, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  return e;
}

}  // namespace vmb
