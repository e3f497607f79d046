// Attention of one new token per sequence over a paged key / value cache.
//
//   o_b,h = sum_t p_t v_t / sum_t p_t,  p_t = exp(sm_scale q_b,h . k_t - m),  t < lengths[b],
// where token t of sequence b lies in slot t % page_size of page table[b][t / page_size]; with a window (WIN) over its
// tokens t >= lengths[b] - window and t < sinks, whose tiles alone are walked.
//
// Every cached key and value is read once for up to 16 query heads that share it (larger groups go in chunks of 16), so the
// work is bound by memory: 4 D bytes and 4 D group flops a token and key head. paged_tiles.cuh deals the tiles over the
// blocks and joins items that are cut. Two blocks per SM, about 128 KB of keys and values in flight on each SM.
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
// 64 sequences of up to 8190 tokens, 40/8 heads, D = 128, pages of 16: 41.5 us, 4.6 TB/s; 3 of up to 262143, 16/4 heads,
// pages of 64: 91 us, 5.9 TB/s (the measured copy rate is 6.5); one of 201 tokens, 8/2 heads, D = 64: 6.5 us, replayed in a graph.
//
// Waits for a stage are bounded (sm100.cuh): a warp that gives up records a code, goes through the rest of its share
// without loads, waits and products, drains its copies and leaves the block's outputs invalid.
#include <algorithm>
#include <numeric>

#include "paged_tiles.cuh"
#include "sm100.cuh"
#include "tma_host.h"

namespace vmb {

__device__ int g_paged_err;

namespace {

using namespace sm100;

constexpr int kTile = 64;  // tokens per tile: 16 per warp
// With a window, sinks may hold nearly all of the weight and small values, so that the rest is what counts: in fp16 the reference stays
// this far below the largest score, P <= 2^15, and weights down to 2^-29 of the largest keep their bits.
template <typename T, bool WIN>
constexpr float kLift = WIN && !Elem<T>::is_bf16 ? 15.f : 0.f;

template <int DP, int NT>
struct Cfg {
  static constexpr int STAGES = DP == 128 ? 3 : 6;
  static constexpr int ATOM = 16 * 128;             // 16 tokens x 64 columns, 128-byte swizzle
  static constexpr int NA = DP / 64;
  static constexpr int STAGE = 2 * NA * ATOM;       // K atoms, V atoms
  static constexpr int RING = kWarps * STAGES * STAGE;
  static constexpr int LD = DP + 4;              // joined accumulators: 8 heads per warp at a time
  static constexpr int JOIN = kWarps * 8 * LD * 4 + kWarps * 8 * 2 * 4;  // accumulators, (max, sum)
  static constexpr int SMEM = RING + JOIN + kWarps * STAGES * 8 + 32;       // + barriers, abort flag, the share's numbers
  static_assert(2 * (SMEM + 1024) <= 233472, "two blocks per SM");
};

struct KParams {
  CUtensorMap tm_k, tm_v;  // boxes of 64 columns x box_rows slots; coordinates (column, slot, head, page, 0)
  PagedParams p;
};

template <typename T, int DP, int NT, bool WIN>
__global__ void __launch_bounds__(32 * kWarps, 2) paged_decode_kernel(const __grid_constant__ KParams kp) {
  using C = Cfg<DP, NT>;
  constexpr int KS = DP / 16;
  constexpr int HEADS = 8 * NT;
  const PagedParams& p = kp.p;
  extern __shared__ __align__(1024) uint8_t smem[];  // everything shared is in here, so that it starts on an atom
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(smem) + warp * C::STAGES * C::STAGE;
  const uint32_t bar0 = smem_u32(smem + C::RING + C::JOIN) + 8u * warp * C::STAGES;
  float* join = reinterpret_cast<float*>(smem + C::RING);          // [warp][8 heads][LD]
  float* join_ml = join + kWarps * 8 * C::LD;                       // [warp][8 heads][max, sum]
  volatile int* abort = reinterpret_cast<int*>(smem + C::RING + C::JOIN + kWarps * C::STAGES * 8);
  long long* share = reinterpret_cast<long long*>(smem + C::RING + C::JOIN + kWarps * C::STAGES * 8 + 8);  // units, blocks that take part

  if (lane == 0) {
    if (warp == 0) *abort = 0;
    for (int s = 0; s < C::STAGES; ++s) mbar_init(bar0 + 8u * s, 1);
    fence_mbar_init();
    prefetch_tmap(&kp.tm_k);
    prefetch_tmap(&kp.tm_v);
  }
  __syncthreads();
  wait_for_kernel_before();
  let_next_kernel_start();
  Cursor cc;
  if (p.whole_items) {  // one block per item (short caches): no cut, no join
    cc.seq = blockIdx.x / p.items;
    cc.item = blockIdx.x % p.items;
    cc.tile = 0;
    cc.enter<WIN, kTile>(p);
    cc.left = cc.tiles;
  } else {
    const long long total = total_units<WIN, kTile>(p, lane) * p.items, parts = parts_of(p, total);
    if (blockIdx.x >= parts) return;
    if (threadIdx.x == 0) share[0] = total, share[1] = parts;
    const long long first = total * blockIdx.x / parts, last = total * (blockIdx.x + 1) / parts;
    seek<WIN, kTile>(p, first, (int)(last - first), lane, cc);
  }

  // whether token t takes part
  auto sees = [&](const Cursor& c, int t) { return t < c.len && (!WIN || t >= c.len - p.window || t < p.sinks); };
  // ---- loading. A stage's boxes: (row group of box_rows tokens) x (K, V) x atoms; lane i issues boxes i, i + 32.
  const int boxes = 16 / p.box_rows * 2 * C::NA;
  Cursor lc = cc;
  if (p.hold_loads && warp == 0) lc.left = 0;
  int issued = 0;
  int page[2], slot[2];  // of this lane's boxes of the stage that is issued next
  auto look_up = [&](const Cursor& c) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int box = lane + 32 * k;
      const int t = c.token<WIN, kTile>() + 16 * warp + box / (2 * C::NA) * p.box_rows;
      page[k] = p.num_pages;  // outside the map: zeros
      slot[k] = 0;
      // (of a group that the window cuts all of the rows are loaded)
      bool wanted = box < boxes && t < c.len;
      if (WIN) wanted = wanted && (sees(c, t) || t + p.box_rows > c.len - p.window);
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
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int box = lane + 32 * k;
      if (box < boxes) {
        const int part = box % (2 * C::NA);  // K atoms, then V atoms
        tma_load(st + part * C::ATOM + box / (2 * C::NA) * p.box_rows * 128, part < C::NA ? &kp.tm_k : &kp.tm_v,
                 64 * (part % C::NA), slot[k], BIdx(lc.item / p.chunks, page[k], 0), bar);
      }
    }
    advance<WIN, kTile>(p, lc);
    if (lc.left > 0) look_up(lc);
  };
  if (lc.left > 0) look_up(lc);
#pragma unroll
  for (int s = 0; s < C::STAGES - 1; ++s) issue(s);

  uint32_t qf[NT][KS][2];
  float acc[NT][KS][4], m[NT][2], l[NT][2];
  // an item's query heads as B fragments (head = lane / 4, columns 2 (lane % 4) ...)
  auto load_q = [&](const Cursor& c) {
    const int h = c.item / p.chunks, g0 = (c.item % p.chunks) * HEADS;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int g = g0 + 8 * nt + lane / 4;
      const T* q = static_cast<const T*>(p.q) + (int64_t)c.seq * p.q_row + (int64_t)(h * p.group + g) * p.q_head;
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
    const int t0 = cc.token<WIN, kTile>() + 16 * warp;
    const int left = ok ? cc.len - t0 : 0;  // tokens of this warp's rows
    uint32_t rows = 0;                      // with a window: those that take part, a bit each
    if (WIN && left > 0) rows = __ballot_sync(0xffffffffu, lane < 16 && sees(cc, t0 + lane));
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
      float s[NT][2][4];  // two chains of products each
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][0][e] = s[nt][1][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
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
          x[e] = (s[nt][0][e] + s[nt][1][e]) * p.scale_log2;
          const int r = lane / 4 + 8 * (e >> 1);
          if (WIN ? !((rows >> r) & 1u) : r >= left) x[e] = -INFINITY;
        }
        float mx[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) {
          mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], w));
          mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], w));
        }
        mx[0] -= kLift<T, WIN>;
        mx[1] -= kLift<T, WIN>;
        if (__any_sync(0xffffffffu, mx[0] > m[nt][0] || mx[1] > m[nt][1])) {
          float al[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mn = fmaxf(m[nt][e], mx[e]);
            al[e] = fast_exp2(m[nt][e] - mn);
            m[nt][e] = mn;
            l[nt][e] *= al[e];
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
        pb[nt][0] = movmatrix(Elem<T>::pack(x[0], x[1]));
        pb[nt][1] = movmatrix(Elem<T>::pack(x[2], x[3]));
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
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

    const Cursor done = cc;
    advance<WIN, kTile>(p, cc);
    const bool to_end = cc.tile == 0;
    if (to_end || cc.left <= 0) {
      // ---- the four warps' parts of this item (or of this block's share of it)
      if (cc.left > 0) load_q(cc);  // of the next item, on its way meanwhile
      const int h = done.item / p.chunks, g0 = (done.item % p.chunks) * HEADS;
      const bool whole = from_start && to_end;
      if (from_start && !p.whole_items && threadIdx.x == 0)
        p.cuts[(int64_t)done.seq * p.items + done.item] = whole ? make_int2(-1, 0) : cut_behind(share[0], share[1], cc.tiles - cc.tile);
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
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            join[(warp * 8 + 2 * (lane % 4) + (e & 1)) * C::LD + 16 * ks + lane / 4 + 8 * (e >> 1)] = acc[nt][ks][e];
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
  if (!ok) {  // a stage did not arrive in time: the copies under way must land before the block ends
    for (int i = max(issued - C::STAGES, 0); i < issued; ++i) mbar_wait_drain(bar0 + 8u * (i % C::STAGES), (i / C::STAGES) & 1);
  }
}

template <typename T, int DP, int NT, bool WIN>
cudaError_t launch(const PagedParams& p, cudaStream_t st) {
  using C = Cfg<DP, NT>;
  KParams kp{};
  kp.p = p;
  auto map = [&](CUtensorMap* m, const void* base, int64_t page, int64_t head, int64_t slot) {
    return tma::make_map_view(m, base, Elem<T>::is_bf16, p.dim, p.page_size, (int64_t)p.kv_heads * p.num_pages,
                              View{slot > 0 ? slot : p.dim, head, page, 0}, p.kv_heads, p.num_pages, p.box_rows);
  };
  if (!map(&kp.tm_k, p.k, p.k_page, p.k_head, p.k_slot) || !map(&kp.tm_v, p.v, p.v_page, p.v_head, p.v_slot))
    return cudaErrorInvalidValue;
  auto kern = paged_decode_kernel<T, DP, NT, WIN>;
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = allow_smem(kern, C::SMEM, ready);
  if (e != cudaSuccess) return e;
  e = launch_early(kern, p.blocks, 32 * kWarps, C::SMEM, st, kp);
  if (e != cudaSuccess || p.whole_items) return e;
  // the join starts while the last blocks still run and waits on the device for what they wrote
  return launch_early(paged_join_kernel<T, DP, NT>, (int64_t)p.batch * p.join_blocks, 512, 0, st, p);
}

template <typename T, bool WIN>
cudaError_t launch_dim(const PagedParams& p, cudaStream_t st) {
  if (p.cols == 128) return p.nt == 2 ? launch<T, 128, 2, WIN>(p, st) : launch<T, 128, 1, WIN>(p, st);
  return p.nt == 2 ? launch<T, 64, 2, WIN>(p, st) : launch<T, 64, 1, WIN>(p, st);
}

}  // namespace

void paged_plan(PagedParams& p) {
  p.group = p.heads / p.kv_heads;
  p.nt = p.group > 8 ? 2 : 1;  // 8 or 16 query heads share a pass over their keys
  p.chunks = (p.group + 8 * p.nt - 1) / (8 * p.nt);
  p.items = p.kv_heads * p.chunks;
  p.join_blocks = (int64_t)p.batch * p.heads <= 4 * 148 ? p.heads : p.items;  // four blocks of 512 threads an SM
  const int64_t tile = p.k_scale ? kPagedTile8 : kTile, warp_rows = tile / kWarps;
  p.box_rows = std::gcd((int)warp_rows, p.page_size);
  // (a copy's place in shared memory is a multiple of 128 bytes, so boxes of one row of 8-bit values take 128 columns)
  int bits = 0;  // 2^(bits - 1) < page_size <= 2^bits; the quotient's excess, below 2^-31, never reaches a whole number
  while ((int64_t(1) << bits) < p.page_size) ++bits;
  p.page_shift = 31 + bits;
  p.page_magic = (uint32_t)(((uint64_t(1) << p.page_shift) + p.page_size - 1) / p.page_size);
  p.cols = p.dim > 64 || (p.k_scale && p.box_rows == 1) ? 128 : 64;
  int64_t tiles = (p.max_len + tile - 1) / tile;  // most that an item can have
  if (p.window) tiles = std::min(tiles, (p.sinks + tile - 1) / tile + (p.window + warp_rows - 1 + tile - 1) / tile);
  // 8-bit: three blocks an SM with rings of two stages hide the ends of many items, two with three stages keep more copies in
  // flight over few long ones (512 items of 64 sequences: 38.3 us with three, 41.1 with two; 12 items of up to 262143 tokens:
  // 54.1 and 51.7); 16 heads need the registers of two. Up to 64 columns four
  // fit (the same calls at D = 64, before small weights took products of their own: 25.5 and 34.9 us with four, 29.8 with three and 41.9 with
  // two; with them 25.9 and 35.9 with four)
  p.per_sm = !p.k_scale || p.nt == 2 ? 2 : p.cols == 64 ? 4 : (int64_t)p.batch * p.items >= 2 * 148 ? 3 : 2;
  // An item stays whole where its tiles cost no more than the cut with its join, which is about six of them where few items leave
  // blocks free, and more where fewer are (half of the tiles, for lengths differ). D = 128, us, whole and cut: 2 items
  // of 257 tokens 8.3 and 10.8 in 16 bits, of 513 12.6 and 10.9, in 8 bits of 513 9.2 and 11.6, of 1025 13.9 and 11.6; 256 items of
  // 513 tokens 14.9 and 19.7, 11.4 and 17.4. The join's launch and the workspace cost the host 5 beside that.
  const int64_t count = (int64_t)p.batch * p.items, room = p.per_sm * 148;
  p.whole_items = tiles <= kMinTiles || (count <= room && tiles * (2 * room - count) <= 12 * room);
  p.blocks = p.whole_items ? count : room;
}

int64_t paged_workspace(const PagedParams& p) {
  if (p.whole_items) return 0;
  const int64_t rows = p.blocks * 2 * 8 * p.nt;
  return rows * p.cols * 4 + rows * 2 * 4 + (int64_t)p.batch * p.items * (int64_t)sizeof(int2);
}

cudaError_t paged_decode(PagedParams p, void* workspace, bool bf16, cudaStream_t st) {
  p.part = static_cast<float*>(workspace);
  p.part_ml = p.part + p.blocks * 2 * 8 * p.nt * p.cols;
  p.cuts = reinterpret_cast<int2*>(p.part_ml + p.blocks * 2 * 8 * p.nt * 2);
  if (p.k_scale) return paged_decode8(p, bf16, st);
  if (p.window) return bf16 ? launch_dim<__nv_bfloat16, true>(p, st) : launch_dim<__half, true>(p, st);
  return bf16 ? launch_dim<__nv_bfloat16, false>(p, st) : launch_dim<__half, false>(p, st);
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
