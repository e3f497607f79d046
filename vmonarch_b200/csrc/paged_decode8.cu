// Attention of one new token per sequence over a paged cache of e4m3 values with a scale for each page and head
// (paged_decode.cu has the 16-bit form and the definitions; with a window WIN).
//
//   o = sum_t p_t vs_t v_t / sum_t p_t,  p_t = exp(sm_scale ks_t q . k_t - m),
// where ks_t and vs_t are the scales of token t's page. Half the bytes a token, and so half the time that a block may spend on
// one: a warp owns 32 tokens of every tile (the loop, the looking up of pages and the softmax's bookkeeping are paid per
// 32), each lane looks up one token's page and copies its two scales, and the softmax keeps its reference until a score
// passes the one that set it by more than 2^8, which a vote over the warp says without a maximum over lanes.
//
// Operands. ldmatrix moves pairs of bytes: it leaves a lane with four neighbouring columns of a key (a permutation of the
// contraction index, in which the queries are loaded too) and, transposed, with two neighbouring columns of two tokens (a
// byte permutation; V^T's rows are then 2 r and 2 r + 1 where the 16-bit form has r and r + 8). e4m3 converts to fp16 exactly, so
// the products are fp16 for bf16 queries too: a row of those is scaled by the power of two that brings its largest element
// below 2^15, which loses nothing above 2^-29 of it. The key scale multiplies the score. The value scale goes into the exponent: the sum takes
// 2^(x - m), the product P = 2^(x + log2 vs - m'), each against a reference of its own, so that pages of any scales meet in one
// 32-bit accumulator; the end of an item brings the accumulators from m' to m. A column in which the largest weights meet small or no
// values is the sum of small ones, so these keep their bits: the references stay 2^7 below the largest score, which puts fp16's
// normal numbers at 2^-21 of the largest weight, and a warp with a weight below that takes the tile's product in bf16, in which
// e4m3 is exact too, with P as the sum of two bf16 values. (GPU time with fp16 alone, of calls without such weights and where every
// tile has some: 64 sequences of up to 8192 tokens, 40/8 heads, D = 128: 95.2 us, 96.5 and 108; 3 of up to 262143, 16/4 heads: 71.9, 73.3
// and 85.5. Weights sorted by size into fp16 products with factors of their own: 146 and 116 at scores of 8 nats' deviation.)
//
// Waits for a stage are bounded as in paged_decode.cu.
#include "paged_tiles.cuh"
#include "sm100.cuh"
#include "tma_host.h"

namespace vmb {

__device__ int g_paged8_err;

namespace {

using namespace sm100;

constexpr int kTile = kPagedTile8;
constexpr int kRows = kTile / kWarps;  // tokens of a tile that a warp owns
// A reference is raised, to 2^-kLift of the largest score, once a score passes it by more than 2^kRaise: P <= 2^15, inside fp16, and the
// score that set it is passed by 2^(kRaise - kLift).
constexpr float kLift = 7.f, kRaise = 15.f;
// Exponents between which a weight is too small for fp16's normal numbers, but not for 32 bits.
constexpr float kLeast = -14.f, kNone = -126.f;
static_assert(kRows == 32, "a lane a token");

template <int DP, int NT, int BLOCKS>
struct Cfg {
  static constexpr int STAGES = DP == 128 ? (BLOCKS == 3 ? 2 : 3) : BLOCKS == 4 ? 3 : 6;
  static constexpr int MAT = kRows * DP;             // a warp's keys or values: rows of DP bytes, swizzled
  static constexpr int STAGE = 2 * MAT;
  static constexpr int RING = kWarps * STAGES * STAGE;
  static constexpr int LD = DP + 4;                  // joined accumulators: 4 heads per warp at a time
  static constexpr int JOIN = kWarps * 4 * LD * 4 + kWarps * 4 * 2 * 4;  // accumulators, (max, sum)
  static constexpr int SCALES = kWarps * STAGES * 2 * kRows * 4;
  static constexpr int SMEM = RING + JOIN + SCALES + kWarps * STAGES * 8 + 32;  // + barriers, abort flag, the share's numbers
  static_assert(BLOCKS * (SMEM + 1024) <= 233472, "shared memory of an SM");
};

// Two e4m3 values (the low or high half of x) as two fp16, exactly.
__device__ __forceinline__ uint32_t f16x2_lo(uint32_t x) {
  uint32_t y;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t f16x2_hi(uint32_t x) {
  uint32_t y;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(y) : "r"(x));
  return y;
}
// 4 bytes from global to shared memory, or zeros.
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ float lds(uint32_t at) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at));
  return x;
}
// Byte offset of 16-byte chunk c of row r: a 128- or 64-byte swizzle, as the copies write it.
template <int DP>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return DP == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

struct KParams {
  // boxes of DP columns x box_rows slots (a multiple of 128 bytes: paged_plan); coordinates (column, slot, head, page, 0)
  CUtensorMap tm_k, tm_v;
  PagedParams p;
};

template <typename T, int DP, int NT, bool WIN, int BLOCKS>
__global__ void __launch_bounds__(32 * kWarps, BLOCKS) paged_decode8_kernel(const __grid_constant__ KParams kp) {
  using C = Cfg<DP, NT, BLOCKS>;
  constexpr int KS = DP / 16;
  constexpr int HEADS = 8 * NT;
  const PagedParams& p = kp.p;
  extern __shared__ __align__(1024) uint8_t smem[];  // everything shared is in here, so that it starts on a swizzle atom
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(smem) + warp * C::STAGES * C::STAGE;
  float* join = reinterpret_cast<float*>(smem + C::RING);          // [warp][4 heads][LD]
  float* join_ml = join + kWarps * 4 * C::LD;                       // [warp][4 heads][max, sum]
  const uint32_t scales = smem_u32(smem + C::RING + C::JOIN) + warp * C::STAGES * 2 * kRows * 4;  // [stage][K, V][token]
  const uint32_t bar0 = smem_u32(smem + C::RING + C::JOIN + C::SCALES) + 8u * warp * C::STAGES;
  volatile int* abort = reinterpret_cast<int*>(smem + C::RING + C::JOIN + C::SCALES + kWarps * C::STAGES * 8);
  // units of all, blocks that take part
  long long* share = reinterpret_cast<long long*>(smem + C::RING + C::JOIN + C::SCALES + kWarps * C::STAGES * 8 + 8);

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
  // ---- loading. Lane i stands for token i of the warp's rows; the first of box_rows lanes issues their keys and values.
  Cursor lc = cc;
  if (p.hold_loads && warp == 0) lc.left = 0;
  int issued = 0;
  int page, slot;  // of this lane's token of the stage that is issued next
  // of the item that is loaded: its key head, page table row and scales
  int head;
  const int32_t* table;
  const float *k_scales, *v_scales;
  auto enter = [&]() {
    head = lc.item / p.chunks;
    table = p.table + (int64_t)lc.seq * p.table_stride;
    k_scales = p.k_scale + head * p.ks_head;
    v_scales = p.v_scale + head * p.vs_head;
  };
  auto look_up = [&](const Cursor& c) {
    const int t = c.token<WIN, kTile>() + kRows * warp + lane;
    page = p.num_pages;  // outside the map: zeros
    slot = 0;
    // (of a group that the window cuts all of the rows are loaded)
    bool wanted = t < c.len;
    if (WIN) wanted = wanted && (sees(c, t) || (t & ~(p.box_rows - 1)) + p.box_rows > c.len - p.window);
    if (wanted) {
      const int i = (int)((uint64_t)t * p.page_magic >> p.page_shift);
      slot = t - i * p.page_size;
      page = table[i];
      if ((unsigned)page >= (unsigned)p.num_pages) page = p.num_pages;
    }
  };
  auto issue = [&](int it) {  // stage it % STAGES <- this warp's rows of lc, then on to the next tile
    if (lc.left > 0) {
      const int s = it % C::STAGES;
      const uint32_t st = ring + s * C::STAGE, bar = bar0 + 8u * s, sc = scales + s * 2 * kRows * 4 + 4 * lane;
      if (lane == 0) mbar_expect_tx(bar, C::STAGE);
      ++issued;
      __syncwarp();
      if ((lane & (p.box_rows - 1)) == 0) {
        tma_load(st + lane * DP, &kp.tm_k, 0, slot, BIdx(head, page, 0), bar);
        tma_load(st + C::MAT + lane * DP, &kp.tm_v, 0, slot, BIdx(head, page, 0), bar);
      }
      const bool valid = page < p.num_pages;
      const int from = valid ? page : 0;
      cp_async4(sc, k_scales + from * p.ks_page, valid);
      cp_async4(sc + 4 * kRows, v_scales + from * p.vs_page, valid);
      advance<WIN, kTile>(p, lc);
      if (lc.left > 0) {
        if (lc.tile == 0) enter();
        look_up(lc);
      }
    }
    cp_async_commit();  // a group a stage, also behind the last
  };
  if (lc.left > 0) {
    enter();
    look_up(lc);
  }
#pragma unroll
  for (int s = 0; s < C::STAGES - 1; ++s) issue(s);

  uint32_t qf[NT][KS][2];
  float acc[NT][KS][4], m[NT][2], mv[NT][2], l[NT][2];  // mv: the accumulators' reference
  float qs[NT][2];                                       // what a score is multiplied with, for heads 2 (lane % 4) and + 1
  // an item's query heads as B fragments (head = lane / 4, columns 4 (lane % 4) ...): loaded, and once they are there, scaled
  auto load_q = [&](const Cursor& c) {
    const int h = c.item / p.chunks, g0 = (c.item % p.chunks) * HEADS;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int g = g0 + 8 * nt + lane / 4;
      const T* q = static_cast<const T*>(p.q) + (int64_t)c.seq * p.q_row + (int64_t)(h * p.group + g) * p.q_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int col = 16 * ks + 4 * (lane % 4);
        const uint2 x = g < p.group && col < p.dim ? *reinterpret_cast<const uint2*>(q + col) : make_uint2(0u, 0u);
        qf[nt][ks][0] = x.x;
        qf[nt][ks][1] = x.y;
      }
    }
  };
  auto scale_q = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float factor = 1.f;
      if (Elem<T>::is_bf16) {
        float top = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const float2 a = Elem<T>::unpack(qf[nt][ks][0]), b = Elem<T>::unpack(qf[nt][ks][1]);
          top = fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))), top);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = (int)(__float_as_uint(top) >> 23) - 127;  // top < 2^(e + 1); 128: not finite
        const int up = top == 0.f || e == 128 ? 0 : min(14 - e, 126);
        factor = __uint_as_float((uint32_t)(127 - up) << 23);
        const float by = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 a = Elem<T>::unpack(qf[nt][ks][i]);
            qf[nt][ks][i] = Elem<__half>::pack(a.x * by, a.y * by);
          }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) qs[nt][i] = p.scale_log2 * __shfl_sync(0xffffffffu, factor, 4 * (2 * (lane % 4) + i));
    }
  };
  auto clear = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][ks][e] = 0.f;
      m[nt][0] = m[nt][1] = mv[nt][0] = mv[nt][1] = -1e30f;
      l[nt][0] = l[nt][1] = 0.f;
    }
  };
  bool from_start = cc.tile == 0, ok = true;
  if (cc.left > 0) {
    load_q(cc);
    scale_q();
  }
  clear();
  for (int it = 0; cc.left > 0; ++it) {
    if (ok && !__all_sync(0xffffffffu, mbar_wait(bar0 + 8u * (it % C::STAGES), (it / C::STAGES) & 1, abort, &g_paged8_err, 1,
                                                 p.wait_limit))) {
      ok = false;  // no more loads and products, but on to the barriers that the block's warps share
      lc.left = 0;
    }
    cp_async_wait<C::STAGES - 2>();  // this stage's scales
    __syncwarp();
    const uint32_t ks_base = ring + (it % C::STAGES) * C::STAGE, vs_base = ks_base + C::MAT;
    // the tokens that take part, a bit each
    const uint32_t rows = __ballot_sync(0xffffffffu, ok && sees(cc, cc.token<WIN, kTile>() + kRows * warp + lane));
    if (rows) {
      if (rows != 0xffffffffu) {  // slots without one: their values enter the product with weight 0
        for (int i = lane; i < kRows * DP / 16; i += 32) {
          const int r = i / (DP / 16);
          if (!((rows >> r) & 1u))
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vs_base + i * 16), "r"(0) : "memory");
        }
        fence_proxy_async_smem();  // the next copy into this stage comes through the async proxy
        __syncwarp();
      }
      // rows lane / 4 + 8 i of the 32: scales of keys, logarithms of those of values
      float k_by[4], v_log[4];
      const uint32_t sc = scales + (it % C::STAGES) * 2 * kRows * 4 + lane / 4 * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        k_by[i] = lds(sc + 32 * i);
        v_log[i] = fast_log2(lds(sc + 4 * kRows + 32 * i));
      }
      float s[NT][2][4];  // [16 tokens]
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][0][e] = s[nt][1][e] = 0.f;
#pragma unroll
      for (int k2 = 0; k2 < KS / 2; ++k2)
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 16 columns of rows 0-7, 8-15 of the half, the next 16 of them
          uint32_t x[4];
          ldsm_x4(ks_base + chunk_at<DP>(16 * h + (lane & 15), 2 * k2 + (lane >> 4)), x[0], x[1], x[2], x[3]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t a[4] = {f16x2_lo(x[2 * e]), f16x2_lo(x[2 * e + 1]), f16x2_hi(x[2 * e]), f16x2_hi(x[2 * e + 1])};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<__half>(s[nt][h], a, qf[nt][2 * k2 + e][0], qf[nt][2 * k2 + e][1]);
          }
        }
      float y[NT][4][2];  // scores that weigh the values, with their scale, then the weights
      bool wide = false;  // whether some of these are too small for fp16
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        // i: rows lane / 4 + 8 i; e: heads 2 (lane % 4) + e
        float x[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            x[i][e] = s[nt][i >> 1][(i & 1) * 2 + e] * (qs[nt][e] * k_by[i]);
            y[nt][i][e] = x[i][e] + v_log[i];
          }
        if (rows != 0xffffffffu) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!((rows >> (lane / 4 + 8 * i)) & 1u)) x[i][0] = y[nt][i][0] = x[i][1] = y[nt][i][1] = -INFINITY;
        }
        float mx[2], my[2], al[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = fmaxf(fmaxf(x[0][e], x[1][e]), fmaxf(x[2][e], x[3][e]));
          my[e] = fmaxf(fmaxf(y[nt][0][e], y[nt][1][e]), fmaxf(y[nt][2][e], y[nt][3][e]));
        }
        const bool above = fmaxf(fmaxf(mx[0] - m[nt][0], my[0] - mv[nt][0]), fmaxf(mx[1] - m[nt][1], my[1] - mv[nt][1])) > kRaise;
        float least[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) least[e] = fminf(fminf(y[nt][0][e], y[nt][1][e]), fminf(y[nt][2][e], y[nt][3][e])) - mv[nt][e];
        if (__any_sync(0xffffffffu, above || fminf(least[0], least[1]) < kLeast)) {
          if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int w = 4; w < 32; w <<= 1) {
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], w));
                my[e] = fmaxf(my[e], __shfl_xor_sync(0xffffffffu, my[e], w));
              }
              const float mn = fmaxf(m[nt][e], mx[e] - kLift), vn = fmaxf(mv[nt][e], my[e] - kLift);
              l[nt][e] *= fast_exp2(m[nt][e] - mn);
              al[e] = fast_exp2(mv[nt][e] - vn);
              m[nt][e] = mn;
              mv[nt][e] = vn;
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[nt][ks][e] *= al[e & 1];
          }
          bool low = false;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) low |= y[nt][i][e] - mv[nt][e] < kLeast && y[nt][i][e] - mv[nt][e] >= kNone;
          wide |= __any_sync(0xffffffffu, low);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[nt][e] += (fast_exp2(x[0][e] - m[nt][e]) + fast_exp2(x[1][e] - m[nt][e])) +
                      (fast_exp2(x[2][e] - m[nt][e]) + fast_exp2(x[3][e] - m[nt][e]));
#pragma unroll
          for (int i = 0; i < 4; ++i) y[nt][i][e] = fast_exp2(y[nt][i][e] - mv[nt][e]);
        }
      }
      auto times_values = [&](auto type) {  // acc += V^T P, in products of that type; bf16: P as the sum of two values
        using M = decltype(type);
        constexpr int PARTS = Elem<M>::is_bf16 ? 2 : 1;
        uint32_t pb[PARTS][NT][2][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t p0 = Elem<M>::pack(y[nt][i][0], y[nt][i][1]);
            pb[0][nt][i >> 1][i & 1] = movmatrix(p0);
            if (PARTS == 2) {
              const float2 f = Elem<M>::unpack(p0);
              pb[PARTS - 1][nt][i >> 1][i & 1] = movmatrix(Elem<M>::pack(y[nt][i][0] - f.x, y[nt][i][1] - f.y));
            }
          }
#pragma unroll
        for (int k2 = 0; k2 < KS / 2; ++k2)
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // 16 columns of tokens 0-7, 8-15 of the half, the next 16 of them
            uint32_t x[4];
            ldsm_x4_t(vs_base + chunk_at<DP>(16 * h + (lane & 15), 2 * k2 + (lane >> 4)), x[0], x[1], x[2], x[3]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              // columns (2 r, 2 r + 1) of two tokens -> two tokens of column 2 r, two of 2 r + 1
              const uint32_t lo = __byte_perm(x[2 * e], 0, 0x3120), hi = __byte_perm(x[2 * e + 1], 0, 0x3120);
              uint32_t a[4] = {f16x2_lo(lo), f16x2_hi(lo), f16x2_lo(hi), f16x2_hi(hi)};
              if (Elem<M>::is_bf16) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float2 f = Elem<__half>::unpack(a[i]);
                  a[i] = Elem<M>::pack(f.x, f.y);
                }
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < PARTS; ++i) mma16816<M>(acc[nt][2 * k2 + e], a, pb[i][nt][h][0], pb[i][nt][h][1]);
            }
          }
      };
      if (wide) times_values(__nv_bfloat16());
      else times_values(__half());
    }
    __syncwarp();  // every lane is done with the stage that the next issue refills
    issue(it + C::STAGES - 1);

    const Cursor done = cc;
    advance<WIN, kTile>(p, cc);
    const bool to_end = cc.tile == 0;
    if (to_end || cc.left <= 0) {
      // ---- the four warps' parts of this item (or of this block's share of it)
      // sums and accumulators to the reference m + kLift, the largest score that raised it; the latter's factor in two parts, for scales
      // near the ends of their range would take it out of its own
      float to_m[NT][2][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          m[nt][e] += kLift;
          l[nt][e] *= fast_exp2(-kLift);
          const float by = mv[nt][e] - m[nt][e], half = rintf(0.5f * by);
          to_m[nt][e][0] = fast_exp2(half);
          to_m[nt][e][1] = fast_exp2(by - half);
        }
      if (cc.left > 0) load_q(cc);  // of the next item, on its way meanwhile
      const int h = done.item / p.chunks, g0 = (done.item % p.chunks) * HEADS;
      const bool whole = from_start && to_end;
      if (from_start && !p.whole_items && threadIdx.x == 0)
        p.cuts[(int64_t)done.seq * p.items + done.item] = whole ? make_int2(-1, 0) : cut_behind(share[0], share[1], cc.tiles - cc.tile);
      const int64_t part = (int64_t)blockIdx.x * 2 + (from_start ? 1 : 0);
#pragma unroll
      for (int round = 0; round < 2 * NT; ++round) {  // heads 8 nt + 2 r + e, r < 4
        const int nt = round >> 1, e = round & 1;
        if (g0 + 8 * nt + e >= p.group) break;
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
        if (lane < 4) *reinterpret_cast<float2*>(join_ml + (warp * 4 + lane) * 2) = make_float2(m[nt][e], l[nt][e]);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          *reinterpret_cast<float2*>(join + (warp * 4 + lane % 4) * C::LD + 16 * ks + 2 * (lane / 4)) =
              make_float2(acc[nt][ks][e] * to_m[nt][e][0] * to_m[nt][e][1], acc[nt][ks][2 + e] * to_m[nt][e][0] * to_m[nt][e][1]);
        __syncthreads();
        for (int i = threadIdx.x; i < 4 * DP; i += 32 * kWarps) {
          const int r = i / DP, d = i % DP, in = 8 * nt + 2 * r + e, g = g0 + in;
          if (g >= p.group) break;  // rows only grow
          float mm = -1e30f, sum = 0.f, o = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, join_ml[(w * 4 + r) * 2]);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float f = fast_exp2(join_ml[(w * 4 + r) * 2] - mm);
            sum = fmaf(f, join_ml[(w * 4 + r) * 2 + 1], sum);
            o = fmaf(f, join[(w * 4 + r) * C::LD + d], o);
          }
          const int64_t head = h * p.group + g;
          if (whole) {
            if (d < p.dim) static_cast<T*>(p.o)[(int64_t)done.seq * p.o_row + head * p.o_head + d] =
                Elem<T>::from_f(sum == 0.f ? 0.f : o / sum);
            if (d == 0 && p.lse) p.lse[(int64_t)done.seq * p.heads + head] = sum == 0.f ? -INFINITY : (mm + log2f(sum)) * kLn2;
          } else {
            p.part[(part * HEADS + in) * DP + d] = o;
            if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (part * HEADS + in) * 2) = make_float2(mm, sum);
          }
        }
        __syncthreads();
      }
      if (cc.left > 0) scale_q();
      clear();
      from_start = true;
    }
  }
  cp_async_wait<0>();
  if (!ok) {  // a stage did not arrive in time: the copies under way must land before the block ends
    for (int i = max(issued - C::STAGES, 0); i < issued; ++i) mbar_wait_drain(bar0 + 8u * (i % C::STAGES), (i / C::STAGES) & 1);
  }
}

template <typename T, int DP, int NT, bool WIN, int BLOCKS>
cudaError_t launch(const PagedParams& p, cudaStream_t st) {
  using C = Cfg<DP, NT, BLOCKS>;
  KParams kp{};
  kp.p = p;
  auto map = [&](CUtensorMap* m, const void* base, int64_t page, int64_t head, int64_t slot) {
    return tma::make_map5(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, base, p.dim, p.page_size, (int64_t)p.kv_heads * p.num_pages,
                          View{slot > 0 ? slot : p.dim, head, page, 0}, p.kv_heads, p.num_pages, DP, p.box_rows,
                          DP == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
  };
  if (!map(&kp.tm_k, p.k, p.k_page, p.k_head, p.k_slot) || !map(&kp.tm_v, p.v, p.v_page, p.v_head, p.v_slot))
    return cudaErrorInvalidValue;
  auto kern = paged_decode8_kernel<T, DP, NT, WIN, BLOCKS>;
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = allow_smem(kern, C::SMEM, ready);
  if (e != cudaSuccess) return e;
  e = launch_early(kern, p.blocks, 32 * kWarps, C::SMEM, st, kp);
  if (e != cudaSuccess || p.whole_items) return e;
  return launch_early(paged_join_kernel<T, DP, NT>, (int64_t)p.batch * p.join_blocks, 512, 0, st, p);
}

template <typename T, bool WIN>
cudaError_t launch_dim(const PagedParams& p, cudaStream_t st) {
  if (p.nt == 2) return p.cols == 128 ? launch<T, 128, 2, WIN, 2>(p, st) : launch<T, 64, 2, WIN, 2>(p, st);
  if (p.cols == 64) return launch<T, 64, 1, WIN, 4>(p, st);
  return p.per_sm == 3 ? launch<T, 128, 1, WIN, 3>(p, st) : launch<T, 128, 1, WIN, 2>(p, st);
}

}  // namespace

cudaError_t paged_decode8(const PagedParams& p, bool bf16, cudaStream_t st) {
  if (p.window) return bf16 ? launch_dim<__nv_bfloat16, true>(p, st) : launch_dim<__half, true>(p, st);
  return bf16 ? launch_dim<__nv_bfloat16, false>(p, st) : launch_dim<__half, false>(p, st);
}

cudaError_t paged8_status(cudaStream_t st, int* out) {
  int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(out, g_paged8_err, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && *out) e = cudaMemcpyToSymbolAsync(g_paged8_err, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  return e;
}

}  // namespace vmb
