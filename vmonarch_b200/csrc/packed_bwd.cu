// Attention over packed sequences of different lengths, backward, on tcgen05 / TMA (packed_fwd.cu has
// the forward and its definitions).
//
//   P_ij = exp(s_ij - lse_i), D_i = sum_c o_ic do_ic, dS_ij = sm_scale P_ij (do_i . v_j - D_i)
//   dV_j = sum_i P_ij do_i,   dK_j = sum_i dS_ij q_i,   dQ_i = sum_j dS_ij k_j
// with the sums over i running over every query head that shares the key head. Three kernels, no
// atomics, so the gradients are the same from run to run:
//
// pre   one row per half-warp: nl = -lse log2(e) and nc = -sm_scale D in planes [head][stat_rows], in
//       which every sequence starts at a multiple of 128 (rows past its end: P = 0), and the mean
//       of the sequence's first keys for dq. Then
//       P = 2^(s c + nl) and dS = P (sm_scale dP + nc): two packed FMAs, one exponential, one product.
//       D takes o with the 16 bits that its rounding left out (o_low): an error of D is shared by a
//       whole row of dS, so it does not average out in dQ_i = sum_j dS_ij k_j where keys have a mean
//       (4000 causal queries, D = 128, bf16: dQ off by 4.1e-3 without it, 2.4e-3 with it, of which its
//       own rounding is 1.7e-3). The forward's rounding of P is in o all the same, and so in D.
// dkdv  CTA = 128 keys of one key head; walks (query head, 64-query tile): S^T = K Q^T and
//       dP^T = V dO^T (SS), P^T and dS^T (16-bit) back to TMEM over them, dV += P^T dO and
//       dK += dS^T Q (TS). thread = key row; two streams of tiles, two warpgroups each. P^T is handed over before dS^T is
//       formed, so that dV and the stream's next S^T run meanwhile (1765 -> 1678 us in the case below). Larger query
//       tiles would make better products (N = 64 runs at 70 % of the rate of N = 128), but two streams of them
//       need 768 columns of TMEM.
//       TMEM: stream b S^T [128b, +64) dP^T [128b + 64, +64), dK [256, +64 NA), dV after it.
// dq    CTA = 128 queries of one head; walks 128-key tiles: S, dP (SS), dS over S, dQ += dS K (TS).
//       thread = query row x 32 keys. A row of dS sums to zero, its rounded values do not quite, and what they
//       leave would weigh the mean that keys share: dQ_i = sum_j dS_ij (k_j - c) for any c, so the sum of the
//       rounded values times the mean of the sequence's first keys is taken off at the end (15600 causal queries
//       around a mean of 0.3, D = 128, bf16: error of dQ 1.49 -> 1.43 times that of its own rounding).
//       TMEM: S0 [0,128) S1 [128,256) dP [256,384) dQ [384, +64 NA).
// A query that sees one key has dS = 0 by its index, where dP - D would leave a rounding.
// Seven products per tile pair instead of five: above D = 64 TMEM cannot hold S, dP, dK, dV and dQ of one tile at
// once, and recomputing S and dP costs less than adding dQ through memory in 32 bits. (Neither dS kept in memory in 16
// bits for dQ nor the 128 columns that are idle up to D = 64 have been tried here.)
// Bound by the tensor products (operands from shared memory) and the latencies between them. 15600 + 1289 + 409 + 1
// causal tokens, 16/4 heads, D = 128, bf16: pre 48 us, dkdv 1650 us (1.22 PFLOP/s of its four products), dq 1160 us
// (1.30 PFLOP/s of its three), 2720 us with the set-ups overlapped; five products at the measured dense rate (1.67 PFLOP/s) would take 1500 us.
//
// Tiles at a sequence's end hold the next sequence's rows. Their scores are dropped by index, and the
// rows that enter a sum with weight 0 (Q and dO here, K in dq) are cleared in shared memory first, so
// that nothing another sequence holds (0 x inf) gets into it. P and dS are 16-bit operands of the tensor
// cores; sums, statistics and accumulators are 32-bit.
#include <type_traits>

#include "common.cuh"
#include "launch.h"
#include "packed.h"
#include "sm100.cuh"
#include "tma_host.h"

namespace vmb {

__device__ int g_packed_bwd_err;

namespace {

using namespace sm100;

constexpr int kAtom = 128 * 128;  // 128 rows x 128 B
constexpr int kAtom64 = 64 * 128;
constexpr int kThreads = 64 + 128 * 4;  // producer, MMA issuer, four compute warpgroups

struct KParams {
  CUtensorMap tm_q, tm_k, tm_v, tm_do;  // dkdv: Q, dO boxes of 64 rows; dq: all of 128
  PackedParams a;
  float scale_log2;
};

// Below 2^-14 fp16 loses bits, which P of a few thousand keys, and dS of small dO, would reach: P is held as 2^8 P, and
// dS as 2^8 s dS with the power of two s that brings sm_scale |dO| into (2^-6, 2^-5], of a row in dq, of the largest of
// the rows that meet in one dK in dkdv. |2^8 s dS| <= 2^8 2^-5 2 |v| stays in range while |v| < 4094; 16000 keys of
// |v| = sqrt(D) lie around 2^-12 (14061 keys, D = 96: errors of dQ and dK 1.51 and 1.53 -> 1.42 and 1.44 times those of
// their own rounding). bf16 has the range, s = 1.
template <typename T>
constexpr float kPScale = Elem<T>::is_bf16 ? 1.f : 256.f;
constexpr float kMaxScale = 1152921504606846976.f;  // 2^60, the scale of rows that need none

// P and dS of two scores, packed to 16 bits.
__device__ __forceinline__ float2 prob2(uint32_t s0, uint32_t s1, float2 sc2, float2 nl2) {
  const float2 t = __ffma2_rn(make_float2(__uint_as_float(s0), __uint_as_float(s1)), sc2, nl2);
  return make_float2(fast_exp2(t.x), fast_exp2(t.y));
}
__device__ __forceinline__ float2 dscore2(float2 p, uint32_t d0, uint32_t d1, float2 sm2, float2 nc2) {
  return __fmul2_rn(p, __ffma2_rn(make_float2(__uint_as_float(d0), __uint_as_float(d1)), sm2, nc2));
}

// Rows [first, rows) of `atoms` consecutive swizzle atoms of `rows` x 128 B, cleared by nthreads threads.
__device__ __forceinline__ void clear_rows(uint32_t base, int atoms, int rows, int first, int tid, int nthreads) {
  const int n = (rows - first) * 8;
  for (int i = tid; i < n * atoms; i += nthreads) {
    const int a = i / n, rem = i - a * n;
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + a * rows * 128 + (first + (rem >> 3)) * 128 +
                                                                 (rem & 7) * 16),
                 "r"(0)
                 : "memory");
  }
}

// Columns [32 c, +32) of an accumulator row: scale (acc - off * centre[column]); zeros where nothing was added.
__device__ __forceinline__ void result_row(uint32_t taddr, int c, bool any, float scale, float off, const float* centre,
                                           uint32_t (&v)[32]) {
  if (any) {
    tmem_ld32(taddr + c * 32, v);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 m = centre ? *reinterpret_cast<const float4*>(centre + 32 * c + i) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[i] = __float_as_uint(fmaf(-off, m.x, __uint_as_float(v[i])) * scale);
      v[i + 1] = __float_as_uint(fmaf(-off, m.y, __uint_as_float(v[i + 1])) * scale);
      v[i + 2] = __float_as_uint(fmaf(-off, m.z, __uint_as_float(v[i + 2])) * scale);
      v[i + 3] = __float_as_uint(fmaf(-off, m.w, __uint_as_float(v[i + 3])) * scale);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = 0u;
  }
}
// 32-column chunks [c0, c1) of an accumulator row to a row of 16-bit values.
template <typename T>
__device__ __forceinline__ void store_result(uint32_t taddr, T* out, bool live, bool sectors, int dim, bool any, int c0, int c1,
                                             float scale, float off = 0.f, const float* centre = nullptr) {
#pragma unroll 1
  for (int c = c0; c < c1; ++c) {
    uint32_t v[32], x[16];
    result_row(taddr, c, any, scale, off, centre, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = Elem<T>::pack(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
    if (live) store_row32(reinterpret_cast<uint16_t*>(out), c * 32, dim, sectors, x);
  }
}

// 32-column chunks [c0, c1) of an accumulator row to a cut unit's 32-bit partial.
__device__ __forceinline__ void store_part(uint32_t taddr, float* to, bool any, int c0, int c1, float scale, float off = 0.f,
                                           const float* centre = nullptr) {
#pragma unroll 1
  for (int c = c0; c < c1; ++c) {
    uint32_t v[32];
    result_row(taddr, c, any, scale, off, centre, v);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      *reinterpret_cast<uint4*>(to + c * 32 + 4 * k) = make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
  }
}

// Adds the pieces of cut units in order: block = (unit, head, matrix, 32 rows), 8 lanes a row, 8 NA columns a
// lane. KV: dK and dV of key units, else dQ of query units. Partials [part][head][matrix][128][64 NA].
template <typename T, int NA, bool KV>
__global__ void __launch_bounds__(256) packed_sum_kernel(const __grid_constant__ PackedParams a) {
  wait_for_kernel_before();
  let_next_kernel_start();
  constexpr int MATS = KV ? 2 : 1;
  const int heads = KV ? a.kv_heads : a.heads;
  int64_t b = blockIdx.x;
  const int rows0 = (int)(b & 3) * 32;
  b >>= 2;
  const int mat = (int)(b % MATS);
  b /= MATS;
  const int head = (int)(b % heads), join = (int)(b / heads);
  const PackedUnit u = a.units[a.joins[2 * join]];
  const int pieces = a.joins[2 * join + 1];
  const int row = rows0 + (threadIdx.x >> 3), sub = threadIdx.x & 7;
  if (row >= (KV ? u.k_valid : u.q_valid)) return;
  float o[8 * NA];
#pragma unroll
  for (int i = 0; i < 8 * NA; ++i) o[i] = 0.f;
#pragma unroll 2
  for (int k = 0; k < pieces; ++k) {
    const float4* v = reinterpret_cast<const float4*>(
        a.part + ((((int64_t)(u.part + k) * heads + head) * MATS + mat) * 128 + row) * (64 * NA) + sub * 8 * NA);
#pragma unroll
    for (int i = 0; i < 2 * NA; ++i) {
      const float4 x = v[i];
      o[4 * i] += x.x;
      o[4 * i + 1] += x.y;
      o[4 * i + 2] += x.z;
      o[4 * i + 3] += x.w;
    }
  }
  const View& v = !KV ? a.dqv : mat ? a.dvv : a.dkv;
  T* out = static_cast<T*>(!KV ? a.dq : mat ? a.dv : a.dk) + ((KV ? u.k_row : u.q_row) + row) * v.rs + head * v.s1;
#pragma unroll
  for (int g = 0; g < NA; ++g) {
    const int col = sub * 8 * NA + 8 * g;
    if (col < a.dim)
      *reinterpret_cast<uint4*>(out + col) =
          make_uint4(Elem<T>::pack(o[8 * g], o[8 * g + 1]), Elem<T>::pack(o[8 * g + 2], o[8 * g + 3]),
                     Elem<T>::pack(o[8 * g + 4], o[8 * g + 5]), Elem<T>::pack(o[8 * g + 6], o[8 * g + 7]));
  }
}

// ------------------------------------------------------------------------------------ statistics
// Block = one 128-query unit of one head; 16 lanes per row, 16 bytes each of o and dO.
template <typename T>
__global__ void __launch_bounds__(256) packed_pre_kernel(const __grid_constant__ PackedParams a) {
  __shared__ float4 sums[16][32];
  __shared__ float least[16];
  wait_for_kernel_before();
  let_next_kernel_start();
  const UnitHead uh = unit_of_block(blockIdx.x, a.n_units, a.heads, a.heads);
  const PackedUnit u = a.units[uh.unit];
  const int head = uh.head, sub = threadIdx.x & 15;
  float* nl = a.stats + (int64_t)head * a.stat_rows + u.stat_row;
  float* nc = nl + (int64_t)a.heads * a.stat_rows;
  float* ns = nc + (int64_t)a.heads * a.stat_rows;
  if (head % a.group == 0) {
    // the mean of up to 128 first keys of the unit's sequence (for dq)
    const int keys = min(u.k_valid, 128), kvh = head / a.group;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
    if (sub * 8 < a.dim) {
      const T* k = static_cast<const T*>(a.k) + (int64_t)u.k_row * a.kv.rs + (int64_t)kvh * a.kv.s1 + sub * 8;
#pragma unroll 8
      for (int r = threadIdx.x >> 4; r < keys; r += 16) {
        const uint4 x = *reinterpret_cast<const uint4*>(k + (int64_t)r * a.kv.rs);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 v = Elem<T>::unpack(xs[i]);
          f[2 * i] += v.x;
          f[2 * i + 1] += v.y;
        }
      }
    }
    sums[threadIdx.x >> 4][2 * sub] = make_float4(f[0], f[1], f[2], f[3]);
    sums[threadIdx.x >> 4][2 * sub + 1] = make_float4(f[4], f[5], f[6], f[7]);
    __syncthreads();
    if (threadIdx.x < 128) {
      float s = 0.f;
#pragma unroll
      for (int g = 0; g < 16; ++g) s += reinterpret_cast<const float*>(sums[g])[threadIdx.x];
      a.centre[((int64_t)kvh * (a.stat_rows >> 7) + (u.stat_row >> 7)) * 128 + threadIdx.x] = keys > 0 ? s / (float)keys : 0.f;
    }
  }
  float low = kMaxScale;
#pragma unroll 2
  for (int r = threadIdx.x >> 4; r < 128; r += 16) {
    const bool valid = r < u.q_valid;
    float d = 0.f, norm = 0.f;
    if (valid && sub * 8 < a.dim) {
      const int64_t row = u.q_row + r;
      auto load = [&](const void* t, const View& v) {
        return *reinterpret_cast<const uint4*>(static_cast<const T*>(t) + row * v.rs + head * v.s1 + sub * 8);
      };
      const uint4 x = load(a.o, a.ov), w = load(a.o_low, a.olv), y = load(a.dout, a.dov);
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ws[4] = {w.x, w.y, w.z, w.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = Elem<T>::unpack(xs[i]), l = Elem<T>::unpack(ws[i]), g = Elem<T>::unpack(ys[i]);
        d = fmaf(f.x + l.x, g.x, fmaf(f.y + l.y, g.y, d));
        norm = fmaf(g.x, g.x, fmaf(g.y, g.y, norm));
      }
    }
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) {
      d += __shfl_xor_sync(0xffffffffu, d, s);
      if (!Elem<T>::is_bf16) norm += __shfl_xor_sync(0xffffffffu, norm, s);
    }
    if (!Elem<T>::is_bf16) {
      // rows without a gradient and those past the end do not count
      const float size = a.sm_scale * sqrtf(norm);
      const float s = valid && size > 0.f && isfinite(size) ? exp2f(fminf(fmaxf(-5.f - ceilf(log2f(size)), -60.f), 60.f))
                                                            : kMaxScale;
      low = fminf(low, s);
      if (sub == 0) ns[r] = s;
    }
    if (sub == 0) {
      // finite, so that a row without keys and the rows past the end have P = 2^(finite - 1e30) = 0
      const float lse = valid ? a.lse[(int64_t)head * a.q_total + u.q_row + r] : -INFINITY;
      nl[r] = lse == -INFINITY ? -1e30f : fmaf(-lse, kLog2e, Elem<T>::is_bf16 ? 0.f : 8.f);
      nc[r] = valid ? -a.sm_scale * d : 0.f;
    }
  }
  if (!Elem<T>::is_bf16) {
    if (sub == 0) least[threadIdx.x >> 4] = low;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int g = 1; g < 16; ++g) low = fminf(low, least[g]);
      a.tile_scale[(int64_t)head * (a.stat_rows >> 7) + (u.stat_row >> 7)] = low;
    }
  }
}

// ------------------------------------------------------------------------------------ dK, dV
template <int NA>
struct DkdvCfg {
  static constexpr int RES = 2 * NA * kAtom;         // K | V
  static constexpr int SLOT_T = 2 * NA * kAtom64;    // Q | dO of 64 queries
  static constexpr int SLOT = SLOT_T + 1024;         // + nl, nc (256 B each)
  static constexpr int NQ = NA == 2 ? 4 : 8;
  static constexpr int SMEM = 1024 + RES + NQ * SLOT;
  static_assert(SMEM <= 232448 - 1024, "shared memory budget");
};

template <typename T, int NA>
__global__ void __launch_bounds__(kThreads, 1) packed_dkdv_kernel(const __grid_constant__ KParams p) {
  using C = DkdvCfg<NA>;
  constexpr int NQ = C::NQ;
  constexpr bool kBf16 = Elem<T>::is_bf16;
  constexpr uint32_t IDESC_SP = idesc_f16(kBf16, 128, 64, false, false);        // S^T, dP^T
  constexpr uint32_t IDESC_ACC = idesc_f16(kBf16, 128, 64 * NA, false, true);   // dK, dV (B MN-major)
  constexpr uint32_t T_DK = 256, T_DV = 256 + 64 * NA;
  // column of the packed P^T / dS^T of queries [16 kk, +16) inside a tile's S^T / dP^T: a warpgroup
  // writes inside the 32 columns that it loaded itself
  auto pcol = [](int kk) -> uint32_t { return 32 * (kk >> 1) + 8 * (kk & 1); };

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[10 + 2 * NQ];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_sh;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sK = sbase, sV = sbase + NA * kAtom, sSlots = sbase + C::RES;
  auto sQ = [&](int s) { return sSlots + s * C::SLOT; };
  auto sDO = [&](int s) { return sSlots + s * C::SLOT + NA * kAtom64; };
  auto sStat = [&](int s) { return sSlots + s * C::SLOT + C::SLOT_T; };
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t BAR_KV = bar0, BAR_DONE = bar0 + 8u;
  auto BAR_S = [&](int b) { return bar0 + 8u * (2 + b); };
  auto BAR_DP = [&](int b) { return bar0 + 8u * (4 + b); };
  auto BAR_P = [&](int b) { return bar0 + 8u * (6 + b); };
  auto BAR_DS = [&](int b) { return bar0 + 8u * (8 + b); };
  auto BAR_QFULL = [&](int s) { return bar0 + 8u * (10 + s); };
  auto BAR_QEMPTY = [&](int s) { return bar0 + 8u * (10 + NQ + s); };
  volatile int* abort = &abort_sh;

  if (threadIdx.x == 0) {
    abort_sh = 0;
    mbar_init(BAR_KV, 1);
    mbar_init(BAR_DONE, 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(BAR_S(b), 1);
      mbar_init(BAR_DP(b), 1);
      mbar_init(BAR_P(b), 256);
      mbar_init(BAR_DS(b), 256);
    }
    for (int s = 0; s < NQ; ++s) {
      mbar_init(BAR_QFULL(s), 1);
      mbar_init(BAR_QEMPTY(s), 1);
    }
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(&tmem_base_sh), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;
  wait_for_kernel_before();
  let_next_kernel_start();

  const UnitHead uh = unit_of_block(blockIdx.x, p.a.n_units, p.a.kv_heads, p.a.head_chunk);
  const PackedUnit u = p.a.units[uh.unit];
  const int kvh = uh.head;
  const int t_first = max(u.vis0, 0) >> 6;
  const int per_head = max(((u.q_valid + 63) >> 6) - t_first, 1);  // tiles of one query head
  const int n = u.end - u.begin;
  // step i -> query head and first local query of its tile
  auto step_head = [&](int i) { return kvh * p.a.group + (u.begin + i) / per_head; };
  auto step_q0 = [&](int i) { return (t_first + (u.begin + i) % per_head) * 64; };

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    if (lane == 0 && n > 0 && !p.a.hold_loads) {
      int armed[NQ];
      for (int s = 0; s < NQ; ++s) armed[s] = 0;
      prefetch_tmap(&p.tm_q);
      prefetch_tmap(&p.tm_do);
      mbar_expect_tx(BAR_KV, C::RES);
      for (int x = 0; x < NA; ++x) {
        tma_load(sK + x * kAtom, &p.tm_k, 64 * x, u.k_row, BIdx(kvh, 0, 0), BAR_KV);
        tma_load(sV + x * kAtom, &p.tm_v, 64 * x, u.k_row, BIdx(kvh, 0, 0), BAR_KV);
      }
      for (int i = 0; i < n; ++i) {
        const int s = i % NQ;
        if (i >= NQ && !mbar_wait(BAR_QEMPTY(s), ((i / NQ) - 1) & 1, abort, &g_packed_bwd_err, 1, p.a.wait_limit)) break;
        const int h = step_head(i), q0 = step_q0(i);
        mbar_expect_tx(BAR_QFULL(s), C::SLOT_T + 512);
        for (int x = 0; x < NA; ++x) {
          tma_load(sQ(s) + x * kAtom64, &p.tm_q, 64 * x, u.q_row + q0, BIdx(h, 0, 0), BAR_QFULL(s));
          tma_load(sDO(s) + x * kAtom64, &p.tm_do, 64 * x, u.q_row + q0, BIdx(h, 0, 0), BAR_QFULL(s));
        }
        const float* st = p.a.stats + (int64_t)h * p.a.stat_rows + u.stat_row + q0;
        bulk_load(sStat(s), st, 256, BAR_QFULL(s));
        bulk_load(sStat(s) + 256, st + (int64_t)p.a.heads * p.a.stat_rows, 256, BAR_QFULL(s));
        if (i + NQ < n) {  // the tile one ring ahead into L2
          const int ha = step_head(i + NQ), qa = u.q_row + step_q0(i + NQ);
          for (int x = 0; x < NA; ++x) {
            tma_prefetch(&p.tm_q, 64 * x, qa, BIdx(ha, 0, 0));
            tma_prefetch(&p.tm_do, 64 * x, qa, BIdx(ha, 0, 0));
          }
        }
        armed[s] = i / NQ + 1;
      }
      mbar_wait_drain(BAR_KV, 0);
      for (int s = 0; s < NQ; ++s)
        if (armed[s] > 0) mbar_wait_drain(BAR_QFULL(s), (armed[s] - 1) & 1);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    const uint32_t leader = elect_one() ? 1u : 0u;
    auto wwait = [&](uint32_t bar, uint32_t parity, int code) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, &g_packed_bwd_err, code, p.a.wait_limit));
    };
    // S^T = K Q^T or dP^T = V dO^T of step i, whose slot has landed
    auto issue = [&](int i, bool dp) {
      const uint32_t tb = tmem + 128 * (i & 1) + (dp ? 64 : 0), sa = dp ? sV : sK, sb = dp ? sDO(i % NQ) : sQ(i % NQ);
#pragma unroll
      for (int kk = 0; kk < 4 * NA; ++kk) {
        const uint32_t oa = (kk >> 2) * kAtom + (kk & 3) * 32, ob = (kk >> 2) * kAtom64 + (kk & 3) * 32;
        mma_ss_if(leader, tb, smem_desc_sw128(sa + oa, 16, 1024), smem_desc_sw128(sb + ob, 16, 1024), IDESC_SP, kk > 0);
      }
      mma_commit_if(leader, dp ? BAR_DP(i & 1) : BAR_S(i & 1));
    };
    auto landed = [&](int i) -> bool {
      if (!wwait(BAR_QFULL(i % NQ), (i / NQ) & 1, 2)) return false;
      tc_fence_after();
      return true;
    };
    bool ok = n <= 0 || wwait(BAR_KV, 0, 2);
    for (int i = 0; ok && i < min(n, 2); ++i) {
      if (!(ok = landed(i))) break;
      issue(i, false);
      issue(i, true);
    }
    // A stream's S^T of step i + 2 runs while its warps still work on dS^T of step i, its dP^T while they work on P^T
    for (int i = 0; ok && i < n; ++i) {
      const int s = i % NQ;
      const uint32_t pt = tmem + 128 * (i & 1), dst = pt + 64;
      if (!wwait(BAR_P(i & 1), (i >> 1) & 1, 4)) break;
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)  // dV += P^T dO over 64 queries
        mma_ts_if(leader, tmem + T_DV, pt + pcol(kk), smem_desc_sw128(sDO(s) + kk * 2048, kAtom64, 1024), IDESC_ACC,
                  (i > 0 || kk > 0) ? 1u : 0u);
      if (i + 2 < n) {
        if (!landed(i + 2)) break;
        issue(i + 2, false);
      }
      if (!wwait(BAR_DS(i & 1), (i >> 1) & 1, 4)) break;
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)  // dK += dS^T Q
        mma_ts_if(leader, tmem + T_DK, dst + pcol(kk), smem_desc_sw128(sQ(s) + kk * 2048, kAtom64, 1024), IDESC_ACC,
                  (i > 0 || kk > 0) ? 1u : 0u);
      mma_commit_if(leader, BAR_QEMPTY(s));
      if (i + 2 < n) issue(i + 2, true);
    }
    if (elect_one()) {
      mma_commit(BAR_DONE);
      mbar_wait_drain(BAR_DONE, 0);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- compute: thread = key row
    const int wg = (warp - 2) >> 2;
    const int stm = wg >> 1, half = wg & 1;  // stream (step parity), 32-query half of its tiles
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const int tid = (wg & 1) * 128 + (threadIdx.x - 64) % 128;  // within the stream's 256 threads
    auto warp_wait = [&](uint32_t bar, uint32_t parity, int code) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, &g_packed_bwd_err, code, p.a.wait_limit));
    };
    const uint32_t ts = tmem + lane_off + 128 * stm, tdp = ts + 64;
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2), sm2 = make_float2(p.a.sm_scale, p.a.sm_scale);
    float ds_scale = 1.f;  // fp16: of all the rows that meet in this unit's dK
    if (!kBf16) {
      const int tiles = (u.q_valid + 127) >> 7;
      ds_scale = kMaxScale;
      for (int i = lane; i < tiles * p.a.group; i += 32)
        ds_scale = fminf(ds_scale, p.a.tile_scale[((int64_t)kvh * p.a.group + i / tiles) * (p.a.stat_rows >> 7) +
                                                  (u.stat_row >> 7) + i % tiles]);
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) ds_scale = fminf(ds_scale, __shfl_xor_sync(0xffffffffu, ds_scale, x));
    }
    const float2 ss2 = make_float2(ds_scale, ds_scale);
    bool ok = true;
    for (int i = stm; i < n; i += 2) {
      const int s = i % NQ;
      if (!warp_wait(BAR_S(stm), (i >> 1) & 1, 8) || !warp_wait(BAR_QFULL(s), (i / NQ) & 1, 8)) { ok = false; break; }
      tc_fence_after();
      const int q0 = step_q0(i), left = u.q_valid - q0;
      // key `row` is seen by the tile's queries [c_lo, left)
      const bool masked = left < 64 || u.vis0 + 127 > q0 || u.lone > q0;
      const int c_lo = u.vis0 + row - q0 - 32 * half, c_hi = left - 32 * half;
      if (left < 64) {
        // S^T is complete, and what dP^T still reads only goes into queries past the end: clear for dK and dV
        clear_rows(sQ(s), 2 * NA, 64, left, tid, 256);
        fence_proxy_async_smem();
      }
      const uint32_t st = sStat(s) + 128 * half;
      float2 pr[16];  // P^T of the thread's 32 queries
      auto p_phase = [&](auto mask) {
        uint32_t sv[32], pk[16];
        tmem_ld32(ts + 32 * half, sv);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float4 l4;
          asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(l4.x), "=f"(l4.y), "=f"(l4.z), "=f"(l4.w) : "r"(st + 4 * e));
          float2 p0 = prob2(sv[e], sv[e + 1], sc2, make_float2(l4.x, l4.y));
          float2 p1 = prob2(sv[e + 2], sv[e + 3], sc2, make_float2(l4.z, l4.w));
          if (mask) {
            if (e < c_lo || e >= c_hi) p0.x = 0.f;
            if (e + 1 < c_lo || e + 1 >= c_hi) p0.y = 0.f;
            if (e + 2 < c_lo || e + 2 >= c_hi) p1.x = 0.f;
            if (e + 3 < c_lo || e + 3 >= c_hi) p1.y = 0.f;
          }
          pk[e >> 1] = Elem<T>::pack(p0.x, p0.y);
          pk[(e >> 1) + 1] = Elem<T>::pack(p1.x, p1.y);
          pr[e >> 1] = kBf16 ? p0 : __fmul2_rn(p0, ss2);
          pr[(e >> 1) + 1] = kBf16 ? p1 : __fmul2_rn(p1, ss2);
        }
        tmem_st16(ts + pcol(2 * half), pk);
      };
      if (masked) p_phase(std::true_type{});
      else p_phase(std::false_type{});
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(BAR_P(stm));
      if (!warp_wait(BAR_DP(stm), (i >> 1) & 1, 8)) { ok = false; break; }
      tc_fence_after();
      const int d_lo = max(c_lo, u.lone - q0 - 32 * half);
      auto ds_phase = [&](int h, auto mask) {
        uint32_t dv[16], dk[8];
        tmem_ld16(tdp + 32 * half + 16 * h, dv);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          float4 c4;
          asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                       : "=f"(c4.x), "=f"(c4.y), "=f"(c4.z), "=f"(c4.w)
                       : "r"(st + 256 + 64 * h + 4 * e));
          float2 d0 = dscore2(pr[8 * h + (e >> 1)], dv[e], dv[e + 1], sm2, make_float2(c4.x, c4.y));
          float2 d1 = dscore2(pr[8 * h + (e >> 1) + 1], dv[e + 2], dv[e + 3], sm2, make_float2(c4.z, c4.w));
          if (mask) {
            const int c = 16 * h + e;
            if (c < d_lo || c >= c_hi) d0.x = 0.f;
            if (c + 1 < d_lo || c + 1 >= c_hi) d0.y = 0.f;
            if (c + 2 < d_lo || c + 2 >= c_hi) d1.x = 0.f;
            if (c + 3 < d_lo || c + 3 >= c_hi) d1.y = 0.f;
          }
          dk[e >> 1] = Elem<T>::pack(d0.x, d0.y);
          dk[(e >> 1) + 1] = Elem<T>::pack(d1.x, d1.y);
        }
        tmem_st8(tdp + pcol(2 * half + h), dk);
      };
      if (masked) {
        ds_phase(0, std::true_type{});
        ds_phase(1, std::true_type{});
      } else {
        ds_phase(0, std::false_type{});
        ds_phase(1, std::false_type{});
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(BAR_DS(stm));
    }
    if (ok) ok = warp_wait(BAR_DONE, 0, 8);
    tc_fence_after();
    // epilogue: warpgroups 0, 1 take dK, 2, 3 dV, half of the columns each
    const int mat = wg >> 1;
    const float unscale = (mat ? 1.f : 1.f / ds_scale) / kPScale<T>;
    ok = named_bar_and(1, 512, ok && !*abort);
    const uint32_t acc = tmem + lane_off + (mat ? T_DV : T_DK);
    if (ok && u.part >= 0) {
      store_part(acc, p.a.part + ((((int64_t)u.part * p.a.kv_heads + kvh) * 2 + mat) * 128 + row) * (64 * NA), n > 0,
                 (wg & 1) * NA, ((wg & 1) + 1) * NA, unscale);
    } else if (ok) {
      const View& v = mat ? p.a.dvv : p.a.dkv;
      T* out = static_cast<T*>(mat ? p.a.dv : p.a.dk);
      store_result<T>(acc, out + (int64_t)(u.k_row + row) * v.rs + (int64_t)kvh * v.s1, row < u.k_valid, whole_sectors(out, v),
                      p.a.dim, n > 0, (wg & 1) * NA, ((wg & 1) + 1) * NA, unscale);
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------------------------ dQ
template <int NA>
struct DqCfg {
  static constexpr int TILE = NA * kAtom;
  static constexpr int NK = NA == 2 ? 3 : 5, NV = NA == 2 ? 2 : 4;
  static constexpr int SMEM = 1024 + (2 + NK + NV) * TILE;
  static_assert(SMEM <= 232448 - 1024, "shared memory budget");
};

template <typename T, int NA>
__global__ void __launch_bounds__(kThreads, 1) packed_dq_kernel(const __grid_constant__ KParams p) {
  using C = DqCfg<NA>;
  constexpr int NK = C::NK, NV = C::NV;
  constexpr uint32_t TILE = C::TILE;
  constexpr bool kBf16 = Elem<T>::is_bf16;
  constexpr uint32_t IDESC_S = idesc_f16(kBf16, 128, 128, false, false);
  constexpr uint32_t IDESC_DQ = idesc_f16(kBf16, 128, 64 * NA, false, true);
  constexpr uint32_t T_DP = 256, T_DQ = 384;
  constexpr int B_Q = 0, B_DONE = 1, B_S = 2, B_DS = 4, B_DP = 6, B_DPFREE = 7, B_KFULL = 8, B_KEMPTY = B_KFULL + NK,
                B_VFULL = B_KEMPTY + NK, B_VEMPTY = B_VFULL + NV, NBARS = B_VEMPTY + NV;

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[NBARS];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_sh;
  __shared__ __align__(16) float centre_sh[64 * NA];  // mean of the sequence's first keys

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sQ = sbase, sDO = sbase + TILE, sK = sbase + 2 * TILE, sV = sK + NK * TILE;
  const uint32_t bar0 = smem_u32(bars);
  auto BAR = [&](int i) { return bar0 + 8u * (uint32_t)i; };
  volatile int* abort = &abort_sh;

  if (threadIdx.x == 0) {
    abort_sh = 0;
    for (int i = 0; i < NBARS; ++i)
      mbar_init(BAR(i), i == B_DS || i == B_DS + 1 || i == B_DPFREE ? 512 : 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(&tmem_base_sh), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;
  wait_for_kernel_before();
  let_next_kernel_start();

  const UnitHead uh = unit_of_block(blockIdx.x, p.a.n_units, p.a.heads, p.a.head_chunk);
  const PackedUnit u = p.a.units[uh.unit];
  const int head = uh.head, kvh = head / p.a.group;
  auto limit = [&](int r) { return max(0, min(u.k_valid, p.a.causal ? u.vis0 + r : u.k_valid)); };
  const int n = u.end - u.begin;

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producers: lane 0 Q, dO, K; lane 1 V
    if (lane < 2 && n > 0 && !p.a.hold_loads) {
      const bool kl = lane == 0;
      const int nslot = kl ? NK : NV;
      const CUtensorMap* map = kl ? &p.tm_k : &p.tm_v;
      prefetch_tmap(map);
      if (kl) {
        mbar_expect_tx(BAR(B_Q), 2 * TILE);
        for (int x = 0; x < NA; ++x) {
          tma_load(sQ + x * kAtom, &p.tm_q, 64 * x, u.q_row, BIdx(head, 0, 0), BAR(B_Q));
          tma_load(sDO + x * kAtom, &p.tm_do, 64 * x, u.q_row, BIdx(head, 0, 0), BAR(B_Q));
        }
      }
      int armed[NK > NV ? NK : NV];
      for (int s = 0; s < nslot; ++s) armed[s] = 0;
      for (int j = 0; j < n; ++j) {
        const int s = j % nslot;
        if (j >= nslot && !mbar_wait(BAR((kl ? B_KEMPTY : B_VEMPTY) + s), ((j / nslot) - 1) & 1, abort, &g_packed_bwd_err, 16, p.a.wait_limit))
          break;
        const uint32_t full = BAR((kl ? B_KFULL : B_VFULL) + s);
        const int row = u.k_row + (u.begin + j) * 128;
        mbar_expect_tx(full, TILE);
        for (int x = 0; x < NA; ++x)
          tma_load((kl ? sK : sV) + s * TILE + x * kAtom, map, 64 * x, row, BIdx(kvh, 0, 0), full);
        if (j + nslot < n)
          for (int x = 0; x < NA; ++x) tma_prefetch(map, 64 * x, row + nslot * 128, BIdx(kvh, 0, 0));
        armed[s] = j / nslot + 1;
      }
      if (kl) mbar_wait_drain(BAR(B_Q), 0);
      for (int s = 0; s < nslot; ++s)
        if (armed[s] > 0) mbar_wait_drain(BAR((kl ? B_KFULL : B_VFULL) + s), (armed[s] - 1) & 1);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    const uint32_t leader = elect_one() ? 1u : 0u;
    auto wwait = [&](int bar, uint32_t parity, int code) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(BAR(bar), parity, abort, &g_packed_bwd_err, code, p.a.wait_limit));
    };
    auto issue = [&](int j, bool dp) -> bool {  // S(j) = Q K^T, or dP(j) = dO V^T
      const int s = dp ? j % NV : j % NK;
      if (!wwait((dp ? B_VFULL : B_KFULL) + s, (j / (dp ? NV : NK)) & 1, 32)) return false;
      tc_fence_after();
      const uint32_t ab = dp ? sDO : sQ, bb = (dp ? sV : sK) + s * TILE;
      const uint32_t d = dp ? tmem + T_DP : tmem + 128u * (uint32_t)(j & 1);
#pragma unroll
      for (int kk = 0; kk < 4 * NA; ++kk) {
        const uint32_t off = (kk >> 2) * kAtom + (kk & 3) * 32;
        mma_ss_if(leader, d, smem_desc_sw128(ab + off, 16, 1024), smem_desc_sw128(bb + off, 16, 1024), IDESC_S, kk > 0);
      }
      mma_commit_if(leader, BAR(dp ? B_DP : B_S + (j & 1)));
      if (dp) mma_commit_if(leader, BAR(B_VEMPTY + s));
      return true;
    };
    bool ok = n <= 0 || wwait(B_Q, 0, 32);
    if (ok && n > 0) ok = issue(0, false) && issue(0, true);
    if (ok && n > 1) ok = issue(1, false);
    for (int j = 0; ok && j < n; ++j) {
      if (j + 1 < n && (!wwait(B_DPFREE, j & 1, 64) || !issue(j + 1, true))) break;
      if (!wwait(B_DS + (j & 1), (j >> 1) & 1, 64)) break;
      tc_fence_after();
      const uint32_t kb = sK + (j % NK) * TILE, sb = tmem + 128u * (uint32_t)(j & 1);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)  // dQ += dS K; keys [16 kk, +16) of warpgroup kk / 2
        mma_ts_if(leader, tmem + T_DQ, sb + 32 * (kk >> 1) + 8 * (kk & 1), smem_desc_sw128(kb + kk * 2048, kAtom, 1024),
                  IDESC_DQ, (j > 0 || kk > 0) ? 1u : 0u);
      mma_commit_if(leader, BAR(B_KEMPTY + j % NK));
      if (j + 2 < n) ok = issue(j + 2, false);
    }
    if (elect_one()) {
      mma_commit(BAR(B_DONE));
      mbar_wait_drain(BAR(B_DONE), 0);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- compute: thread = query row x 32 keys
    const int wg = (warp - 2) >> 2;
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const int tid = threadIdx.x - 64;
    const float* stat = p.a.stats + (int64_t)head * p.a.stat_rows + u.stat_row + row;
    const int64_t plane = (int64_t)p.a.heads * p.a.stat_rows;
    const float row_scale = kBf16 ? 1.f : stat[2 * plane];
    const int my_lim = limit(row), lim_lo = limit(0);
    const float ds_scale = my_lim > 1 ? row_scale : 0.f;  // a softmax over one key has no gradient
    const float fl = stat[0], fc = stat[plane] * ds_scale, fs = p.a.sm_scale * ds_scale;
    const float2 nl2 = make_float2(fl, fl), nc2 = make_float2(fc, fc);
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2), sm2 = make_float2(fs, fs);
    auto warp_wait = [&](int bar, uint32_t parity, int code) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(BAR(bar), parity, abort, &g_packed_bwd_err, code, p.a.wait_limit));
    };
    if (tid < 64 * NA) centre_sh[tid] = p.a.centre[((int64_t)kvh * (p.a.stat_rows >> 7) + (u.stat_row >> 7)) * 128 + tid];
    float sum = 0.f;  // of this thread's rounded dS
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      if (!warp_wait(B_S + (j & 1), (j >> 1) & 1, 64) || !warp_wait(B_DP, j & 1, 64)) { ok = false; break; }
      tc_fence_after();
      const int k0 = (u.begin + j) * 128;
      const uint32_t ts = tmem + lane_off + 128u * (uint32_t)(j & 1) + 32 * wg;
      uint32_t sv[32], dv[32], pk[16];
      tmem_ld32(ts, sv);
      tmem_ld32(tmem + lane_off + T_DP + 32 * wg, dv);
      tmem_wait_ld();
      tc_fence_before();
      mbar_arrive(BAR(B_DPFREE));
      if (u.k_valid - k0 < 128) {  // S(j) is complete: only dQ still reads the key tile
        clear_rows(sK + (j % NK) * TILE, NA, 128, u.k_valid - k0, tid, 512);
        fence_proxy_async_smem();
      }
      const bool masked = lim_lo - k0 < 128;
      const int valid = my_lim - k0 - 32 * wg;
      auto scores = [&](auto mask) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float2 d = dscore2(prob2(sv[e], sv[e + 1], sc2, nl2), dv[e], dv[e + 1], sm2, nc2);
          if (mask) {
            if (e >= valid) d.x = 0.f;
            if (e + 1 >= valid) d.y = 0.f;
          }
          pk[e >> 1] = Elem<T>::pack(d.x, d.y);
        }
      };
      if (masked) scores(std::true_type{});
      else scores(std::false_type{});
      tmem_st16(ts, pk);
      float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        s0 = __fadd2_rn(s0, Elem<T>::unpack(pk[e]));
        s1 = __fadd2_rn(s1, Elem<T>::unpack(pk[e + 1]));
      }
      sum += (s0.x + s1.x) + (s0.y + s1.y);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(BAR(B_DS + (j & 1)));
    }
    // by warpgroup and row, over the dO tile: every dP has been read by now
    float* sums = reinterpret_cast<float*>(smem_raw + (sDO - smem_u32(smem_raw)));
    if (ok) sums[wg * 128 + row] = sum;
    if (ok) ok = warp_wait(B_DONE, 0, 64);
    tc_fence_after();
    // epilogue: a warpgroup takes 32 columns
    ok = named_bar_and(1, 512, ok && !*abort);
    if (ok && wg < 2 * NA) {
      const float unscale = 1.f / (row_scale * kPScale<T>);
      const float off = (sums[row] + sums[128 + row]) + (sums[256 + row] + sums[384 + row]);
      T* out = static_cast<T*>(p.a.dq);
      if (u.part >= 0)
        store_part(tmem + lane_off + T_DQ, p.a.part + (((int64_t)u.part * p.a.heads + head) * 128 + row) * (64 * NA), n > 0, wg,
                   wg + 1, unscale, off, centre_sh);
      else
        store_result<T>(tmem + lane_off + T_DQ, out + (int64_t)(u.q_row + row) * p.a.dqv.rs + (int64_t)head * p.a.dqv.s1,
                        row < u.q_valid, whole_sectors(out, p.a.dqv), p.a.dim, n > 0, wg, wg + 1, unscale, off, centre_sh);
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

template <typename Kern>
cudaError_t run(Kern kern, int smem, std::atomic<uint64_t>& ready, int64_t blocks, const KParams& p, cudaStream_t st) {
  cudaError_t e = allow_smem(kern, smem, ready);
  if (e != cudaSuccess) return e;
  return launch_early(kern, blocks, kThreads, smem, st, p);
}

template <typename T, int NA>
cudaError_t launch(const PackedParams& dq, const PackedParams& kv, cudaStream_t st) {
  constexpr bool bf16 = Elem<T>::is_bf16;
  if (dq.n_units > 0) {
    // pieces of a cut unit write the same values
    cudaError_t e = launch_early(packed_pre_kernel<T>, (int64_t)dq.n_units * dq.heads, 256, 0, st, dq);
    if (e != cudaSuccess) return e;
  }
  static std::atomic<uint64_t> ready_kv{0}, ready_q{0};
  KParams p{};
  p.scale_log2 = dq.sm_scale * kLog2e;
  auto map = [&](CUtensorMap* m, const void* base, int64_t rows, int heads, const View& v, int box) {
    return rows == 0 || tma::make_map_view(m, base, bf16, dq.dim, rows, heads, v, heads, 1, box);
  };
  if (!map(&p.tm_k, dq.k, dq.k_total, dq.kv_heads, dq.kv, 128) || !map(&p.tm_v, dq.v, dq.k_total, dq.kv_heads, dq.vv, 128))
    return cudaErrorInvalidValue;
  if (kv.n_units > 0) {
    if (!map(&p.tm_q, kv.q, kv.q_total, kv.heads, kv.qv, 64) || !map(&p.tm_do, kv.dout, kv.q_total, kv.heads, kv.dov, 64))
      return cudaErrorInvalidValue;
    p.a = kv;
    cudaError_t e = run(packed_dkdv_kernel<T, NA>, DkdvCfg<NA>::SMEM, ready_kv, (int64_t)kv.n_units * kv.kv_heads, p, st);
    if (e != cudaSuccess) return e;
    if (kv.n_joins > 0 &&
        (e = launch_early(packed_sum_kernel<T, NA, true>, (int64_t)kv.n_joins * kv.kv_heads * 8, 256, 0, st, kv)) != cudaSuccess)
      return e;
  }
  if (dq.n_units > 0) {
    if (!map(&p.tm_q, dq.q, dq.q_total, dq.heads, dq.qv, 128) || !map(&p.tm_do, dq.dout, dq.q_total, dq.heads, dq.dov, 128))
      return cudaErrorInvalidValue;
    p.a = dq;
    cudaError_t e = run(packed_dq_kernel<T, NA>, DqCfg<NA>::SMEM, ready_q, (int64_t)dq.n_units * dq.heads, p, st);
    if (e != cudaSuccess) return e;
    if (dq.n_joins > 0) return launch_early(packed_sum_kernel<T, NA, false>, (int64_t)dq.n_joins * dq.heads * 4, 256, 0, st, dq);
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t packed_bwd(const PackedParams& dq, const PackedParams& kv, bool bf16, cudaStream_t st) {
  if (dq.dim > 64) return bf16 ? launch<__nv_bfloat16, 2>(dq, kv, st) : launch<__half, 2>(dq, kv, st);
  return bf16 ? launch<__nv_bfloat16, 1>(dq, kv, st) : launch<__half, 1>(dq, kv, st);
}

cudaError_t packed_bwd_status(cudaStream_t st, int* out) {
  int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(out, g_packed_bwd_err, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && *out) e = cudaMemcpyToSymbolAsync(g_packed_bwd_err, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  return e;
}

}  // namespace vmb
