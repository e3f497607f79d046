// Attention over packed sequences of different lengths, forward, on tcgen05 / TMA (head dims up to
// 128, multiples of 8; grouped heads; causal or not).
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(s_ij - m_i),  s_ij = sm_scale q_i . k_j,
// over the keys j of query i's own sequence that it sees: all of them, or with `causal` the first
// nk - nq + i + 1 (the last query sees the last key). A query that sees no key has o = 0 and
// lse = -inf.
//
// CTA = one head and one unit of up to 256 queries (two 128-row tiles, one per softmax warpgroup) of
// one sequence. 10 warps: TMA producer, MMA issuer, two warpgroups of softmax and epilogue, thread =
// query row. The two streams walk the same ring of 128-key tiles and never wait for one another, so
// one's exponentials run beside the other's matrix products. Online softmax with a lazily raised
// reference: the exponentials of an unmasked tile go against the current reference and are redone
// only when a 64-key half's sum passes 2^14. P is 16-bit (the rounding the tensor cores need; l sums
// the unrounded p), everything else 32-bit.
// TMEM (512 columns): S_0 [0,128), S_1 [128,256), O_0 [256, +64 NA), O_1 [256 + 64 NA, +64 NA).
//
// The sequences share one tensor, so a tile's rows past the sequence end are the next sequence's.
// Scores past the end (or after the diagonal) are dropped by index. A value row that no query of the
// tile sees enters P V with p = 0, and 0 x inf = NaN, so in a tile that is masked for some row the
// threads look the value tile over (one multiply by zero per pair) and clear what is not finite;
// the epilogue then adds those values back, from global memory, to the queries that do see them.
//
// Head dims below 64 NA load as zeros past the tensor's columns (TMA) and store only their own.
#include "common.cuh"
#include "launch.h"
#include "packed.h"
#include "sm100.cuh"
#include "tma_host.h"

namespace vmb {

__device__ int g_packed_err;

namespace {

using namespace sm100;

constexpr int kAtom = 128 * 128;  // one swizzle atom column block: 128 rows x 128 B
constexpr int kThreads = 320;
constexpr float kRescaleThreshold = 8.0f;
constexpr float kSumThreshold = 16384.0f;

struct KParams {
  CUtensorMap tm_q, tm_k, tm_v;
  PackedParams a;
  float scale_log2;
};

template <int NA>
struct Cfg {
  static constexpr int TILE = NA * kAtom;
  static constexpr int NK = NA == 2 ? 3 : 5, NV = NA == 2 ? 2 : 4;
  static constexpr int SMEM = 1024 + (2 + NK + NV) * TILE;
  static_assert(SMEM <= 232448 - 1024, "shared memory budget");
  static_assert(NK + NV >= 4, "the epilogue stages O and what its rounding leaves, both streams, in the rings");
};

__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int N, bool MASK>
__device__ __forceinline__ float row_max(const uint32_t (&sr)[N], int valid) {
  auto at = [&](int i) { return (MASK && i >= valid) ? -1e30f : __uint_as_float(sr[i]); };
  float mr[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) mr[k] = fmax3(at(3 * k), at(3 * k + 1), at(3 * k + 2));
#pragma unroll
  for (int i = 12; i < N; i += 2) mr[(i >> 1) & 3] = fmax3(mr[(i >> 1) & 3], at(i), at(i + 1));
  return fmax3(fmaxf(mr[0], mr[1]), mr[2], mr[3]);
}

// p = 2^(s * scale - m) of N keys, packed to 16 bits; returns their sum. Keys >= valid have p = 0.
template <typename T, int N, bool MASK>
__device__ __forceinline__ float probs(const uint32_t (&sr)[N], uint32_t (&pk)[N / 2], float sc, float m, int valid) {
  float2 la[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(-m, -m);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    float2 d = __ffma2_rn(make_float2(__uint_as_float(sr[2 * i]), __uint_as_float(sr[2 * i + 1])), sc2, nm2);
    if (MASK) {
      if (2 * i >= valid) d.x = -1e30f;
      if (2 * i + 1 >= valid) d.y = -1e30f;
    }
    const float2 pp = make_float2(fast_exp2(d.x), fast_exp2(d.y));
    la[i & 1] = __fadd2_rn(la[i & 1], pp);
    pk[i] = Elem<T>::pack(pp.x, pp.y);
  }
  return (la[0].x + la[0].y) + (la[1].x + la[1].y);
}

// x * 0 + acc over a pair: NaN once either half was an infinity or NaN.
template <typename T>
__device__ __forceinline__ uint32_t zero_fma2(uint32_t x, uint32_t acc) {
  if constexpr (Elem<T>::is_bf16) {
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&x), __floats2bfloat162_rn(0.f, 0.f),
                                     *reinterpret_cast<__nv_bfloat162*>(&acc));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&x), __floats2half2_rn(0.f, 0.f),
                              *reinterpret_cast<__half2*>(&acc));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}
template <typename T>
__device__ __forceinline__ bool finite16(uint32_t h) {  // one element in the low half
  constexpr uint32_t kExp = Elem<T>::is_bf16 ? 0x7f80u : 0x7c00u;
  return (h & kExp) != kExp;
}

// Clears what is not finite in row `row` of a [128][64 NA] tile; true if there was any.
template <typename T, int NA>
__device__ __forceinline__ bool clean_row(uint32_t tile, int row) {
  uint32_t acc = 0;
#pragma unroll
  for (int c = 0; c < 8 * NA; ++c) {
    uint32_t x[4];
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                 : "r"(tile + (c >> 3) * kAtom + row * 128 + (c & 7) * 16));
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = zero_fma2<T>(x[e], acc);
  }
  if (finite16<T>(acc) && finite16<T>(acc >> 16)) return false;
#pragma unroll 1
  for (int w = 0; w < 32 * NA; ++w) {
    const uint32_t at = tile + (w >> 5) * kAtom + row * 128 + (w & 31) * 4;
    uint32_t x;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(at));
    if (!finite16<T>(x)) x &= 0xffff0000u;
    if (!finite16<T>(x >> 16)) x &= 0x0000ffffu;
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(x) : "memory");
  }
  fence_proxy_async_smem();  // read by the P V MMA (async proxy)
  return true;
}

template <typename T, int NA>
__global__ void __launch_bounds__(kThreads, 1) packed_fwd_kernel(const __grid_constant__ KParams p) {
  using C = Cfg<NA>;
  constexpr int NK = C::NK, NV = C::NV;
  constexpr uint32_t TILE = C::TILE;
  constexpr bool kBf16 = Elem<T>::is_bf16;
  constexpr uint32_t IDESC_S = idesc_f16(kBf16, 128, 128, false, false);
  constexpr uint32_t IDESC_S32 = idesc_f16(kBf16, 128, 32, false, false);  // a last tile of <= 32 keys
  constexpr uint32_t IDESC_PV = idesc_f16(kBf16, 128, 64 * NA, false, true);
  constexpr uint32_t T_O = 256;

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[11 + 2 * (NK + NV)];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_sh, dirty_sh;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const UnitHead uh = unit_of_block(blockIdx.x, p.a.n_units, p.a.heads, p.a.head_chunk);
  const PackedUnit u = p.a.units[uh.unit];
  const int head = uh.head, kvh = head / p.a.group;
  // keys that local query r sees
  auto limit = [&](int r) { return max(0, min(u.k_valid, p.a.causal ? u.vis0 + r : u.k_valid)); };
  // key tiles of stream w: those that its last query sees
  int n_kt[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int rows = min(u.q_valid - 128 * w, 128);
    const int tiles = rows > 0 ? (limit(128 * w + rows - 1) + 127) >> 7 : 0;
    n_kt[w] = max(0, min(tiles, u.end) - u.begin);
  }
  const int n_max = max(n_kt[0], n_kt[1]);
  const uint32_t streams = (n_kt[0] > 0) + (n_kt[1] > 0);

  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sQ = sbase, sK = sbase + 2 * TILE, sV = sK + NK * TILE;
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t BAR_Q = bar0, BAR_DONE = bar0 + 8u;
  auto BAR_KFULL = [&](int s) { return bar0 + 8u * (2 + s); };
  auto BAR_VFULL = [&](int s) { return bar0 + 8u * (2 + NK + s); };
  auto BAR_KEMPTY = [&](int s) { return bar0 + 8u * (2 + NK + NV + s); };
  auto BAR_VEMPTY = [&](int s) { return bar0 + 8u * (2 + 2 * NK + NV + s); };
  auto BAR_SFULL = [&](int w) { return bar0 + 8u * (2 + 2 * (NK + NV) + w); };
  auto BAR_PHALF = [&](int w) { return bar0 + 8u * (4 + 2 * (NK + NV) + w); };
  auto BAR_PFULL = [&](int w) { return bar0 + 8u * (6 + 2 * (NK + NV) + w); };
  auto BAR_PVH = [&](int w) { return bar0 + 8u * (8 + 2 * (NK + NV) + w); };
  volatile int* abort = &abort_sh;

  if (threadIdx.x == 0) {
    abort_sh = 0;
    dirty_sh = 0;
    mbar_init(BAR_Q, 1);
    mbar_init(BAR_DONE, 1);
    for (int s = 0; s < NK; ++s) {
      mbar_init(BAR_KFULL(s), 1);
      mbar_init(BAR_KEMPTY(s), max(streams, 1u));
    }
    for (int s = 0; s < NV; ++s) {
      mbar_init(BAR_VFULL(s), 1);
      mbar_init(BAR_VEMPTY(s), max(streams, 1u));
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(BAR_SFULL(w), 1);
      mbar_init(BAR_PHALF(w), 128);
      mbar_init(BAR_PFULL(w), 128);
      mbar_init(BAR_PVH(w), 1);
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

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producers
    // lane 0: Q, then the K ring; lane 1: the V ring
    if (lane < 2 && n_max > 0) {
      const bool kl = lane == 0;
      const int nslot = kl ? NK : NV;
      const CUtensorMap* map = kl ? &p.tm_k : &p.tm_v;
      prefetch_tmap(map);
      if (kl) {
        mbar_expect_tx(BAR_Q, streams * TILE);
        for (int w = 0; w < 2; ++w)
          if (n_kt[w] > 0)
            for (int a = 0; a < NA; ++a)
              tma_load(sQ + w * TILE + a * kAtom, &p.tm_q, 64 * a, u.q_row + 128 * w, BIdx(head, 0, 0), BAR_Q);
      }
      int armed[NK > NV ? NK : NV];
      for (int s = 0; s < nslot; ++s) armed[s] = 0;
      for (int t = 0; t < n_max; ++t) {
        const int s = t % nslot;
        if (t >= nslot && !mbar_wait(kl ? BAR_KEMPTY(s) : BAR_VEMPTY(s), ((t / nslot) - 1) & 1, abort, &g_packed_err, 1))
          break;
        const uint32_t full = kl ? BAR_KFULL(s) : BAR_VFULL(s);
        const uint32_t slot = (kl ? sK : sV) + s * TILE;
        const int row = u.k_row + (u.begin + t) * 128;
        mbar_expect_tx(full, TILE);
        for (int a = 0; a < NA; ++a) tma_load(slot + a * kAtom, map, 64 * a, row, BIdx(kvh, 0, 0), full);
        if (t + nslot < n_max)  // the tile one ring ahead into L2
          for (int a = 0; a < NA; ++a) tma_prefetch(map, 64 * a, row + nslot * 128, BIdx(kvh, 0, 0));
        armed[s] = t / nslot + 1;
      }
      // drain: every armed phase must have landed before the CTA may exit
      if (kl) mbar_wait_drain(BAR_Q, 0);
      for (int s = 0; s < nslot; ++s)
        if (armed[s] > 0) mbar_wait_drain(kl ? BAR_KFULL(s) : BAR_VFULL(s), (armed[s] - 1) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    const uint32_t leader = elect_one() ? 1u : 0u;
    auto wwait = [&](uint32_t bar, uint32_t parity, int code) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, &g_packed_err, code));
    };
    // keys of stream w's tile t that some of its queries sees (MMAs of <= 32 keys are shortened)
    auto tile_keys = [&](int w, int t) {
      return limit(min(u.q_valid, 128 * (w + 1)) - 1) - (u.begin + t) * 128;
    };
    auto issue_s = [&](int w, int t) -> bool {
      const int s = t % NK;
      if (!wwait(BAR_KFULL(s), (t / NK) & 1, 2)) return false;
      tc_fence_after();
      const uint32_t kb = sK + s * TILE, qb = sQ + w * TILE;
      const uint32_t idesc = tile_keys(w, t) <= 32 ? IDESC_S32 : IDESC_S;
#pragma unroll
      for (int kk = 0; kk < 4 * NA; ++kk) {
        const uint32_t off = (kk >> 2) * kAtom + (kk & 3) * 32;
        mma_ss_if(leader, tmem + 128 * w, smem_desc_sw128(qb + off, 16, 1024), smem_desc_sw128(kb + off, 16, 1024), idesc,
                  kk > 0);
      }
      mma_commit_if(leader, BAR_SFULL(w));
      return true;
    };
    bool ok = n_max == 0 || wwait(BAR_Q, 0, 2);
    for (int w = 0; w < 2; ++w)
      if (ok && n_kt[w] > 0) ok = issue_s(w, 0);
    for (int j = 0; ok && j < 2 * n_max; ++j) {
      const int w = j & 1, t = j >> 1;
      if (t >= n_kt[w]) continue;
      const uint32_t vb = sV + (t % NV) * TILE;
      const uint32_t a_tm = tmem + 128 * w, o_tm = tmem + T_O + 64 * NA * w;
      const int ksteps = tile_keys(w, t) <= 32 ? 2 : 8;  // 16 keys per step
      if (!wwait(BAR_PHALF(w), t & 1, 4) || !wwait(BAR_VFULL(t % NV), (t / NV) & 1, 4)) break;
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        mma_ts_if(leader & (kk < ksteps ? 1u : 0u), o_tm, a_tm + kk * 8, smem_desc_sw128(vb + kk * 2048, kAtom, 1024),
                  IDESC_PV, (t > 0 || kk > 0) ? 1u : 0u);
      mma_commit_if(leader, BAR_PVH(w));  // a softmax that rescales O mid-tile waits for it
      if (!wwait(BAR_PFULL(w), t & 1, 4)) break;
      tc_fence_after();
#pragma unroll
      for (int kk = 4; kk < 8; ++kk)
        mma_ts_if(leader & (kk < ksteps ? 1u : 0u), o_tm, a_tm + kk * 8, smem_desc_sw128(vb + kk * 2048, kAtom, 1024),
                  IDESC_PV, 1u);
      if (t + 1 < n_kt[w]) ok = issue_s(w, t + 1);
    }
    if (elect_one()) {  // DONE: every MMA complete (the epilogue reads O; TMEM may be freed)
      mma_commit(BAR_DONE);
      mbar_wait_drain(BAR_DONE, 0);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax streams + epilogue
    const int w = (warp - 2) >> 2;  // stream
    const int quad = warp & 3;      // TMEM lane quadrant this warp may access
    const int row = quad * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t tS = tmem + lane_off + 128 * w, tO = tmem + lane_off + T_O + 64 * NA * w;
    const int my_lim = limit(128 * w + row);
    const int lim_lo = limit(128 * w), lim_hi = limit(min(u.q_valid, 128 * (w + 1)) - 1);
    float m_ref = -1e30f, l = 0.f;
    bool ok = true;
    auto warp_wait = [&](uint32_t bar, uint32_t parity, int code) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, &g_packed_err, code));
    };
    // O and l to the reference max(m_ref, mx). Warp-uniform; no P V into O_w may be in flight.
    auto rescale = [&](float mx) {
      const float m_new = fmaxf(m_ref, mx);
      const float alpha = fast_exp2(m_ref - m_new);
#pragma unroll 1
      for (int c = 0; c < 2 * NA; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + c * 32, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
        tmem_st32(tO + c * 32, o);
      }
      tmem_wait_st();
      l *= alpha;
      m_ref = m_new;
    };

    for (int t = 0; t < n_kt[w]; ++t) {
      if (!warp_wait(BAR_SFULL(w), t & 1, 8)) { ok = false; break; }
      tc_fence_after();
      if (warp == 2 + 4 * w && lane == 0) {
        // S_w(t) complete, so is P V_w(t - 1) before it: K(t) and V(t - 1) are free of this stream
        mbar_arrive(BAR_KEMPTY(t % NK));
        if (t >= 1) mbar_arrive(BAR_VEMPTY((t - 1) % NV));
      }
      const int k0 = (u.begin + t) * 128;
      const bool full = lim_lo - k0 >= 128;  // no query of the stream misses a key of the tile
      if (t > 0 && full) {
        // the exponentials against the current reference; a half past the threshold is redone from
        // the scores in registers, after the rescale
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          uint32_t s[64], pk[32];
          tmem_ld32(tS + 64 * hf, s);
          tmem_ld32(tS + 64 * hf + 32, s + 32);
          tmem_wait_ld();
          float lt = probs<T, 64, false>(s, pk, p.scale_log2, m_ref, 64);
          if (__any_sync(0xffffffffu, !(lt <= kSumThreshold))) {
            // first half: S_w(t) complete implies every earlier P V is; second: the first half's P V
            if (hf == 1 && !warp_wait(BAR_PVH(w), t & 1, 16)) { ok = false; break; }
            tc_fence_after();
            rescale(row_max<64, false>(s, 64) * p.scale_log2);
            lt = probs<T, 64, false>(s, pk, p.scale_log2, m_ref, 64);
          }
          l += lt;
          tmem_st32(tS + 32 * hf, pk);
          if (hf == 0) {
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(BAR_PHALF(w));
          }
        }
        if (!ok) break;
      } else {
        // the first tile (sets the reference) and the masked ones: the maximum first
        const int valid = my_lim - k0;
        uint32_t sr[128];
        tmem_ld32(tS, sr);
        tmem_ld32(tS + 32, sr + 32);
        tmem_ld32(tS + 64, sr + 64);
        tmem_ld32(tS + 96, sr + 96);
        if (!full) {
          // values that some query must not see: clear what is not finite (thread = key row)
          if (!warp_wait(BAR_VFULL(t % NV), (t / NV) & 1, 8)) { ok = false; break; }
          if (clean_row<T, NA>(sV + (t % NV) * TILE, row)) dirty_sh = 1;
        }
        tmem_wait_ld();
        const float mx = (full ? row_max<128, false>(sr, 128) : row_max<128, true>(sr, valid)) * p.scale_log2;
        if (t == 0) m_ref = mx;
        else if (__any_sync(0xffffffffu, mx > m_ref + kRescaleThreshold)) rescale(mx);
        {
          const uint32_t(&sh)[64] = *reinterpret_cast<const uint32_t(*)[64]>(&sr[0]);
          uint32_t pk[32];
          if (full) l += probs<T, 64, false>(sh, pk, p.scale_log2, m_ref, 64);
          else l += probs<T, 64, true>(sh, pk, p.scale_log2, m_ref, valid);
          tmem_st32(tS, pk);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(BAR_PHALF(w));
        }
        {
          // the second half is loaded again (only its own P overwrites it), so that the first half's
          // scores alone live through the exponentials
          uint32_t pk[32];
          if (lim_hi - k0 > 64) {
            uint32_t sh[64];
            tmem_ld32(tS + 64, sh);
            tmem_ld32(tS + 96, sh + 32);
            tmem_wait_ld();
            if (full) l += probs<T, 64, false>(sh, pk, p.scale_log2, m_ref, 64);
            else l += probs<T, 64, true>(sh, pk, p.scale_log2, m_ref, valid - 64);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) pk[i] = 0u;
          }
          tmem_st32(tS + 32, pk);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(BAR_PFULL(w));
    }

    // epilogue: O / l in 16 bits (and for a backward the rest that the rounding leaves, 16 bits more)
    // through the idle rings, whole rows to global memory
    if (ok) ok = warp_wait(BAR_DONE, 0, 8);
    tc_fence_after();
    const uint32_t stage = sK + (uint32_t)w * TILE;
    const int rows = min(u.q_valid - 128 * w, 128);
    const bool any = n_kt[w] > 0;
    if (ok && rows > 0) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const bool dirty = *reinterpret_cast<volatile int*>(&dirty_sh) != 0;
#pragma unroll 1
      for (int c = 0; c < 2 * NA; ++c) {
        uint32_t o[32];
        if (any) {
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (dirty && any) {
          // values of the masked tiles that were cleared: back to the queries that see them
          const T* v = static_cast<const T*>(p.a.v) + (int64_t)u.k_row * p.a.vv.rs + (int64_t)kvh * p.a.vv.s1;
          const int j0 = max(limit(0) & ~127, u.begin * 128), j1 = min(my_lim, u.end * 128);
#pragma unroll 1
          for (int j = j0; j < j1; ++j)
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float x = c * 32 + i < p.a.dim ? Elem<T>::to_f(v[(int64_t)j * p.a.vv.rs + c * 32 + i]) : 0.f;
              if (!isfinite(x)) o[i] = __float_as_uint(__uint_as_float(o[i]) + x);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t x[4], y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float a = __uint_as_float(o[8 * k + 2 * i]) * inv, b = __uint_as_float(o[8 * k + 2 * i + 1]) * inv;
            x[i] = Elem<T>::pack(a, b);
            const float2 r = Elem<T>::unpack(x[i]);
            y[i] = Elem<T>::pack(a - r.x, b - r.y);
          }
          const uint32_t at = stage + (c >> 1) * kAtom + row * 128 + ((((c & 1) * 4 + k) ^ (row & 7)) << 4);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3])
                       : "memory");
          if (p.a.o_low)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + 2 * TILE), "r"(y[0]), "r"(y[1]), "r"(y[2]),
                         "r"(y[3])
                         : "memory");
        }
      }
      if (p.a.lse && row < rows)
        p.a.lse[(int64_t)head * p.a.q_total + u.q_row + 128 * w + row] =
            l == 0.f ? __int_as_float(0xff800000) : (m_ref + log2f(l)) * kLn2;
    }
    ok = named_bar_and(2 + w, 128, ok && !*abort);
    if (ok && rows > 0) {
      constexpr int CH = 8 * NA;  // 16-byte chunks per row
      auto store = [&](void* t, const View& v, uint32_t from) {
        T* out = static_cast<T*>(t) + (int64_t)(u.q_row + 128 * w) * v.rs + (int64_t)head * v.s1;
        for (int i = row; i < rows * CH; i += 128) {
          const int r = i / CH, ch = i % CH;
          uint32_t x[4];
          asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                       : "r"(from + (ch >> 3) * kAtom + r * 128 + (((ch & 7) ^ (r & 7)) << 4)));
          if (ch * 8 < p.a.dim) *reinterpret_cast<uint4*>(out + (int64_t)r * v.rs + ch * 8) = make_uint4(x[0], x[1], x[2], x[3]);
        }
      };
      store(p.a.o, p.a.ov, stage);
      if (p.a.o_low) store(p.a.o_low, p.a.olv, stage + 2 * TILE);
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

template <typename T, int NA>
cudaError_t launch(const KParams& p, cudaStream_t st) {
  auto kern = packed_fwd_kernel<T, NA>;
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = allow_smem(kern, Cfg<NA>::SMEM, ready);
  if (e != cudaSuccess) return e;
  const int64_t blocks = (int64_t)p.a.n_units * p.a.heads;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  kern<<<(unsigned)blocks, kThreads, Cfg<NA>::SMEM, st>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_dim(const KParams& p, cudaStream_t st) {
  return p.a.dim > 64 ? launch<T, 2>(p, st) : launch<T, 1>(p, st);
}

}  // namespace

cudaError_t packed_fwd(const PackedParams& a, bool bf16, cudaStream_t st) {
  KParams p{};
  p.a = a;
  p.scale_log2 = a.sm_scale * kLog2e;
  if (!tma::make_map_view(&p.tm_q, a.q, bf16, a.dim, a.q_total, a.heads, a.qv, a.heads, 1, 128)) return cudaErrorInvalidValue;
  if (a.k_total > 0) {
    if (!tma::make_map_view(&p.tm_k, a.k, bf16, a.dim, a.k_total, a.kv_heads, a.kv, a.kv_heads, 1, 128) ||
        !tma::make_map_view(&p.tm_v, a.v, bf16, a.dim, a.k_total, a.kv_heads, a.vv, a.kv_heads, 1, 128))
      return cudaErrorInvalidValue;
  }
  return bf16 ? launch_dim<__nv_bfloat16>(p, st) : launch_dim<__half>(p, st);
}

cudaError_t packed_status(cudaStream_t st, int* out) {
  int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(out, g_packed_err, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && *out) e = cudaMemcpyToSymbolAsync(g_packed_err, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  return e;
}

}  // namespace vmb
