// Attention over packed sequences of different lengths, forward, on tcgen05 / TMA (head dims up to
// 128, multiples of 8; grouped heads; causal or not).
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(s_ij - m_i),  s_ij = sm_scale q_i . k_j,
// over the keys j of query i's own sequence that it sees: all of them, or with `causal` the first
// nk - nq + i + 1 (the last query sees the last key). A query that sees no key has o = 0 and
// lse = -inf.
//
// Work item = one head and one unit of up to 256 queries (two 128-row tiles, one per softmax warpgroup) of
// one sequence, or a piece of its key tiles. 10 warps: TMA producers, MMA issuer, two warpgroups of softmax and
// epilogue, thread = query row. The two streams walk the same ring of 128-key tiles and never wait for one
// another, so one's exponentials run beside the other's matrix products. Online softmax with a lazily raised
// reference: the exponentials of an unmasked tile go against the current reference and are redone
// only when a 64-key half's sum passes 2^14; a warp skips the keys that none of its queries sees. P is 16-bit (the rounding the tensor cores need; l sums
// the unrounded p), everything else 32-bit.
// TMEM (512 columns): S_0 [0,128), S_1 [128,256), O_0 [256, +64 NA), O_1 [256 + 64 NA, +64 NA).
//
// The grid has a block per work item, and a running block takes over blocks that have not started
// (clusterlaunchcontrol), most work first: the next item's queries, keys and first scores are under way while the
// softmax warps write the last item's output straight from registers, and the set-up is paid once per SM.
// Bound by the instructions of the softmax warps (part of the exponentials as polynomials gained nothing):
// 2 us a 256 x 128 tile at D = 128, 4.2 us an item beside its tiles. 32760 causal tokens, 16/4 heads, D = 128, bf16:
// 3600 us, 1.22 PFLOP/s in short runs, 4090 us, 1.07 under the power cap; 16 prompts of 1 to 4093 tokens, 40/8 heads: 403 us,
// 0.84 PFLOP/s in short runs (the measured dense rate is 1.67).
// An item that is cut leaves 32-bit partials (max, sum, O), joined by a second kernel; the host cuts
// where few items would leave SMs without work.
//
// The sequences share one tensor, so a tile's rows past the sequence end are the next sequence's.
// Scores past the end (or after the diagonal) are dropped by index. A value row that a query does not
// see enters its P V with p = 0, and 0 x inf = NaN, so in a tile that is masked for some query of the unit the
// threads of both streams look the value tile over (one multiply by zero per pair) and clear what is not finite;
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
};

// Asks for a block of the grid that has not started: 16 bytes of answer, completing on `bar`.
__device__ __forceinline__ void request_block(uint32_t answer, uint32_t bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer),
               "r"(bar)
               : "memory");
}
// The block that the answer names, or -1 when there is none left.
__device__ __forceinline__ int answered_block(uint32_t answer) {
  int id;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\tld.shared.b128 h, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tmov.b32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n\t}"
      : "=r"(id)
      : "r"(answer)
      : "memory");
  return id;
}

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

// Clears what is not finite in row `row` of a [128][64 NA] tile, once `*dirty` is `mark`. Both streams may do so to one
// tile at a time: each finds a value or its clearing, and the mark with the latter.
template <typename T, int NA>
__device__ __forceinline__ void clean_row(uint32_t tile, int row, volatile int* dirty, int mark) {
  uint32_t acc = 0;
#pragma unroll
  for (int c = 0; c < 8 * NA; ++c) {  // neighbouring rows begin at different chunks: no bank conflicts
    uint32_t x[4];
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                 : "r"(tile + (c >> 3) * kAtom + row * 128 + ((c + row) & 7) * 16));
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = zero_fma2<T>(x[e], acc);
  }
  const bool clean = finite16<T>(acc) && finite16<T>(acc >> 16);
  if (!clean) *dirty = mark;
  __threadfence_block();
  if (!clean) {
#pragma unroll 1
    for (int w = 0; w < 32 * NA; ++w) {
      const uint32_t at = tile + (w >> 5) * kAtom + row * 128 + (w & 31) * 4;
      uint32_t x;
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(at));
      if (!finite16<T>(x)) x &= 0xffff0000u;
      if (!finite16<T>(x >> 16)) x &= 0x0000ffffu;
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(x) : "memory");
    }
  }
  // read by the P V MMA (async proxy), whichever thread cleared it (16 mixed prompts: 408 us with the fence always, 403 so)
  if (*dirty == mark) fence_proxy_async_smem();
}

// A work item, made by the K producer and read by every role from shared memory.
struct Item {
  PackedUnit u;
  int head, kvh;     // head -1: no more work
  int n_kt[2], n_max;  // key tiles of the two streams
  int brief;         // bit w: stream w's last tile has at most 32 keys that count
  int causal;
  // keys that local query r sees
  __device__ __forceinline__ int limit(int r) const { return max(0, min(u.k_valid, causal ? u.vis0 + r : u.k_valid)); }
  __device__ __forceinline__ void set(const PackedParams& a, const PackedUnit& unit, int h) {
    u = unit;
    head = h;
    kvh = h / a.group;
    causal = a.causal;
    brief = 0;
#pragma unroll
    for (int w = 0; w < 2; ++w) {  // tiles that stream w's last query sees
      const int rows = min(u.q_valid - 128 * w, 128);
      const int last = rows > 0 ? limit(128 * w + rows - 1) : 0;
      n_kt[w] = max(0, min((last + 127) >> 7, u.end) - u.begin);
      if (last - (u.begin + n_kt[w] - 1) * 128 <= 32) brief |= 1 << w;
    }
    n_max = max(n_kt[0], n_kt[1]);
  }
};

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
  // barriers: queries full / free, slots full / free, per stream S, first half of P, P, first half of P V, O full,
  // O free, and the work ring: answer, block known, block read
  constexpr int B_QFULL = 0, B_QFREE = 1, B_KFULL = 2, B_KFREE = B_KFULL + NK, B_VFULL = B_KFREE + NK, B_VFREE = B_VFULL + NV,
                B_S = B_VFREE + NV, B_PHALF = B_S + 2, B_PFULL = B_PHALF + 2, B_PVH = B_PFULL + 2, B_OFULL = B_PVH + 2,
                B_OFREE = B_OFULL + 2, B_ANSWER = B_OFREE + 2, B_WFULL = B_ANSWER + 1, B_WFREE = B_WFULL + 2,
                NBARS = B_WFREE + 2;

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(16) uint4 answer_sh;
  __shared__ __align__(8) uint64_t bars[NBARS];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_sh, dirty_sh[2];
  __shared__ Item work_sh[2];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sQ = sbase, sK = sbase + 2 * TILE, sV = sK + NK * TILE;
  const uint32_t bar0 = smem_u32(bars);
  auto BAR = [&](int i) { return bar0 + 8u * (uint32_t)i; };
  volatile int* abort = &abort_sh;

  if (threadIdx.x == 0) {
    abort_sh = 0;
    dirty_sh[0] = dirty_sh[1] = 0;
    for (int i = 0; i < NBARS; ++i) {
      const bool rows = (i >= B_PHALF && i < B_PVH) || i == B_OFREE || i == B_OFREE + 1;
      const bool slots = (i >= B_KFREE && i < B_VFULL) || (i >= B_VFREE && i < B_S);  // freed by both streams
      // a block id is read by the V producer, the MMA warp and eight softmax warps
      mbar_init(BAR(i), rows ? 128 : i >= B_WFREE ? 10 : slots ? 2 : 1);
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

  // The K producer hands the items on through work_sh: item i in place i & 1 until its ten readers are done with it.
  auto work_wait = [&](int i, int code) -> bool {
    // (the one wait that runs out when loads are held, so the one with a limit that a test can shorten)
    return mbar_wait(BAR(B_WFULL + (i & 1)), (i >> 1) & 1, abort, &g_packed_err, code, p.a.wait_limit);
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producers
    // lane 0: work ring, Q and the K ring; lane 1: the V ring
    // (hold_loads, a test of the timeout path: no work is handed on, so every other role's wait runs out)
    if (lane < 2 && !p.a.hold_loads) {
      const bool kl = lane == 0;
      const int nslot = kl ? NK : NV;
      const CUtensorMap* map = kl ? &p.tm_k : &p.tm_v;
      prefetch_tmap(map);
      int tiles = 0, queries = 0, asked = 0;  // loaded so far by this lane; answers asked for
      bool ok = true;
      Item it;
      int block = blockIdx.x;
      for (int i = 0; ok; ++i) {
        if (kl) {
          it.head = -1;
          if (block >= 0) {
            const UnitHead uh = unit_of_block(block, p.a.n_units, p.a.heads, p.a.head_chunk);
            it.set(p.a, p.a.units[uh.unit], uh.head);
          }
          if (i >= 2 && !(ok = mbar_wait(BAR(B_WFREE + (i & 1)), ((i - 2) >> 1) & 1, abort, &g_packed_err, 1))) break;
          work_sh[i & 1] = it;
          mbar_arrive(BAR(B_WFULL + (i & 1)));
        } else {
          if (!(ok = work_wait(i, 1))) break;
          it = work_sh[i & 1];
          mbar_arrive(BAR(B_WFREE + (i & 1)));
        }
        if (it.head < 0) break;
        if (kl) {  // ask for the item after this one, long before it is needed
          fence_proxy_async_smem();
          mbar_expect_tx(BAR(B_ANSWER), 16);
          request_block(smem_u32(&answer_sh), BAR(B_ANSWER));
          ++asked;
        }
        if (kl && it.n_max > 0) {
          if (queries > 0) ok = mbar_wait(BAR(B_QFREE), (queries - 1) & 1, abort, &g_packed_err, 1);
          if (!ok) break;
          mbar_expect_tx(BAR(B_QFULL), ((it.n_kt[0] > 0) + (it.n_kt[1] > 0)) * TILE);
          for (int w = 0; w < 2; ++w)
            if (it.n_kt[w] > 0)
              for (int a = 0; a < NA; ++a)
                tma_load(sQ + w * TILE + a * kAtom, &p.tm_q, 64 * a, it.u.q_row + 128 * w, BIdx(it.head, 0, 0), BAR(B_QFULL));
          ++queries;
        }
        for (int t = 0; t < it.n_max; ++t, ++tiles) {
          const int s = tiles % nslot;
          if (tiles >= nslot &&
              !mbar_wait(BAR((kl ? B_KFREE : B_VFREE) + s), ((tiles / nslot) - 1) & 1, abort, &g_packed_err, 1)) {
            ok = false;
            break;
          }
          const uint32_t full = BAR((kl ? B_KFULL : B_VFULL) + s), slot = (kl ? sK : sV) + s * TILE;
          const int row = it.u.k_row + (it.u.begin + t) * 128;
          mbar_expect_tx(full, TILE);
          for (int a = 0; a < NA; ++a) tma_load(slot + a * kAtom, map, 64 * a, row, BIdx(it.kvh, 0, 0), full);
          if (t + nslot < it.n_max)  // the tile one ring ahead into L2
            for (int a = 0; a < NA; ++a) tma_prefetch(map, 64 * a, row + nslot * 128, BIdx(it.kvh, 0, 0));
        }
        if (!ok) break;
        if (kl) {
          if (!(ok = mbar_wait(BAR(B_ANSWER), i & 1, abort, &g_packed_err, 1))) break;
          block = answered_block(smem_u32(&answer_sh));
        }
      }
      // drain: what was asked for must have landed before the CTA may exit
      if (kl && queries > 0) mbar_wait_drain(BAR(B_QFULL), (queries - 1) & 1);
      if (kl && asked > 0) mbar_wait_drain(BAR(B_ANSWER), (asked - 1) & 1);
      for (int t = max(tiles - nslot, 0); t < tiles; ++t)
        mbar_wait_drain(BAR((kl ? B_KFULL : B_VFULL) + t % nslot), (t / nslot) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    const uint32_t leader = elect_one() ? 1u : 0u;
    auto wwait = [&](int bar, uint32_t parity, int code) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(BAR(bar), parity, abort, &g_packed_err, code));
    };
    // ring positions of the K tile that is scored next and of the V tile that is weighed next (every tile is loaded
    // once for both streams), per-stream tiles and units so far
    int queries = 0, steps[2] = {0, 0}, outs[2] = {0, 0}, ks0 = 0, kp0 = 0, vs0 = 0, vp0 = 0;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      if (!(ok = __all_sync(0xffffffffu, work_wait(i, 2)))) break;
      const int head = work_sh[i & 1].head, n_max = work_sh[i & 1].n_max;
      const int n_kt[2] = {work_sh[i & 1].n_kt[0], work_sh[i & 1].n_kt[1]};
      // a stream's last tile of <= 32 keys: shorter products
      const bool brief[2] = {(work_sh[i & 1].brief & 1) != 0, (work_sh[i & 1].brief & 2) != 0};
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR(B_WFREE + (i & 1)));
      if (head < 0) break;
      if (n_max == 0) continue;
      // S of stream w's tile t, whose K tile is in slot s since its phase `parity`
      auto issue_s = [&](int w, int t, int s, uint32_t parity) -> bool {
        if (!wwait(B_KFULL + s, parity, 2)) return false;
        tc_fence_after();
        const uint32_t kb = sK + s * TILE, qb = sQ + w * TILE;
        const uint32_t idesc = brief[w] && t + 1 == n_kt[w] ? IDESC_S32 : IDESC_S;
#pragma unroll
        for (int kk = 0; kk < 4 * NA; ++kk) {
          const uint32_t off = (kk >> 2) * kAtom + (kk & 3) * 32;
          mma_ss_if(leader, tmem + 128 * w, smem_desc_sw128(qb + off, 16, 1024), smem_desc_sw128(kb + off, 16, 1024), idesc,
                    kk > 0);
        }
        mma_commit_if(leader, BAR(B_S + w));
        return true;
      };
      ok = wwait(B_QFULL, queries & 1, 2);
      ++queries;
      for (int w = 0; w < 2; ++w)
        if (ok && n_kt[w] > 0) ok = issue_s(w, 0, ks0, kp0);
      if (ok && n_max == 1) mma_commit_if(leader, BAR(B_QFREE));
      for (int t = 0; ok && t < n_max; ++t) {
        if (++ks0 == NK) ks0 = 0, kp0 ^= 1;  // the next K tile
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (!ok || t >= n_kt[w]) continue;
          const int c = steps[w] + t;
          const uint32_t vb = sV + vs0 * TILE;
          const uint32_t a_tm = tmem + 128 * w, o_tm = tmem + T_O + 64 * NA * w;
          const int ksteps = brief[w] && t + 1 == n_kt[w] ? 2 : 8;  // 16 keys per step
          if (!(ok = wwait(B_PHALF + w, c & 1, 4) && wwait(B_VFULL + vs0, vp0, 4))) break;
          // the stream's O of the last unit has been read
          if (t == 0 && outs[w] > 0 && !(ok = wwait(B_OFREE + w, (outs[w] - 1) & 1, 4))) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_ts_if(leader & (kk < ksteps ? 1u : 0u), o_tm, a_tm + kk * 8, smem_desc_sw128(vb + kk * 2048, kAtom, 1024),
                      IDESC_PV, (t > 0 || kk > 0) ? 1u : 0u);
          mma_commit_if(leader, BAR(B_PVH + w));  // a softmax that rescales O mid-tile waits for it
          if (!(ok = wwait(B_PFULL + w, c & 1, 4))) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 4; kk < 8; ++kk)
            mma_ts_if(leader & (kk < ksteps ? 1u : 0u), o_tm, a_tm + kk * 8, smem_desc_sw128(vb + kk * 2048, kAtom, 1024),
                      IDESC_PV, 1u);
          if (t + 1 < n_kt[w]) ok = issue_s(w, t + 1, ks0, kp0);
          else mma_commit_if(leader, BAR(B_OFULL + w));
        }
        if (ok && t + 2 == n_max) mma_commit_if(leader, BAR(B_QFREE));  // the last scores are on their way
        if (++vs0 == NV) vs0 = 0, vp0 ^= 1;
      }
      for (int w = 0; w < 2; ++w) {
        steps[w] += n_kt[w];
        outs[w] += n_kt[w] > 0;
      }
    }
    // every MMA issued must be complete before TMEM can be freed: one more round of the queries' barrier
    __syncwarp();
    if (elect_one()) {
      __shared__ __align__(8) uint64_t done_sh;
      const uint32_t done = smem_u32(&done_sh);
      mbar_init(done, 1);
      fence_mbar_init();
      mma_commit(done);
      mbar_wait_drain(done, 0);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax streams + epilogue
    const int w = (warp - 2) >> 2;  // stream
    const int quad = warp & 3;      // TMEM lane quadrant this warp may access
    const int row = quad * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t tS = tmem + lane_off + 128 * w, tO = tmem + lane_off + T_O + 64 * NA * w;
    auto warp_wait = [&](int bar, uint32_t parity, int code) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(BAR(bar), parity, abort, &g_packed_err, code));
    };
    const bool sectors = whole_sectors(p.a.o, p.a.ov) && whole_sectors(p.a.o_low, p.a.olv);
    int steps = 0, outs = 0, ring = 0;  // tiles and units of this stream so far, tiles of the ring
    const bool leads = warp == 2 + 4 * w && lane == 0;  // frees ring slots for the stream
    bool ok = true;
    for (int i = 0; ok; ++i) {
      if (!(ok = __all_sync(0xffffffffu, work_wait(i, 8)))) break;
      if (work_sh[i & 1].head < 0) break;
      // what the loop over the tiles needs; the epilogue reads the rest again (the loop wants the registers)
      int n_kt, begin, my_lim, lim_lo;
      bool live;
      {
        const Item& it = work_sh[i & 1];
        n_kt = it.n_kt[w];
        begin = it.u.begin;
        // rows past the unit's last query are not stored: they take its limit, and no part in the reference
        live = 128 * w + row < it.u.q_valid;
        my_lim = it.limit(min(128 * w + row, it.u.q_valid - 1));
        lim_lo = it.limit(0);  // of the unit's first query, for both streams
      }
      float m_ref = -1e30f, l = 0.f;
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
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st32(tO + c * 32, o);
        }
        tmem_wait_st();
        l *= alpha;
        m_ref = m_new;
      };

      for (int t = 0; t < n_kt; ++t, ++steps) {
        if (!(ok = warp_wait(B_S + w, steps & 1, 8))) break;
        tc_fence_after();
        if (leads) {
          // S_w(t) complete, so is P V_w(t - 1) before it: K(t) and V(t - 1) are free of this stream
          mbar_arrive(BAR(B_KFREE + (ring + t) % NK));
          if (t >= 1) mbar_arrive(BAR(B_VFREE + (ring + t - 1) % NV));
        }
        const int k0 = (begin + t) * 128;
        // Two 64-key halves; a half's P lets its P V start. The exponentials go against the current reference (the
        // unit's first half sets it); a half past the threshold is redone from the scores in registers, once
        // no P V into O is under way: S_w(t) complete implies that every earlier one is done, and in the second
        // half the first half's is waited for.
        if (t > 0 && lim_lo - k0 >= 128) {  // no query of the unit misses a key of the tile
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            uint32_t s[64], pk[32];
            tmem_ld32(tS + 64 * hf, s);
            tmem_ld32(tS + 64 * hf + 32, s + 32);
            tmem_wait_ld();
            float lt = probs<T, 64, false>(s, pk, p.scale_log2, m_ref, 64);
            if (__any_sync(0xffffffffu, live && !(lt <= kSumThreshold))) {
              if (hf == 1 && !(ok = warp_wait(B_PVH + w, steps & 1, 16))) break;
              tc_fence_after();
              rescale(row_max<64, false>(s, 64) * p.scale_log2);
              lt = probs<T, 64, false>(s, pk, p.scale_log2, m_ref, 64);
            }
            l += lt;
            tmem_st32(tS + 32 * hf, pk);
            if (hf == 0) {
              tmem_wait_st();
              tc_fence_before();
              mbar_arrive(BAR(B_PHALF + w));
            }
          }
        } else {
          if (lim_lo - k0 < 128) {
            // Values that some query of the unit must not see: clear what is not finite (thread = key row). Both streams
            // look, also the one whose queries see the whole tile: the other's clearing may come before its product or
            // after, and the epilogue adds back what was cleared in the tiles from here on.
            const int sv = (ring + t) % NV;
            if (!(ok = warp_wait(B_VFULL + sv, ((ring + t) / NV) & 1, 8))) break;
            clean_row<T, NA>(sV + sv * TILE, row, &dirty_sh[i & 1], i + 1);
          }
#pragma unroll 1
          for (int hf = 0; hf < 2; ++hf) {
            const int seen = my_lim - k0 - 64 * hf;               // keys of the half that this query sees,
            const int least = __shfl_sync(0xffffffffu, seen, 0);  // the warp's first query (limits only grow)
            const int most = __shfl_sync(0xffffffffu, seen, 31);  // and its last
            uint32_t pk[32];
            if (most <= 0) {
#pragma unroll
              for (int e = 0; e < 32; ++e) pk[e] = 0u;
            } else {
              uint32_t s[64];
              tmem_ld32(tS + 64 * hf, s);
              tmem_ld32(tS + 64 * hf + 32, s + 32);
              tmem_wait_ld();
              if (hf == 0 && t == 0) m_ref = (least >= 64 ? row_max<64, false>(s, 64) : row_max<64, true>(s, seen)) * p.scale_log2;
              float lt = 0.f;
#pragma unroll 1
              for (int pass = 0; pass < 2; ++pass) {
                if (least >= 64) {
                  lt = probs<T, 64, false>(s, pk, p.scale_log2, m_ref, 64);
                } else {
                  // masked, 32 keys at a time: a warp computes only those that one of its queries sees
                  const uint32_t(&s0)[32] = *reinterpret_cast<const uint32_t(*)[32]>(&s[0]);
                  const uint32_t(&s1)[32] = *reinterpret_cast<const uint32_t(*)[32]>(&s[32]);
                  uint32_t(&p0)[16] = *reinterpret_cast<uint32_t(*)[16]>(&pk[0]);
                  uint32_t(&p1)[16] = *reinterpret_cast<uint32_t(*)[16]>(&pk[16]);
                  lt = probs<T, 32, true>(s0, p0, p.scale_log2, m_ref, seen);
                  if (most > 32) {
                    lt += probs<T, 32, true>(s1, p1, p.scale_log2, m_ref, seen - 32);
                  } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) p1[e] = 0u;
                  }
                }
                if (pass || !__any_sync(0xffffffffu, live && !(lt <= kSumThreshold))) break;
                if (hf == 1 && !(ok = warp_wait(B_PVH + w, steps & 1, 16))) break;
                tc_fence_after();
                rescale(row_max<64, true>(s, seen) * p.scale_log2);
              }
              if (!ok) break;
              l += lt;
            }
            tmem_st32(tS + 32 * hf, pk);
            if (hf == 0) {
              tmem_wait_st();
              tc_fence_before();
              mbar_arrive(BAR(B_PHALF + w));
            }
          }
        }
        if (!ok) break;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(BAR(B_PFULL + w));
      }
      if (!ok) break;

      // epilogue: O / l in 16 bits (and for a backward the rest that the rounding leaves, 16 bits more), or a
      // piece's O, m and l in 32; whole rows from registers to global memory
      if (n_kt > 0) {
        if (!(ok = warp_wait(B_OFULL + w, outs & 1, 8))) break;
        ++outs;
        tc_fence_after();
      }
      const Item& it = work_sh[i & 1];
      const PackedUnit& u = it.u;
      if (leads) {
        // the stream's last V tile, and the tiles that only the other stream uses: each once it has landed, so
        // that this stream's word for a slot never runs ahead of the slot's phase
        if (n_kt > 0) mbar_arrive(BAR(B_VFREE + (ring + n_kt - 1) % NV));
        for (int t = n_kt; ok && t < it.n_max; ++t) {
          const int r = ring + t;
          ok = mbar_wait(BAR(B_KFULL + r % NK), (r / NK) & 1, abort, &g_packed_err, 8) &&
               mbar_wait(BAR(B_VFULL + r % NV), (r / NV) & 1, abort, &g_packed_err, 8);
          if (!ok) break;
          mbar_arrive(BAR(B_KFREE + r % NK));
          mbar_arrive(BAR(B_VFREE + r % NV));
        }
      }
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      ring += it.n_max;
      const bool dirty = *reinterpret_cast<volatile int*>(&dirty_sh[i & 1]) == i + 1;
      const float inv = u.part >= 0 ? 1.f : l == 0.f ? 0.f : 1.f / l;
      const int64_t grow = u.q_row + 128 * w + row;
      uint16_t* out = static_cast<uint16_t*>(p.a.o) + grow * p.a.ov.rs + (int64_t)it.head * p.a.ov.s1;
      uint16_t* low = static_cast<uint16_t*>(p.a.o_low) + grow * p.a.olv.rs + (int64_t)it.head * p.a.olv.s1;
      const int64_t prow = ((int64_t)u.part * p.a.heads + it.head) * 256 + 128 * w + row;  // row of a piece's partial
#pragma unroll 1
      for (int c = 0; c < 2 * NA; ++c) {
        uint32_t o[32];
        __syncwarp();
        if (n_kt > 0) {
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
          if (c + 1 == 2 * NA) {  // O is in registers: the next item's products may overwrite it
            tc_fence_before();
            mbar_arrive(BAR(B_OFREE + w));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (!live) continue;
        if (dirty && n_kt > 0) {
          // values of the masked tiles that were cleared: back to the queries that see them
          const T* v = static_cast<const T*>(p.a.v) + (int64_t)u.k_row * p.a.vv.rs + (int64_t)it.kvh * p.a.vv.s1;
          const int j0 = max(it.limit(0) & ~127, u.begin * 128), j1 = min(my_lim, u.end * 128);
#pragma unroll 1
          for (int j = j0; j < j1; ++j)
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float x = c * 32 + e < p.a.dim ? Elem<T>::to_f(v[(int64_t)j * p.a.vv.rs + c * 32 + e]) : 0.f;
              if (!isfinite(x)) o[e] = __float_as_uint(__uint_as_float(o[e]) + x);
            }
        }
        if (u.part >= 0) {
          float* to = p.a.part + prow * (64 * NA) + c * 32;
#pragma unroll
          for (int k = 0; k < 4; ++k) st_global_v8(to + 8 * k, o + 8 * k);
          continue;
        }
        uint32_t x[16];
        const float2 inv2 = make_float2(inv, inv);
        auto scaled = [&](int e) { return __fmul2_rn(make_float2(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1])), inv2); };
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 a = scaled(e);
          x[e] = Elem<T>::pack(a.x, a.y);
        }
        store_row32(out, c * 32, p.a.dim, sectors, x);
        if (p.a.o_low) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 a = scaled(e), r = Elem<T>::unpack(x[e]);
            x[e] = Elem<T>::pack(a.x - r.x, a.y - r.y);
          }
          store_row32(low, c * 32, p.a.dim, sectors, x);
        }
      }
      if (live) {
        if (u.part >= 0)
          reinterpret_cast<float2*>(p.a.part_ml)[prow] = make_float2(m_ref, l);
        else if (p.a.lse)
          p.a.lse[(int64_t)it.head * p.a.q_total + grow] = l == 0.f ? __int_as_float(0xff800000) : (m_ref + log2f(l)) * kLn2;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR(B_WFREE + (i & 1)));
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// Joins the pieces of cut units: block = (unit, head, 32 rows), 8 lanes a row, 8 NA columns a lane.
template <typename T, int NA>
__global__ void __launch_bounds__(256) packed_fwd_join_kernel(const __grid_constant__ PackedParams a) {
  wait_for_kernel_before();
  let_next_kernel_start();
  const int64_t uh = blockIdx.x >> 3;
  const int join = (int)(uh / a.heads), head = (int)(uh % a.heads);
  const PackedUnit u = a.units[a.joins[2 * join]];
  const int pieces = a.joins[2 * join + 1];
  const int row = (blockIdx.x & 7) * 32 + (threadIdx.x >> 3), sub = threadIdx.x & 7;
  if (row >= u.q_valid) return;
  auto at = [&](int k) { return ((int64_t)(u.part + k) * a.heads + head) * 256 + row; };
  float m = -1e30f, l = 0.f;
  for (int k = 0; k < pieces; ++k) m = fmaxf(m, reinterpret_cast<const float2*>(a.part_ml)[at(k)].x);
  float o[8 * NA];
#pragma unroll
  for (int i = 0; i < 8 * NA; ++i) o[i] = 0.f;
  for (int k = 0; k < pieces; ++k) {
    const float2 ml = reinterpret_cast<const float2*>(a.part_ml)[at(k)];
    const float f = fast_exp2(ml.x - m);
    l = fmaf(ml.y, f, l);
    const float4* v = reinterpret_cast<const float4*>(a.part + at(k) * (64 * NA) + sub * 8 * NA);
#pragma unroll
    for (int i = 0; i < 2 * NA; ++i) {
      const float4 x = v[i];
      o[4 * i] = fmaf(x.x, f, o[4 * i]);
      o[4 * i + 1] = fmaf(x.y, f, o[4 * i + 1]);
      o[4 * i + 2] = fmaf(x.z, f, o[4 * i + 2]);
      o[4 * i + 3] = fmaf(x.w, f, o[4 * i + 3]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t grow = u.q_row + row;
#pragma unroll
  for (int g = 0; g < NA; ++g) {
    const int col = sub * 8 * NA + 8 * g;
    if (col >= a.dim) continue;
    uint32_t x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = o[8 * g + 2 * i] * inv, q = o[8 * g + 2 * i + 1] * inv;
      x[i] = Elem<T>::pack(p, q);
      const float2 r = Elem<T>::unpack(x[i]);
      y[i] = Elem<T>::pack(p - r.x, q - r.y);
    }
    *reinterpret_cast<uint4*>(static_cast<T*>(a.o) + grow * a.ov.rs + head * a.ov.s1 + col) = make_uint4(x[0], x[1], x[2], x[3]);
    if (a.o_low)
      *reinterpret_cast<uint4*>(static_cast<T*>(a.o_low) + grow * a.olv.rs + head * a.olv.s1 + col) = make_uint4(y[0], y[1], y[2], y[3]);
  }
  if (sub == 0 && a.lse)
    a.lse[(int64_t)head * a.q_total + grow] = l == 0.f ? __int_as_float(0xff800000) : (m + log2f(l)) * kLn2;
}

template <typename T, int NA>
cudaError_t launch(const KParams& p, cudaStream_t st) {
  auto kern = packed_fwd_kernel<T, NA>;
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = allow_smem(kern, Cfg<NA>::SMEM, ready);
  if (e != cudaSuccess) return e;
  e = launch_early(kern, (int64_t)p.a.n_units * p.a.heads, kThreads, Cfg<NA>::SMEM, st, p);
  if (e != cudaSuccess || p.a.n_joins == 0) return e;
  return launch_early(packed_fwd_join_kernel<T, NA>, (int64_t)p.a.n_joins * p.a.heads * 8, 256, 0, st, p.a);
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
