// Gated residual with a norm after a block and a modulated norm before the next one.
//
//   y^ = y ry post_weight, ry = 1 / sqrt(mean(y^2) + eps)      (without post_weight: y^ = y)
//   x' = x + gate y^
//   n  = (x' - mean) rx, rx = 1 / sqrt(mean((x' - mean)^2) + eps)   (rms: mean = 0)
//   h  = n weight (1 + scale) + shift
// with gate, scale and shift one row per sequence, weights one for all. Backward, with g = dh weight
// (1 + scale):
//   dx = dx' + rx (g - [mean(g)] - n mean(g n)),   t = dx gate post_weight,
//   dy = ry (t - y ry mean(t y ry))                (without post_weight: dy = dx gate)
//   A_s = sum dx y ry, B_s = sum dh n, C_s = sum dh over the rows of sequence s:
//   dgate_s = post_weight A_s, dscale_s = weight B_s, dshift_s = C_s,
//   dpost_weight = sum_s gate_s A_s, dweight = sum_s (1 + scale_s) B_s.
// x' enters n unrounded in both directions (the backward forms it again from x and y, which costs no more
// bytes than reading the rounded x' would); all arithmetic is 32-bit, rounded once at each output.
//
// Bound by memory: 8 bytes an element forward (x, y in, x', h out), 12 backward. A block takes an equal
// share of all rows; groups of TPR threads hold a row each, 8 VPT columns a thread, and go through the share
// behind a ring of cp.async stages, in which every thread reads back only what it loaded itself; a group's
// warps meet at a barrier of their own, so one group's sums run beside another's arithmetic. What the
// row-wise work needs of the parameters (gate post_weight, weight (1 + scale), shift) is combined once per
// sequence into shared memory: from L2 it would be more than the rows' own traffic. The column sums
// of the backward stay in registers over a block's rows of a sequence; each (block, sequence) leaves one
// 32-bit partial row, added in a fixed order by a second kernel. 16637 rows of 5120 columns, layer norm and post norm,
// fp32 parameters: forward 131 us, backward 232 us with its sums, calls in a row (79 % and 67 % of the measured copy rate);
// 24 rows, two rms norms: 5.2 us, replayed in a graph.
#include <algorithm>

#include "common.cuh"
#include "gated_norm.h"
#include "launch.h"

namespace vmb {
namespace {

constexpr int kSmemLimit = 220 * 1024;  // dynamic shared memory of an SM's blocks together

// Eight columns as four pairs: the packed f32x2 instructions do two products or sums at once.
struct V8 {
  float2 v[4];
};
__device__ __forceinline__ float2 pair(float a) { return make_float2(a, a); }
__device__ __forceinline__ V8 splat(float a) { return V8{{pair(a), pair(a), pair(a), pair(a)}}; }
template <typename T>
__device__ __forceinline__ V8 unpack8(uint4 x) {
  return V8{{Elem<T>::unpack(x.x), Elem<T>::unpack(x.y), Elem<T>::unpack(x.z), Elem<T>::unpack(x.w)}};
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const V8& f) {
  return make_uint4(Elem<T>::pack(f.v[0].x, f.v[0].y), Elem<T>::pack(f.v[1].x, f.v[1].y),
                    Elem<T>::pack(f.v[2].x, f.v[2].y), Elem<T>::pack(f.v[3].x, f.v[3].y));
}
__device__ __forceinline__ void put8(float* s, const V8& f) {
  reinterpret_cast<float4*>(s)[0] = make_float4(f.v[0].x, f.v[0].y, f.v[1].x, f.v[1].y);
  reinterpret_cast<float4*>(s)[1] = make_float4(f.v[2].x, f.v[2].y, f.v[3].x, f.v[3].y);
}
__device__ __forceinline__ V8 get8(const float* s) {
  const float4 a = reinterpret_cast<const float4*>(s)[0], b = reinterpret_cast<const float4*>(s)[1];
  return V8{{make_float2(a.x, a.y), make_float2(a.z, a.w), make_float2(b.x, b.y), make_float2(b.z, b.w)}};
}
// The same in shared rows that are read 8 columns a thread: the halves of all vectors apart ([2][cols / 8] of four
// floats), so that neighbouring threads read neighbouring 16 bytes.
__device__ __forceinline__ void put_apart(float* s, int cols, int col, const V8& f) {
  float4* q = reinterpret_cast<float4*>(s) + (col >> 3);
  q[0] = make_float4(f.v[0].x, f.v[0].y, f.v[1].x, f.v[1].y);
  q[cols >> 3] = make_float4(f.v[2].x, f.v[2].y, f.v[3].x, f.v[3].y);
}
__device__ __forceinline__ V8 get_apart(const float* s, int cols, int col) {
  const float4* q = reinterpret_cast<const float4*>(s) + (col >> 3);
  const float4 a = q[0], b = q[cols >> 3];
  return V8{{make_float2(a.x, a.y), make_float2(a.z, a.w), make_float2(b.x, b.y), make_float2(b.z, b.w)}};
}
__device__ __forceinline__ float sum8(const V8& f) {
  const float2 a = __fadd2_rn(__fadd2_rn(f.v[0], f.v[1]), __fadd2_rn(f.v[2], f.v[3]));
  return a.x + a.y;
}
__device__ __forceinline__ float dot8(const V8& f, const V8& g) {
  const float2 a = __ffma2_rn(f.v[0], g.v[0], __fmul2_rn(f.v[1], g.v[1]));
  const float2 b = __ffma2_rn(f.v[2], g.v[2], __fmul2_rn(f.v[3], g.v[3]));
  return (a.x + b.x) + (a.y + b.y);
}
template <typename T, typename P>
struct Io;  // 8 elements of a parameter
template <typename T>
struct Io<T, float> {
  static __device__ __forceinline__ V8 load(const void* base, int64_t at) { return get8(static_cast<const float*>(base) + at); }
};
template <typename T>
struct Io<T, T> {
  static __device__ __forceinline__ V8 load(const void* base, int64_t at) {
    return unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(base) + at));
  }
};

// Sums N <= 8 values over a warp with about log2(32) + N shuffles instead of 5 N: while there are several
// values, a step hands half of them to the other half of the lanes. NP: N rounded up to a power of two;
// afterwards the lanes [i 32 / NP, +32 / NP) hold value i's sum in v[0].
template <int NP>
__device__ __forceinline__ void warp_sums(float (&v)[NP]) {
  int width = 16;
#pragma unroll
  for (int n = NP / 2; n > 0; n >>= 1, width >>= 1) {
    const bool hi = threadIdx.x & width;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float send = hi ? v[i] : v[i + n], keep = hi ? v[i + n] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, width);
    }
  }
#pragma unroll
  for (; width > 0; width >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], width);
}

// Where the warps of a row meet: two buffers in turn of up to eight values a warp (a thread that writes one again
// has passed the barrier of the other since). A group's slots begin at a multiple of four and are padded
// with zeros to 4 N4, the most warps that a row of this instance has.
template <int N4>
struct Meet {
  static constexpr int kSlots = 64, kFloats = 2 * 8 * kSlots;
  float* buf;  // [2][8][kSlots]
  int group, tpr, slot, base;
  __device__ __forceinline__ Meet(float* shared, int tpr_) : buf(shared), tpr(tpr_) {
    group = threadIdx.x / tpr;
    base = group * 4 * N4;
    slot = base + (threadIdx.x - group * tpr) / 32;
    for (int i = threadIdx.x; i < kFloats; i += blockDim.x) buf[i] = 0.f;
    __syncthreads();
  }
  // v[i] = its sum over the row's threads
  template <int N>
  __device__ __forceinline__ void sum(float (&v)[N], int& flip) const {
    constexpr int NP = N <= 1 ? 1 : N <= 2 ? 2 : N <= 4 ? 4 : 8, LANES = 32 / NP;
    const int lane = threadIdx.x & 31;
    float t[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) t[i] = i < N ? v[i] : 0.f;
    warp_sums<NP>(t);
    if constexpr (N4 > 0) {
      float* b = buf + flip;
      flip ^= 8 * kSlots;
      if (lane % LANES == 0) b[(lane / LANES) * kSlots + slot] = t[0];
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(tpr) : "memory");
      const float* from = b + (lane / LANES) * kSlots + base + lane % LANES;
      t[0] = 0.f;
#pragma unroll
      for (int w = 0; w < 4 * N4; w += LANES) t[0] += w + LANES <= 4 * N4 || w + lane % LANES < 4 * N4 ? from[w] : 0.f;
#pragma unroll
      for (int x = LANES / 2; x > 0; x >>= 1) t[0] += __shfl_xor_sync(0xffffffffu, t[0], x);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = NP == 1 ? t[0] : __shfl_sync(0xffffffffu, t[0], i * LANES);
  }
};

struct Share {
  int64_t r0, r1;  // rows of this block
  int seq;         // sequence of r0
};
__device__ __forceinline__ int64_t seq_begin(const GatedNormParams& p, int s) {
  return p.seq_start ? p.seq_start[s] : (s == 0 ? 0 : p.rows);
}
// The last sequence that begins at or before `row`, 32 candidates a step (every warp for itself).
__device__ __forceinline__ int seq_of(const GatedNormParams& p, int64_t row) {
  int lo = 0, n = p.seqs;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32, at = (threadIdx.x & 31) * step;
    const unsigned hit = __ballot_sync(0xffffffffu, at < n && seq_begin(p, lo + at) <= row);
    const int k = hit ? 31 - __clz(hit) : 0;  // begins only grow: the hits are the first lanes
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}
__device__ __forceinline__ Share share_of_block(const GatedNormParams& p) {
  Share s;
  s.r0 = p.rows * blockIdx.x / gridDim.x;
  s.r1 = p.rows * (blockIdx.x + 1) / gridDim.x;
  s.seq = seq_of(p, s.r0);
  return s;
}

__device__ __forceinline__ void wait_stages(int pending) {
  if (pending >= 3) cp_async_wait<3>();
  else if (pending == 2) cp_async_wait<2>();
  else if (pending == 1) cp_async_wait<1>();
  else cp_async_wait<0>();
}
template <typename T>
__device__ __forceinline__ T* at(const void* base, int row, int stride, int col) {
  return const_cast<T*>(static_cast<const T*>(base)) + (int64_t)row * stride + col;
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}

// The parameters of a sequence, combined: [gate post | weight (1 + scale) | shift], 8 columns a thread.
template <typename T, typename P>
__device__ __forceinline__ void load_params(const GatedNormParams& p, int seq, int col, bool on, float* gw, float* sw,
                                            float* sh) {
  if (!on) return;
  const int64_t row = (int64_t)seq * p.cols + col;
  V8 gate = splat(1.f), post = gate, weight = gate, scale = splat(0.f), shift = scale;
  if (p.gate) gate = Io<T, P>::load(p.gate, row);
  if (p.post_weight) post = Io<T, P>::load(p.post_weight, col);
  if (p.weight) weight = Io<T, P>::load(p.weight, col);
  if (p.scale) scale = Io<T, P>::load(p.scale, row);
  if (sh && p.shift) shift = Io<T, P>::load(p.shift, row);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    gate.v[i] = __fmul2_rn(gate.v[i], post.v[i]);
    weight.v[i] = __fmul2_rn(weight.v[i], __fadd2_rn(scale.v[i], pair(1.f)));
  }
  put_apart(gw, p.cols, col, gate);
  put_apart(sw, p.cols, col, weight);
  if (sh) put_apart(sh, p.cols, col, shift);
}

template <typename T, typename P, bool HAS_Y, int VPT, int N4, int MAXT>
__global__ void __launch_bounds__(MAXT) gated_norm_fwd_kernel(const __grid_constant__ GatedNormParams p) {
  constexpr int NIN = HAS_Y ? 2 : 1;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) float meeting[Meet<N4>::kFloats];
  const int tpr = p.tpr, groups = blockDim.x / tpr;
  const Meet<N4> meet(meeting, tpr);
  int flip = 0, col[VPT];
  bool on[VPT];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    col[v] = (v * tpr + (int)threadIdx.x - meet.group * tpr) * 8;
    on[v] = col[v] < p.cols;
  }
  float* gw = reinterpret_cast<float*>(smem);
  float *sw = gw + p.cols, *sh = sw + p.cols;
  const uint32_t ring = smem_u32(sh + p.cols) + threadIdx.x * 16, piece = blockDim.x * 16, stage = NIN * VPT * piece;
  const float inv_c = 1.f / (float)p.cols;
  const bool post = HAS_Y && p.post_weight != nullptr, layer = p.layer != 0;

  const Share s = share_of_block(p);
  int seq = s.seq;
  for (int64_t a = s.r0; a < s.r1;) {
    while (seq + 1 < p.seqs && seq_begin(p, seq + 1) <= a) ++seq;
    const int64_t b = min(s.r1, seq + 1 < p.seqs ? seq_begin(p, seq + 1) : p.rows);
    // rows of this group: a + group, a + group + groups, ...
    const int n = (int)max((b - a - meet.group + groups - 1) / groups, (int64_t)0);
    int to_load = n, load_row = (int)a + meet.group;
    uint32_t put = ring, get = ring;
    const uint32_t end = ring + p.stages * stage;
    auto issue = [&]() {
      if (to_load > 0) {
        --to_load;
#pragma unroll
        for (int v = 0; v < VPT; ++v)
          if (on[v]) {
            cp_async16(put + v * piece, at<T>(p.x, load_row, p.x_row, col[v]), 16);
            if (HAS_Y) cp_async16(put + (VPT + v) * piece, at<T>(p.y, load_row, p.y_row, col[v]), 16);
          }
        load_row += groups;
        put = put + stage == end ? ring : put + stage;
      }
      cp_async_commit();
    };
    for (int i = 0; i < p.stages - 1; ++i) issue();
    __syncthreads();  // the last run's parameters are no longer read
    if (meet.group == 0)
#pragma unroll
      for (int v = 0; v < VPT; ++v) load_params<T, P>(p, seq, col[v], on[v], gw, sw, sh);
    __syncthreads();
    int row = (int)a + meet.group;
    for (int it = 0; it < n; ++it, row += groups) {
      wait_stages(p.stages - 2);
      V8 x[VPT], y[HAS_Y ? VPT : 1];
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        x[v] = splat(0.f);
        if (on[v]) x[v] = unpack8<T>(ld_shared16(get + v * piece));
        if constexpr (HAS_Y) {
          y[v] = splat(0.f);
          if (on[v]) y[v] = unpack8<T>(ld_shared16(get + (VPT + v) * piece));
        }
      }
      get = get + stage == end ? ring : get + stage;
      issue();
      float ry = 1.f, mean = 0.f, rx[1] = {0.f};
      if constexpr (HAS_Y) {
        if (post) {
#pragma unroll
          for (int v = 0; v < VPT; ++v) rx[0] += dot8(y[v], y[v]);
        }
#pragma unroll
        for (int v = 0; v < VPT; ++v)
          if (on[v]) {
            const V8 g = get_apart(gw, p.cols, col[v]);
#pragma unroll
            for (int i = 0; i < 4; ++i) y[v].v[i] = __fmul2_rn(y[v].v[i], g.v[i]);
          }
        if (post && layer) {
          // x' = x + ry (g y) is linear in ry, so its mean comes out of the same meeting as ry
          float t[3] = {rx[0], 0.f, 0.f};
#pragma unroll
          for (int v = 0; v < VPT; ++v) {
            t[1] += sum8(x[v]);
            t[2] += sum8(y[v]);
          }
          meet.sum(t, flip);
          ry = rsqrtf(fmaf(t[0], inv_c, p.eps));
          mean = fmaf(t[2], ry, t[1]) * inv_c;
        } else if (post) {
          meet.sum(rx, flip);
          ry = rsqrtf(fmaf(rx[0], inv_c, p.eps));
        }
#pragma unroll
        for (int v = 0; v < VPT; ++v)
          if (on[v]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[v].v[i] = __ffma2_rn(y[v].v[i], pair(ry), x[v].v[i]);
            *reinterpret_cast<uint4*>(at<T>(p.x_new, row, p.cols, col[v])) = pack8<T>(x[v]);
          }
      }
      if (layer) {
        // the mean first, then squares of differences: no cancellation where the mean is large
        if (!post) {
          rx[0] = 0.f;
#pragma unroll
          for (int v = 0; v < VPT; ++v) rx[0] += sum8(x[v]);
          meet.sum(rx, flip);
          mean = rx[0] * inv_c;
        }
#pragma unroll
        for (int v = 0; v < VPT; ++v)
          if (on[v])
#pragma unroll
            for (int i = 0; i < 4; ++i) x[v].v[i] = __fadd2_rn(x[v].v[i], pair(-mean));
      }
      rx[0] = 0.f;
#pragma unroll
      for (int v = 0; v < VPT; ++v) rx[0] += dot8(x[v], x[v]);
      meet.sum(rx, flip);
      rx[0] = rsqrtf(fmaf(rx[0], inv_c, p.eps));
#pragma unroll
      for (int v = 0; v < VPT; ++v)
        if (on[v]) {
          const V8 w = get_apart(sw, p.cols, col[v]), t = get_apart(sh, p.cols, col[v]);
          V8 h;
#pragma unroll
          for (int i = 0; i < 4; ++i) h.v[i] = __ffma2_rn(__fmul2_rn(x[v].v[i], pair(rx[0])), w.v[i], t.v[i]);
          *reinterpret_cast<uint4*>(at<T>(p.h, row, p.cols, col[v])) = pack8<T>(h);
          if (p.stats && col[v] == 0) {
            p.stats[row] = ry;
            p.stats[p.rows + row] = mean;
            p.stats[2 * p.rows + row] = rx[0];
          }
        }
    }
    cp_async_wait<0>();
    a = b;
  }
}

template <typename T, typename P, bool HAS_Y, int N4, int MAXT>
__global__ void __launch_bounds__(MAXT) gated_norm_bwd_kernel(const __grid_constant__ GatedNormParams p) {
  constexpr int NIN = HAS_Y ? 4 : 3;  // x, dh, dx', y
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) float meeting[Meet<N4>::kFloats];
  const int tpr = p.tpr, groups = blockDim.x / tpr;
  const Meet<N4> meet(meeting, tpr);
  const int group = meet.group, col = ((int)threadIdx.x - group * tpr) * 8;
  const bool on = col < p.cols;
  int flip = 0;
  float* gw = reinterpret_cast<float*>(smem);
  float* sw = gw + p.cols;
  const uint32_t ring = smem_u32(sw + p.cols) + threadIdx.x * 16, piece = blockDim.x * 16, stage = NIN * piece;
  const float inv_c = 1.f / (float)p.cols;
  const bool post = HAS_Y && p.post_weight != nullptr;

  const Share s = share_of_block(p);
  int seq = s.seq;
  for (int64_t a = s.r0; a < s.r1;) {
    while (seq + 1 < p.seqs && seq_begin(p, seq + 1) <= a) ++seq;
    const int64_t b = min(s.r1, seq + 1 < p.seqs ? seq_begin(p, seq + 1) : p.rows);
    const int n = (int)max((b - a - group + groups - 1) / groups, (int64_t)0);
    int to_load = n, load_row = (int)a + group;
    uint32_t put = ring, get = ring;
    const uint32_t end = ring + p.stages * stage;
    auto issue = [&]() {
      if (to_load > 0) {
        --to_load;
        if (on) {
          cp_async16(put, at<T>(p.x, load_row, p.x_row, col), 16);
          if (p.dh) cp_async16(put + piece, at<T>(p.dh, load_row, p.dh_row, col), 16);
          if (p.dx_new) cp_async16(put + 2 * piece, at<T>(p.dx_new, load_row, p.dx_new_row, col), 16);
          if (HAS_Y) cp_async16(put + 3 * piece, at<T>(p.y, load_row, p.y_row, col), 16);
        }
        load_row += groups;
        put = put + stage == end ? ring : put + stage;
      }
      cp_async_commit();
    };
    for (int i = 0; i < p.stages - 1; ++i) issue();
    __syncthreads();  // the last run's parameters and sums are no longer read
    if (group == 0) load_params<T, P>(p, seq, col, on, gw, sw, nullptr);
    __syncthreads();
    V8 sa = splat(0.f), sb = sa, sc = sa;
    int row = (int)a + group;
    // the rows' statistics, one row ahead of their use
    float nry = 0.f, nmean = 0.f, nrx = 0.f;
    auto load_stats = [&](int r) {
      nry = p.stats[r];
      nmean = p.stats[p.rows + r];
      nrx = p.stats[2 * p.rows + r];
    };
    if (n > 0) load_stats(row);
    for (int it = 0; it < n; ++it, row += groups) {
      wait_stages(p.stages - 2);
      const float ry = nry, mean = nmean, rx = nrx;
      V8 xn, yn, dh;  // n, y ry and dh of the formulas; columns past the width hold zeros
      auto read = [&]() {
        xn = yn = dh = splat(0.f);
        if (!on) return;
        xn = unpack8<T>(ld_shared16(get));
        if (p.dh) dh = unpack8<T>(ld_shared16(get + piece));
        if constexpr (HAS_Y) {
          yn = unpack8<T>(ld_shared16(get + 3 * piece));
          const V8 g = get_apart(gw, p.cols, col);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            yn.v[i] = __fmul2_rn(yn.v[i], pair(ry));
            xn.v[i] = __ffma2_rn(g.v[i], yn.v[i], xn.v[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) xn.v[i] = __fmul2_rn(__fadd2_rn(xn.v[i], pair(-mean)), pair(rx));
      };
      auto weigh = [&]() {  // dh -> g of the formulas
        if (!on) return;
        const V8 w = get_apart(sw, p.cols, col);
#pragma unroll
        for (int i = 0; i < 4; ++i) dh.v[i] = __fmul2_rn(dh.v[i], w.v[i]);
      };
      read();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sb.v[i] = __ffma2_rn(dh.v[i], xn.v[i], sb.v[i]);
        sc.v[i] = __fadd2_rn(sc.v[i], dh.v[i]);
      }
      weigh();
      float acc[2] = {dot8(dh, xn), sum8(dh)};
      V8 dx = splat(0.f);
      auto read_dx = [&]() {
        if (on && p.dx_new) dx = unpack8<T>(ld_shared16(get + 2 * piece));
      };
      auto next = [&]() {
        get = get + stage == end ? ring : get + stage;
        issue();
      };
      read_dx();
      next();
      if (it + 1 < n) load_stats(row + groups);
      meet.sum(acc, flip);
      const float2 gn = pair(-acc[0] * inv_c * rx), gm = pair(p.layer ? -acc[1] * inv_c * rx : 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dx.v[i] = __fadd2_rn(dx.v[i], __ffma2_rn(dh.v[i], pair(rx), __ffma2_rn(xn.v[i], gn, gm)));
        if constexpr (HAS_Y) sa.v[i] = __ffma2_rn(dx.v[i], yn.v[i], sa.v[i]);
      }
      if (on) *reinterpret_cast<uint4*>(at<T>(p.dx, row, p.cols, col)) = pack8<T>(dx);
      if constexpr (HAS_Y) {
        V8 t = splat(0.f);  // t of the formulas
        if (on) {
          const V8 g = get_apart(gw, p.cols, col);
#pragma unroll
          for (int i = 0; i < 4; ++i) t.v[i] = __fmul2_rn(dx.v[i], g.v[i]);
        }
        if (post) {
          float dot[1] = {dot8(t, yn)};
          meet.sum(dot, flip);
          const float2 m = pair(-dot[0] * inv_c * ry);
#pragma unroll
          for (int i = 0; i < 4; ++i) t.v[i] = __ffma2_rn(yn.v[i], m, __fmul2_rn(t.v[i], pair(ry)));
        }
        if (on) *reinterpret_cast<uint4*>(at<T>(p.dy, row, p.cols, col)) = pack8<T>(t);
      }
    }
    cp_async_wait<0>();
    if (p.part) {
      // this block's column sums of the sequence: slot blockIdx + seq (both only grow, so no two share one)
      float* out = p.part + ((int64_t)blockIdx.x + seq) * 3 * p.cols;
      if (groups > 1) {
        // the groups' sums one after another through the parameters' place ([gw | sw] and the ring behind it)
        __syncthreads();
        for (int g2 = 0; g2 < groups; ++g2) {
          if (group == g2 && on) {
            float* acc3 = reinterpret_cast<float*>(smem);
#pragma unroll
            for (int q = 0; q < 3; ++q) {
              V8& mine = q == 0 ? sa : q == 1 ? sb : sc;
              if (g2 > 0) {
                const V8 f = get8(acc3 + q * p.cols + col);
#pragma unroll
                for (int i = 0; i < 4; ++i) mine.v[i] = __fadd2_rn(mine.v[i], f.v[i]);
              }
              put8(acc3 + q * p.cols + col, mine);
              if (g2 == groups - 1) put8(out + q * p.cols + col, mine);
            }
          }
          __syncthreads();
        }
      } else if (on) {
        put8(out + col, sa);
        put8(out + p.cols + col, sb);
        put8(out + 2 * p.cols + col, sc);
      }
    }
    a = b;
  }
}

// The same for wide rows. A row is read from the ring twice: once for its five sums (dx = dx' + rx (g - mean(g) - n mean(g n)) is linear in its
// two means, so with the sums of u (dx' + rx g), u and u n, u = y ry gate post_weight, the sum over t y ry comes out
// of the same meeting), once for the outputs; only the column sums live in registers throughout.
template <typename T, typename P, bool HAS_Y, int VPT, int N4, int MAXT>
__global__ void __launch_bounds__(MAXT) gated_norm_bwd_wide_kernel(const __grid_constant__ GatedNormParams p) {
  constexpr int NIN = HAS_Y ? 4 : 3;  // x, dh, dx', y
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) float meeting[Meet<N4>::kFloats];
  const int tpr = p.tpr, groups = blockDim.x / tpr;
  const Meet<N4> meet(meeting, tpr);
  const int group = meet.group;
  int flip = 0, col[VPT];
  bool on[VPT];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    col[v] = (v * tpr + (int)threadIdx.x - group * tpr) * 8;
    on[v] = col[v] < p.cols;
  }
  float* gw = reinterpret_cast<float*>(smem);
  float* sw = gw + p.cols;
  const uint32_t ring = smem_u32(sw + p.cols) + threadIdx.x * 16, piece = blockDim.x * 16, stage = NIN * VPT * piece;
  const float inv_c = 1.f / (float)p.cols;
  const bool post = HAS_Y && p.post_weight != nullptr;

  const Share s = share_of_block(p);
  int seq = s.seq;
  for (int64_t a = s.r0; a < s.r1;) {
    while (seq + 1 < p.seqs && seq_begin(p, seq + 1) <= a) ++seq;
    const int64_t b = min(s.r1, seq + 1 < p.seqs ? seq_begin(p, seq + 1) : p.rows);
    const int n = (int)max((b - a - group + groups - 1) / groups, (int64_t)0);
    int to_load = n, load_row = (int)a + group;
    uint32_t put = ring, get = ring;
    const uint32_t end = ring + p.stages * stage;
    auto issue = [&]() {
      if (to_load > 0) {
        --to_load;
#pragma unroll
        for (int v = 0; v < VPT; ++v)
          if (on[v]) {
            cp_async16(put + v * piece, at<T>(p.x, load_row, p.x_row, col[v]), 16);
            if (p.dh) cp_async16(put + (VPT + v) * piece, at<T>(p.dh, load_row, p.dh_row, col[v]), 16);
            if (p.dx_new) cp_async16(put + (2 * VPT + v) * piece, at<T>(p.dx_new, load_row, p.dx_new_row, col[v]), 16);
            if (HAS_Y) cp_async16(put + (3 * VPT + v) * piece, at<T>(p.y, load_row, p.y_row, col[v]), 16);
          }
        load_row += groups;
        put = put + stage == end ? ring : put + stage;
      }
      cp_async_commit();
    };
    for (int i = 0; i < p.stages - 1; ++i) issue();
    __syncthreads();  // the last run's parameters and sums are no longer read
    if (group == 0)
#pragma unroll
      for (int v = 0; v < VPT; ++v) load_params<T, P>(p, seq, col[v], on[v], gw, sw, nullptr);
    __syncthreads();
    V8 sa[VPT], sb[VPT], sc[VPT];
#pragma unroll
    for (int v = 0; v < VPT; ++v) sa[v] = sb[v] = sc[v] = splat(0.f);
    int row = (int)a + group;
    // the rows' statistics, one row ahead of their use
    float nry = 0.f, nmean = 0.f, nrx = 0.f;
    auto load_stats = [&](int r) {
      nry = p.stats[r];
      nmean = p.stats[p.rows + r];
      nrx = p.stats[2 * p.rows + r];
    };
    if (n > 0) load_stats(row);
    for (int it = 0; it < n; ++it, row += groups) {
      issue();  // into the stage that the last row was read from
      wait_stages(p.stages - 1);
      const float ry = nry, mean = nmean, rx = nrx;
      // n, y ry, dh and dx' of the formulas, gate post_weight, weight (1 + scale), for one vector of columns
      V8 xn, yn, dh, dx, g, w;
      auto read = [&](int v) {
        xn = unpack8<T>(ld_shared16(get + v * piece));
        dh = dx = splat(0.f);
        if (p.dh) dh = unpack8<T>(ld_shared16(get + (VPT + v) * piece));
        if (p.dx_new) dx = unpack8<T>(ld_shared16(get + (2 * VPT + v) * piece));
        w = get_apart(sw, p.cols, col[v]);
        if constexpr (HAS_Y) {
          yn = unpack8<T>(ld_shared16(get + (3 * VPT + v) * piece));
          g = get_apart(gw, p.cols, col[v]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            yn.v[i] = __fmul2_rn(yn.v[i], pair(ry));
            xn.v[i] = __ffma2_rn(g.v[i], yn.v[i], xn.v[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) xn.v[i] = __fmul2_rn(__fadd2_rn(xn.v[i], pair(-mean)), pair(rx));
      };
      float acc[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < VPT; ++v)
        if (on[v]) {
          read(v);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sb[v].v[i] = __ffma2_rn(dh.v[i], xn.v[i], sb[v].v[i]);
            sc[v].v[i] = __fadd2_rn(sc[v].v[i], dh.v[i]);
            dh.v[i] = __fmul2_rn(dh.v[i], w.v[i]);  // g of the formulas
          }
          acc[0] += dot8(dh, xn);
          acc[1] += sum8(dh);
          if (post) {
            V8 u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              u.v[i] = __fmul2_rn(yn.v[i], g.v[i]);
              dx.v[i] = __ffma2_rn(dh.v[i], pair(rx), dx.v[i]);
            }
            acc[2] += dot8(u, dx);
            acc[3] += sum8(u);
            acc[4] += dot8(u, xn);
          }
        }
      if (it + 1 < n) load_stats(row + groups);
      if (post) {
        meet.sum(acc, flip);
      } else {
        float two[2] = {acc[0], acc[1]};
        meet.sum(two, flip);
        acc[0] = two[0];
        acc[1] = two[1];
      }
      const float gn = -acc[0] * inv_c * rx, gm = p.layer ? -acc[1] * inv_c * rx : 0.f;
      const float m = -fmaf(gm, acc[3], fmaf(gn, acc[4], acc[2])) * inv_c;  // -mean(t y ry)
#pragma unroll
      for (int v = 0; v < VPT; ++v)
        if (on[v]) {
          read(v);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dh.v[i] = __fmul2_rn(dh.v[i], w.v[i]);
            dx.v[i] = __fadd2_rn(dx.v[i], __ffma2_rn(dh.v[i], pair(rx), __ffma2_rn(xn.v[i], pair(gn), pair(gm))));
            if constexpr (HAS_Y) {
              sa[v].v[i] = __ffma2_rn(dx.v[i], yn.v[i], sa[v].v[i]);
              dh.v[i] = __fmul2_rn(dx.v[i], g.v[i]);  // t of the formulas
              if (post) dh.v[i] = __fmul2_rn(__ffma2_rn(yn.v[i], pair(m), dh.v[i]), pair(ry));
            }
          }
          *reinterpret_cast<uint4*>(at<T>(p.dx, row, p.cols, col[v])) = pack8<T>(dx);
          if constexpr (HAS_Y) *reinterpret_cast<uint4*>(at<T>(p.dy, row, p.cols, col[v])) = pack8<T>(dh);
        }
      get = get + stage == end ? ring : get + stage;
    }
    cp_async_wait<0>();
    if (p.part) {
      // this block's column sums of the sequence: slot blockIdx + seq (both only grow, so no two share one). The
      // groups' sums one after another through shared memory (the parameters' place and the ring behind it)
      float* out = p.part + ((int64_t)blockIdx.x + seq) * 3 * p.cols;
      float* sums = reinterpret_cast<float*>(smem);
      if (groups > 1) __syncthreads();
      for (int g2 = 0; g2 < groups; ++g2) {
        if (group == g2)
#pragma unroll
          for (int v = 0; v < VPT; ++v)
            if (on[v])
#pragma unroll
              for (int q = 0; q < 3; ++q) {
                V8& mine = q == 0 ? sa[v] : q == 1 ? sb[v] : sc[v];
                if (g2 > 0) {
                  const V8 f = get_apart(sums + q * p.cols, p.cols, col[v]);
#pragma unroll
                  for (int i = 0; i < 4; ++i) mine.v[i] = __fadd2_rn(mine.v[i], f.v[i]);
                }
                if (g2 == groups - 1) put8(out + q * p.cols + col[v], mine);
                else put_apart(sums + q * p.cols, p.cols, col[v], mine);
              }
        if (groups > 1) __syncthreads();
      }
    }
    a = b;
  }
}

template <typename P>
__device__ __forceinline__ float param(const void* t, int64_t i, float none) {
  if (!t) return none;
  if constexpr (sizeof(P) == 4) return static_cast<const float*>(t)[i];
  else return Elem<P>::to_f(static_cast<const P*>(t)[i]);
}
template <typename P>
__device__ __forceinline__ void put_param(void* t, int64_t i, float v) {
  if (!t) return;
  if constexpr (sizeof(P) == 4) static_cast<float*>(t)[i] = v;
  else static_cast<P*>(t)[i] = Elem<P>::from_f(v);
}

// Sums a sequence's partial rows: block = (32 columns, sequence), 16 groups over the blocks that hold rows of it.
template <typename P>
__global__ void __launch_bounds__(512) gated_norm_sums_kernel(const __grid_constant__ GatedNormParams p, int blocks) {
  __shared__ float red[3][16][33];
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, seq = blockIdx.y;
  const int c = blockIdx.x * 32 + lane;
  const int64_t b0 = seq_begin(p, seq), b1 = seq + 1 < p.seqs ? seq_begin(p, seq + 1) : p.rows;
  float v[3] = {0.f, 0.f, 0.f};
  if (b1 > b0 && c < p.cols) {
    // block holding row r: the last k with rows * k / blocks <= r
    const int k0 = (int)(((b0 + 1) * blocks - 1) / p.rows), k1 = (int)((b1 * blocks - 1) / p.rows);
#pragma unroll 4
    for (int k = k0 + grp; k <= k1; k += 16)
#pragma unroll
      for (int q = 0; q < 3; ++q) v[q] += p.part[(((int64_t)k + seq) * 3 + q) * p.cols + c];
  }
#pragma unroll
  for (int q = 0; q < 3; ++q) red[q][grp][lane] = v[q];
  __syncthreads();
  if (grp || c >= p.cols) return;
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    v[q] = 0.f;
    for (int g = 0; g < 16; ++g) v[q] += red[q][g][lane];
  }
  const int64_t at = (int64_t)seq * p.cols + c;
  put_param<P>(p.dgate, at, v[0] * param<P>(p.post_weight, c, 1.f));
  put_param<P>(p.dscale, at, v[1] * param<P>(p.weight, c, 1.f));
  put_param<P>(p.dshift, at, v[2]);
  const float dp = v[0] * param<P>(p.gate, at, 1.f), dw = v[1] * (1.f + param<P>(p.scale, at, 0.f));
  if (p.seqs == 1) {
    put_param<P>(p.dpost_weight, c, dp);
    put_param<P>(p.dweight, c, dw);
  } else if (p.dpost_weight || p.dweight) {
    p.seq_part[at * 2] = dp;
    p.seq_part[at * 2 + 1] = dw;
  }
}
// The weights' gradients over the sequences, in order.
template <typename P>
__global__ void __launch_bounds__(128) gated_norm_weights_kernel(const __grid_constant__ GatedNormParams p) {
  const int c = blockIdx.x * 128 + threadIdx.x;
  if (c >= p.cols) return;
  float a = 0.f, b = 0.f;
#pragma unroll 8
  for (int s = 0; s < p.seqs; ++s) {
    const float2 v = *reinterpret_cast<const float2*>(p.seq_part + ((int64_t)s * p.cols + c) * 2);
    a += v.x;
    b += v.y;
  }
  put_param<P>(p.dpost_weight, c, a);
  put_param<P>(p.dweight, c, b);
}

// ------------------------------------------------------------------------------------ host
// Threads that hold a row of 8 vpt columns each, whole warps.
int row_threads(int cols, int vpt) { return (cols / (8 * vpt) + (cols % (8 * vpt) ? 1 : 0) + 31) / 32 * 32; }

struct Shape {
  int threads, tpr, stages, blocks, smem;
};
// `most` threads or one row; as many stages, up to four, as fit beside the combined parameters; every block
// that is resident gets an equal share of the rows.
Shape shape_of(int cols, int64_t rows, int vpt, int most, int per_sm, int nparam, int nin) {
  Shape s;
  s.tpr = row_threads(cols, vpt);
  int groups = std::min(16, std::max(1, most / s.tpr));
  const int row = s.tpr * 16 * nin * vpt, par = nparam * cols * 4;
  while (groups > 1 && par + 2 * groups * row > kSmemLimit) --groups;
  s.threads = s.tpr * groups;
  const int stage = groups * row;
  while (per_sm > 1 && par + 3 * stage > kSmemLimit / per_sm) --per_sm;
  s.stages = std::max(2, std::min(4, (kSmemLimit / per_sm - par) / stage));
  // the groups' column sums pass through three rows of the shared memory
  s.smem = std::max(par + s.stages * stage, groups > 1 ? 3 * cols * 4 : 0);
  s.blocks = (int)std::min<int64_t>(rows, (int64_t)148 * per_sm);
  return s;
}

template <typename Kern>
cudaError_t run(Kern kern, std::atomic<uint64_t>& ready, const Shape& s, GatedNormParams p, cudaStream_t st) {
  cudaError_t e = allow_smem(kern, kSmemLimit, ready);
  if (e != cudaSuccess) return e;
  p.tpr = s.tpr;
  p.stages = s.stages;
  kern<<<s.blocks, s.threads, s.smem, st>>>(p);
  return cudaGetLastError();
}

// Forward. Few rows (a serving step: one a block at most): one vector a thread, the shortest way through a row
// (24 rows of 5120, two rms norms: 5.2 us, with four vectors 7.4 us, replayed in a graph). Else four vectors a thread: a row's sums then cost a
// quarter per column, and four rows of 5120 columns are under way on an SM with 640 threads (16576 rows, layer
// norm with a post norm: 119 us, two vectors 130 us; the floor is 104 us). Rows that would leave lanes
// without a vector take fewer, and so do rows so wide that four vectors would leave an SM less than 512 threads.
template <typename T, typename P, bool Y>
cudaError_t forward(const GatedNormParams& p, cudaStream_t st) {
  static std::atomic<uint64_t> ready[10];
  const int nin = Y ? 2 : 1;
  if (p.rows <= 148 || p.cols <= 256) {
    const Shape s = shape_of(p.cols, p.rows, 1, p.rows <= 148 ? 1 : 640, 1, 3, nin);
    if (s.tpr <= 32) return run(gated_norm_fwd_kernel<T, P, Y, 1, 0, 1024>, ready[0], s, p, st);
    if (s.tpr <= 128) return run(gated_norm_fwd_kernel<T, P, Y, 1, 1, 1024>, ready[1], s, p, st);
    if (s.tpr <= 256) return run(gated_norm_fwd_kernel<T, P, Y, 1, 2, 1024>, ready[2], s, p, st);
    if (s.tpr <= 640) return run(gated_norm_fwd_kernel<T, P, Y, 1, 5, 1024>, ready[3], s, p, st);
    return run(gated_norm_fwd_kernel<T, P, Y, 1, 8, 1024>, ready[4], s, p, st);
  }
  if (p.cols <= 512) return run(gated_norm_fwd_kernel<T, P, Y, 2, 0, 640>, ready[5], shape_of(p.cols, p.rows, 2, 640, 1, 3, nin), p, st);
  const Shape s = shape_of(p.cols, p.rows, 4, 640, 1, 3, nin);
  if (s.tpr <= 32) return run(gated_norm_fwd_kernel<T, P, Y, 4, 0, 640>, ready[6], s, p, st);
  if (s.tpr <= 128) return run(gated_norm_fwd_kernel<T, P, Y, 4, 1, 640>, ready[7], s, p, st);
  if (s.threads < 512) return run(gated_norm_fwd_kernel<T, P, Y, 2, 4, 640>, ready[8], shape_of(p.cols, p.rows, 2, 640, 1, 3, nin), p, st);
  return run(gated_norm_fwd_kernel<T, P, Y, 4, 2, 640>, ready[9], s, p, st);
}

// Backward: one vector a thread, whose row lives in registers between its two readings (16576 rows of 5120
// columns: 213 us, read twice with two vectors a thread 283 us; the floor is 157 us). Rows of more than 640
// threads would spill at one vector: two vectors a thread there, read twice (10360 rows of 8192 columns: 245 us, the
// other way 485 us).
bool wide(const GatedNormParams& p) { return row_threads(p.cols, 1) > 640; }
Shape backward_shape(const GatedNormParams& p) {
  const int nin = p.y ? 4 : 3;
  if (wide(p)) return shape_of(p.cols, p.rows, 2, 512, 1, 2, nin);
  return shape_of(p.cols, p.rows, 1, 256, row_threads(p.cols, 1) <= 256 ? 2 : 1, 2, nin);
}
template <typename T, typename P, bool Y>
cudaError_t backward(const GatedNormParams& p, cudaStream_t st) {
  const Shape s = backward_shape(p);
  if (p.rows > 0) {
    static std::atomic<uint64_t> ready[5];
    cudaError_t e;
    if (wide(p)) e = run(gated_norm_bwd_wide_kernel<T, P, Y, 2, 4, 512>, ready[4], s, p, st);
    else if (s.tpr <= 32) e = run(gated_norm_bwd_kernel<T, P, Y, 0, 256>, ready[0], s, p, st);
    else if (s.tpr <= 128) e = run(gated_norm_bwd_kernel<T, P, Y, 1, 256>, ready[1], s, p, st);
    else if (s.tpr <= 256) e = run(gated_norm_bwd_kernel<T, P, Y, 2, 256>, ready[2], s, p, st);
    else e = run(gated_norm_bwd_kernel<T, P, Y, 5, 640>, ready[3], s, p, st);
    if (e != cudaSuccess) return e;
  }
  if (!p.part) return cudaSuccess;
  gated_norm_sums_kernel<P><<<dim3((p.cols + 31) / 32, p.seqs), 512, 0, st>>>(p, s.blocks);
  if (p.seqs > 1 && (p.dpost_weight || p.dweight))
    gated_norm_weights_kernel<P><<<(p.cols + 127) / 128, 128, 0, st>>>(p);
  return cudaGetLastError();
}

template <typename T, typename P>
cudaError_t dispatch(const GatedNormParams& p, bool bwd, cudaStream_t st) {
  if (bwd) return p.y ? backward<T, P, true>(p, st) : backward<T, P, false>(p, st);
  return p.y ? forward<T, P, true>(p, st) : forward<T, P, false>(p, st);
}
template <typename T>
cudaError_t dispatch_params(const GatedNormParams& p, bool f32, bool bwd, cudaStream_t st) {
  return f32 ? dispatch<T, float>(p, bwd, st) : dispatch<T, T>(p, bwd, st);
}

}  // namespace

int gated_norm_blocks(const GatedNormParams& p) { return backward_shape(p).blocks; }

cudaError_t gated_norm(const GatedNormParams& p, bool bf16, bool f32_params, bool bwd, cudaStream_t st) {
  return bf16 ? dispatch_params<__nv_bfloat16>(p, f32_params, bwd, st) : dispatch_params<__half>(p, f32_params, bwd, st);
}

}  // namespace vmb
