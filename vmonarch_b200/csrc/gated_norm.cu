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
// share of all rows; TPR threads hold a row, 8 columns each, and go through the share R rows at a time
// behind a ring of cp.async stages, in which every thread reads back only what it loaded itself. What the
// row-wise work needs of the parameters (gate post_weight, weight (1 + scale), shift) is combined once per
// sequence into shared memory: from L2 it would be more than the rows' own traffic. The column sums
// of the backward stay in registers over a block's rows of a sequence; each (block, sequence) leaves one
// 32-bit partial row, added in a fixed order by a second kernel.
#include <algorithm>

#include "common.cuh"
#include "gated_norm.h"
#include "launch.h"

namespace vmb {
namespace {

constexpr int kMaxWarps = 32;
constexpr int kSmemLimit = 220 * 1024;  // dynamic shared memory of an SM's blocks together

template <typename T, typename P>
struct Io;  // 8 elements of a parameter as floats
template <typename T>
struct Io<T, float> {
  static __device__ __forceinline__ void load(const void* base, int64_t at, float* f) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
};
template <typename T>
__device__ __forceinline__ void unpack8(uint4 v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = Elem<T>::unpack(w[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(Elem<T>::pack(f[0], f[1]), Elem<T>::pack(f[2], f[3]), Elem<T>::pack(f[4], f[5]), Elem<T>::pack(f[6], f[7]));
}
template <typename T>
struct Io<T, T> {
  static __device__ __forceinline__ void load(const void* base, int64_t at, float* f) {
    unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(base) + at), f);
  }
};

__device__ __forceinline__ void put8(float* s, const float* f) {
  reinterpret_cast<float4*>(s)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(s)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void get8(const float* s, float* f) {
  const float4 a = reinterpret_cast<const float4*>(s)[0], b = reinterpret_cast<const float4*>(s)[1];
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// Sums N values over the `wpr` warps of a row's threads. sums: [2][N][kMaxWarps + pad], alternating.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* sums, int& flip, int group, int wpr) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], s);
  if (wpr == 1) return;
  // two buffers in turn: a thread that writes one again has passed the barrier of the other since
  float* b = sums + flip * (4 * kMaxWarps);
  flip ^= 1;
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) b[i * kMaxWarps + (threadIdx.x >> 5)] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float t = 0.f;
    for (int w = 0; w < wpr; ++w) t += b[i * kMaxWarps + group * wpr + w];
    v[i] = t;
  }
}

struct Share {
  int64_t r0, r1;  // rows of this block
  int seq;         // sequence of r0
};
__device__ __forceinline__ int64_t seq_begin(const GatedNormParams& p, int s) {
  return p.seq_start ? p.seq_start[s] : (s == 0 ? 0 : p.rows);
}
__device__ __forceinline__ Share share_of_block(const GatedNormParams& p) {
  Share s;
  s.r0 = p.rows * blockIdx.x / gridDim.x;
  s.r1 = p.rows * (blockIdx.x + 1) / gridDim.x;
  int lo = 0, hi = p.seqs;  // last sequence that begins at or before r0
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (seq_begin(p, mid) <= s.r0) lo = mid;
    else hi = mid;
  }
  s.seq = lo;
  return s;
}

// NIN row tensors, R rows a stage and group: the ring of this thread's 16-byte pieces.
template <int NIN, int R>
struct Ring {
  uint8_t* base;
  int stages;
  __device__ __forceinline__ uint4* at(int stage, int r, int in) const {
    return reinterpret_cast<uint4*>(base) + ((stage * R + r) * NIN + in) * blockDim.x + threadIdx.x;
  }
};
__device__ __forceinline__ void wait_stages(int pending) {
  if (pending >= 3) cp_async_wait<3>();
  else if (pending == 2) cp_async_wait<2>();
  else if (pending == 1) cp_async_wait<1>();
  else cp_async_wait<0>();
}

// The parameters of a sequence, combined: [gate post | weight (1 + scale) | shift], 8 columns a thread.
template <typename T, typename P>
__device__ __forceinline__ void load_params(const GatedNormParams& p, int seq, int col, bool on, float* gw, float* sw,
                                            float* sh) {
  float a[8], b[8];
  auto one = [&](float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 1.f;
  };
  if (!on) return;
  const int64_t row = (int64_t)seq * p.cols + col;
  one(a);
  one(b);
  if (p.gate) Io<T, P>::load(p.gate, row, a);
  if (p.post_weight) Io<T, P>::load(p.post_weight, col, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] *= b[i];
  put8(gw + col, a);
  one(a);
  one(b);
  if (p.weight) Io<T, P>::load(p.weight, col, a);
  if (p.scale) {
    Io<T, P>::load(p.scale, row, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] += 1.f;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] *= b[i];
  put8(sw + col, a);
  if (sh) {
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = 0.f;
    if (p.shift) Io<T, P>::load(p.shift, row, a);
    put8(sh + col, a);
  }
}

template <typename T, typename P, bool HAS_Y, int R, int MAXT>
__global__ void __launch_bounds__(MAXT) gated_norm_fwd_kernel(const __grid_constant__ GatedNormParams p) {
  constexpr int NIN = HAS_Y ? 2 : 1;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float sums[2 * 4 * kMaxWarps];
  const int tpr = p.tpr, wpr = tpr >> 5, group = threadIdx.x / tpr, groups = blockDim.x / tpr;
  const int col = (threadIdx.x % tpr) * 8;
  const bool on = col < p.cols;
  float* gw = reinterpret_cast<float*>(smem);
  float *sw = gw + p.cols, *sh = sw + p.cols;
  const Ring<NIN, R> ring{reinterpret_cast<uint8_t*>(sh + p.cols), p.stages};
  const float inv_c = 1.f / (float)p.cols;
  const bool post = HAS_Y && p.post_weight != nullptr, layer = p.layer != 0;
  int flip = 0;

  const Share s = share_of_block(p);
  int seq = s.seq;
  for (int64_t a = s.r0; a < s.r1;) {
    while (seq + 1 < p.seqs && seq_begin(p, seq + 1) <= a) ++seq;
    const int64_t b = min(s.r1, seq + 1 < p.seqs ? seq_begin(p, seq + 1) : p.rows);
    const int n = (int)((b - a + (int64_t)groups * R - 1) / (groups * R));  // stages of this run of rows
    auto row_of = [&](int it, int r) { return a + ((int64_t)it * groups + group) * R + r; };
    auto issue = [&](int it) {
      if (it < n && on)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int64_t row = row_of(it, r);
          if (row >= b) continue;
          cp_async16(smem_u32(ring.at(it % p.stages, r, 0)), static_cast<const T*>(p.x) + row * p.x_row + col, 16);
          if (HAS_Y) cp_async16(smem_u32(ring.at(it % p.stages, r, NIN - 1)), static_cast<const T*>(p.y) + row * p.y_row + col, 16);
        }
      cp_async_commit();
    };
    for (int i = 0; i < p.stages - 1; ++i) issue(i);
    __syncthreads();  // the last run's parameters are no longer read
    if (group == 0) load_params<T, P>(p, seq, col, on, gw, sw, sh);
    __syncthreads();
    for (int it = 0; it < n; ++it) {
      wait_stages(p.stages - 2);
      float x[R][8], y[HAS_Y ? R : 1][8], acc[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool live = on && row_of(it, r) < b;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        unpack8<T>(live ? *ring.at(it % p.stages, r, 0) : zero, x[r]);
        if constexpr (HAS_Y) unpack8<T>(live ? *ring.at(it % p.stages, r, 1) : zero, y[r]);
      }
      issue(it + p.stages - 1);
      float ry[R], mean[R], rx[R];
#pragma unroll
      for (int r = 0; r < R; ++r) ry[r] = 1.f, mean[r] = 0.f;
      if constexpr (HAS_Y) {
        if (post) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            acc[r] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[r] = fmaf(y[r][i], y[r][i], acc[r]);
          }
          row_sum<R>(acc, sums, flip, group, wpr);
#pragma unroll
          for (int r = 0; r < R; ++r) ry[r] = rsqrtf(fmaf(acc[r], inv_c, p.eps));
        }
        float g[8];
        if (on) get8(gw + col, g);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[r][i] = on ? fmaf(g[i], y[r][i] * ry[r], x[r][i]) : 0.f;
      }
      if (layer) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          acc[r] = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[r] += x[r][i];
        }
        row_sum<R>(acc, sums, flip, group, wpr);
#pragma unroll
        for (int r = 0; r < R; ++r) mean[r] = acc[r] * inv_c;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        acc[r] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float d = on ? x[r][i] - mean[r] : 0.f;
          acc[r] = fmaf(d, d, acc[r]);
        }
      }
      row_sum<R>(acc, sums, flip, group, wpr);
#pragma unroll
      for (int r = 0; r < R; ++r) rx[r] = rsqrtf(fmaf(acc[r], inv_c, p.eps));
      if (on) {
        float w[8], t[8];
        get8(sw + col, w);
        get8(sh + col, t);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int64_t row = row_of(it, r);
          if (row >= b) continue;
          if (HAS_Y) *reinterpret_cast<uint4*>(static_cast<T*>(p.x_new) + row * p.cols + col) = pack8<T>(x[r]);
          float h[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) h[i] = fmaf((x[r][i] - mean[r]) * rx[r], w[i], t[i]);
          *reinterpret_cast<uint4*>(static_cast<T*>(p.h) + row * p.cols + col) = pack8<T>(h);
          if (p.stats && col == 0) {
            p.stats[row] = ry[r];
            p.stats[p.rows + row] = mean[r];
            p.stats[2 * p.rows + row] = rx[r];
          }
        }
      }
    }
    cp_async_wait<0>();
    a = b;
  }
}

template <typename T, typename P, bool HAS_Y, int R, int MAXT>
__global__ void __launch_bounds__(MAXT) gated_norm_bwd_kernel(const __grid_constant__ GatedNormParams p) {
  constexpr int NIN = HAS_Y ? 4 : 3;  // x, dh, dx', y
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float sums[2 * 4 * kMaxWarps];
  static_assert(2 * R <= 4, "row_sum's buffers hold four sums");
  const int tpr = p.tpr, wpr = tpr >> 5, group = threadIdx.x / tpr, groups = blockDim.x / tpr;
  const int col = (threadIdx.x % tpr) * 8;
  const bool on = col < p.cols;
  float* gw = reinterpret_cast<float*>(smem);
  float* sw = gw + p.cols;
  const Ring<NIN, R> ring{reinterpret_cast<uint8_t*>(sw + p.cols), p.stages};
  const float inv_c = 1.f / (float)p.cols;
  const bool post = HAS_Y && p.post_weight != nullptr, layer = p.layer != 0;
  int flip = 0;

  const Share s = share_of_block(p);
  int seq = s.seq;
  for (int64_t a = s.r0; a < s.r1;) {
    while (seq + 1 < p.seqs && seq_begin(p, seq + 1) <= a) ++seq;
    const int64_t b = min(s.r1, seq + 1 < p.seqs ? seq_begin(p, seq + 1) : p.rows);
    const int n = (int)((b - a + (int64_t)groups * R - 1) / (groups * R));
    auto row_of = [&](int it, int r) { return a + ((int64_t)it * groups + group) * R + r; };
    auto issue = [&](int it) {
      if (it < n && on)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int64_t row = row_of(it, r);
          if (row >= b) continue;
          const int st = it % p.stages;
          cp_async16(smem_u32(ring.at(st, r, 0)), static_cast<const T*>(p.x) + row * p.x_row + col, 16);
          if (p.dh) cp_async16(smem_u32(ring.at(st, r, 1)), static_cast<const T*>(p.dh) + row * p.dh_row + col, 16);
          if (p.dx_new) cp_async16(smem_u32(ring.at(st, r, 2)), static_cast<const T*>(p.dx_new) + row * p.dx_new_row + col, 16);
          if (HAS_Y) cp_async16(smem_u32(ring.at(st, r, NIN - 1)), static_cast<const T*>(p.y) + row * p.y_row + col, 16);
        }
      cp_async_commit();
    };
    for (int i = 0; i < p.stages - 1; ++i) issue(i);
    __syncthreads();  // the last run's parameters and sums are no longer read
    if (group == 0) load_params<T, P>(p, seq, col, on, gw, sw, nullptr);
    __syncthreads();
    float sa[8], sb[8], sc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sa[i] = sb[i] = sc[i] = 0.f;
    for (int it = 0; it < n; ++it) {
      wait_stages(p.stages - 2);
      float xn[R][8], yn[HAS_Y ? R : 1][8], dh[R][8], acc[2 * R], ry[R], rx[R];
      uint4 dxr[R];
      float g[8], w[8];
      if (on) {
        get8(gw + col, g);
        get8(sw + col, w);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t row = row_of(it, r);
        const bool live = on && row < b;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const int st = it % p.stages;
        float mean = 0.f;
        ry[r] = rx[r] = 0.f;
        if (row < b) {
          ry[r] = p.stats[row];
          mean = p.stats[p.rows + row];
          rx[r] = p.stats[2 * p.rows + row];
        }
        unpack8<T>(live ? *ring.at(st, r, 0) : zero, xn[r]);
        unpack8<T>(live && p.dh ? *ring.at(st, r, 1) : zero, dh[r]);
        dxr[r] = live && p.dx_new ? *ring.at(st, r, 2) : zero;
        if constexpr (HAS_Y) {
          unpack8<T>(live ? *ring.at(st, r, NIN - 1) : zero, yn[r]);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            yn[r][i] *= ry[r];
            if (live) xn[r][i] = fmaf(g[i], yn[r][i], xn[r][i]);
          }
        }
        acc[2 * r] = acc[2 * r + 1] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          xn[r][i] = live ? (xn[r][i] - mean) * rx[r] : 0.f;
          sb[i] = fmaf(dh[r][i], xn[r][i], sb[i]);
          sc[i] += dh[r][i];
          dh[r][i] = live ? dh[r][i] * w[i] : 0.f;  // g of the formulas
          acc[2 * r] = fmaf(dh[r][i], xn[r][i], acc[2 * r]);
          acc[2 * r + 1] += dh[r][i];
        }
      }
      issue(it + p.stages - 1);
      row_sum<2 * R>(acc, sums, flip, group, wpr);
      float acc2[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float gn = acc[2 * r] * inv_c, gm = layer ? acc[2 * r + 1] * inv_c : 0.f;
        float d[8];
        unpack8<T>(dxr[r], d);
        acc2[r] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          d[i] = fmaf(rx[r], dh[r][i] - gm - xn[r][i] * gn, d[i]);
          dh[r][i] = on ? d[i] : 0.f;  // dx
          if constexpr (HAS_Y) {
            sa[i] = row_of(it, r) < b && on ? fmaf(d[i], yn[r][i], sa[i]) : sa[i];
            xn[r][i] = on ? d[i] * g[i] : 0.f;  // t
            acc2[r] = fmaf(xn[r][i], yn[r][i], acc2[r]);
          }
        }
      }
      if (post) row_sum<R>(acc2, sums, flip, group, wpr);
      if (on) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int64_t row = row_of(it, r);
          if (row >= b) continue;
          *reinterpret_cast<uint4*>(static_cast<T*>(p.dx) + row * p.cols + col) = pack8<T>(dh[r]);
          if constexpr (HAS_Y) {
            if (post) {
              const float m = acc2[r] * inv_c;
#pragma unroll
              for (int i = 0; i < 8; ++i) xn[r][i] = ry[r] * (xn[r][i] - yn[r][i] * m);
            }
            *reinterpret_cast<uint4*>(static_cast<T*>(p.dy) + row * p.cols + col) = pack8<T>(xn[r]);
          }
        }
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
            float f[8];
#pragma unroll
            for (int q = 0; q < 3; ++q) {
              float* mine = q == 0 ? sa : q == 1 ? sb : sc;
              if (g2 > 0) {
                get8(acc3 + q * p.cols + col, f);
#pragma unroll
                for (int i = 0; i < 8; ++i) mine[i] += f[i];
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
// Threads that hold a row: 8 columns each, whole warps.
int row_threads(int cols) { return (cols / 8 + 31) / 32 * 32; }

struct Shape {
  int threads, tpr, stages, blocks, smem;
};
// Threads: whole rows of TPR = cols / 8 rounded up to warps, 256 threads or one row. Stages: up to four,
// what fits beside the combined parameters; blocks: an equal share for every block that is resident.
Shape shape_of(int cols, int64_t rows, int nparam, int nin, int r, int regs_cap_threads) {
  Shape s;
  s.tpr = row_threads(cols);
  const int groups = s.tpr <= 128 ? 256 / s.tpr : 1;
  s.threads = s.tpr * groups;
  const int stage = s.threads * 16 * nin * r, par = nparam * cols * 4;
  // blocks per SM that registers allow (regs_cap_threads threads resident), each with its part of shared memory
  int per_sm = std::max(1, regs_cap_threads / s.threads);
  while (per_sm > 1 && par + 2 * stage > kSmemLimit / per_sm) --per_sm;
  s.stages = std::max(2, std::min(4, (kSmemLimit / per_sm - par) / stage));
  // the groups' column sums pass through three rows of the shared memory
  s.smem = std::max(par + s.stages * stage, groups > 1 ? 3 * cols * 4 : 0);
  s.blocks = (int)std::min<int64_t>((rows + groups * r - 1) / (groups * r), (int64_t)148 * per_sm);
  return s;
}

Shape backward_shape(const GatedNormParams& p) {
  return shape_of(p.cols, p.rows, 2, p.y ? 4 : 3, 1, row_threads(p.cols) > 640 ? 1024 : 640);
}

template <typename Kern>
cudaError_t run(Kern kern, std::atomic<uint64_t>& ready, const Shape& s, const GatedNormParams& p, cudaStream_t st) {
  cudaError_t e = allow_smem(kern, kSmemLimit, ready);
  if (e != cudaSuccess) return e;
  kern<<<s.blocks, s.threads, s.smem, st>>>(p);
  return cudaGetLastError();
}

template <typename T, typename P, bool HAS_Y, int MAXT>
cudaError_t forward(GatedNormParams p, cudaStream_t st) {
  constexpr int R = MAXT > 640 ? 1 : 2;
  const Shape s = shape_of(p.cols, p.rows, 3, HAS_Y ? 2 : 1, R, MAXT > 640 ? 1024 : 768);
  p.tpr = s.tpr;
  p.stages = s.stages;
  static std::atomic<uint64_t> ready{0};
  return run(gated_norm_fwd_kernel<T, P, HAS_Y, R, MAXT>, ready, s, p, st);
}

template <typename T, typename P, bool HAS_Y, int MAXT>
cudaError_t backward(GatedNormParams p, cudaStream_t st) {
  const Shape s = backward_shape(p);
  p.tpr = s.tpr;
  p.stages = s.stages;
  if (p.rows > 0) {
    static std::atomic<uint64_t> ready{0};
    cudaError_t e = run(gated_norm_bwd_kernel<T, P, HAS_Y, 1, MAXT>, ready, s, p, st);
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
  const int threads = row_threads(p.cols);
  auto go = [&](auto has_y) {
    constexpr bool Y = decltype(has_y)::value;
    if (threads <= 256) return bwd ? backward<T, P, Y, 256>(p, st) : forward<T, P, Y, 256>(p, st);
    if (threads <= 640) return bwd ? backward<T, P, Y, 640>(p, st) : forward<T, P, Y, 640>(p, st);
    return bwd ? backward<T, P, Y, 1024>(p, st) : forward<T, P, Y, 1024>(p, st);
  };
  return p.y ? go(std::true_type{}) : go(std::false_type{});
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
