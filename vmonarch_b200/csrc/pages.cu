// Moves of a paged key / value cache: new rows into their slots, whole pages to other pages. Both are
// copies bound by memory: every byte is read once and written once, 16 bytes a thread and tensor,
// neighbouring threads on neighbouring bytes of a row (a page of one head is contiguous in the usual
// layout, so the rows of a copy follow one another). 32760 tokens of 8 heads, D = 128, appended to pages of 16:
// 47.5 us, 2047 such pages copied: 47 us, 5.7 TB/s (the measured copy rate is 6.5).
//
// Rows that go into e4m3 pools (append_e4m3_kernel) share a scale with what their page holds: the least power of two s
// with |x| <= 448 s, for a page, head and tensor (a power of two costs a floating format no precision, and a page
// that grows to a larger one keeps its values but for those that become subnormal). Rows of one page follow one another, so a
// run of them belongs to one team of warps: largest value, scale, the page brought to it where it grows, rows divided and
// stored, in one pass and without atomics.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "launch.h"
#include "paged.h"

namespace vmb {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint4 load16(const void* base, int64_t elem) {
  return __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + elem));
}
__device__ __forceinline__ void store16(void* base, int64_t elem, uint4 v) {
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + elem) = v;
}

// COPY: rows are (pair, head, slot); else (row, head). SCALED: the pages' scales go with them.
template <bool COPY, bool SCALED>
__global__ void __launch_bounds__(kThreads) page_move_kernel(const __grid_constant__ PageMoveParams p) {
  const uint32_t ch = p.dim / 8, inner = (uint32_t)(COPY ? p.page_size : 1) * ch, per = (uint32_t)p.kv_heads * inner;
  const int64_t idx = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t i = idx / per;
  if (i >= p.count) return;
  const uint32_t rem = (uint32_t)(idx - i * per), h = rem / inner, in = rem - h * inner, slot = in / ch, c = (in - slot * ch) * 8;
  if (COPY) {
    const int s = p.src[i], d = p.dst[i];
    if ((unsigned)s >= (unsigned)p.num_pages || (unsigned)d >= (unsigned)p.num_pages) return;
    const int64_t ko = h * p.k_head + slot * p.k_slot + c, vo = h * p.v_head + slot * p.v_slot + c;
    const uint4 k = load16(p.k, s * p.k_page + ko), v = load16(p.v, s * p.v_page + vo);
    store16(p.k, d * p.k_page + ko, k);
    store16(p.v, d * p.v_page + vo, v);
    if (SCALED && in == 0) {
      p.k_scale[d * p.ks_page + h * p.ks_head] = p.k_scale[s * p.ks_page + h * p.ks_head];
      p.v_scale[d * p.vs_page + h * p.vs_head] = p.v_scale[s * p.vs_page + h * p.vs_head];
    }
  } else {
    const int at = p.dst[i];
    if (at < 0 || at / p.page_size >= p.num_pages) return;
    const int64_t page = at / p.page_size, sl = at % p.page_size;
    const uint4 k = load16(p.k_src, i * p.k_row + h * p.k_shead + c), v = load16(p.v_src, i * p.v_row + h * p.v_shead + c);
    store16(p.k, page * p.k_page + h * p.k_head + sl * p.k_slot + c, k);
    store16(p.v, page * p.v_page + h * p.v_head + sl * p.v_slot + c, v);
  }
}

template <bool COPY, bool SCALED = false>
cudaError_t launch(const PageMoveParams& p, cudaStream_t st) {
  const int64_t n = p.count * p.kv_heads * (COPY ? p.page_size : 1) * (p.dim / 8);
  const int64_t blocks = (n + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  page_move_kernel<COPY, SCALED><<<(unsigned)blocks, kThreads, 0, st>>>(p);
  return cudaGetLastError();
}

// ------------------------------------------------------------------------------------ rows into e4m3 pools
constexpr int kTeamWarps = 4;  // warps of a block
constexpr int kTeamBlocks = 6; // blocks of an SM
constexpr int kHeld = 4;       // pieces of 16 columns that a lane holds at a time

// The least power of two s >= 2^-126 with top <= 448 s (448 = 1.75 x 2^8), for a finite top >= 0.
__device__ __forceinline__ float pow2_scale(float top) {
  const uint32_t b = __float_as_uint(top);
  const int e = (int)(b >> 23) - ((b & 0x7fffffu) <= 0x600000u ? 8 : 7);  // biased
  return __uint_as_float((uint32_t)max(e, 1) << 23);
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Sixteen values as e4m3, divided by a scale. POW2: times its inverse, exact in bf16 (fp16's exponents do not reach).
template <typename T, bool POW2>
__device__ __forceinline__ uint4 quantized(const uint4 (&x)[2], float scale, float inv) {
  const uint32_t w[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
  uint32_t q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float2 f;
    if (POW2 && Elem<T>::is_bf16) {
      const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), __floats2bfloat162_rn(inv, inv));
      f = Elem<T>::unpack(*reinterpret_cast<const uint32_t*>(&y));
    } else {
      f = Elem<T>::unpack(w[i]);
      f = POW2 ? make_float2(f.x * inv, f.y * inv) : make_float2(f.x / scale, f.y / scale);
    }
    q[i] = pack_e4m3x2(f.x, f.y);
  }
  return make_uint4(q[0] | q[1] << 16, q[2] | q[3] << 16, q[4] | q[5] << 16, q[6] | q[7] << 16);
}

// A team of TW warps (a warp, or the block) takes the runs that begin in its `group` rows, for one head and tensor.
template <typename T, int TW>
__global__ void __launch_bounds__(32 * kTeamWarps, kTeamBlocks) append_e4m3_kernel(const __grid_constant__ PageMoveParams p) {
  __shared__ uint32_t tops[2][kTeamWarps];
  constexpr uint32_t kInf = Elem<T>::is_bf16 ? 0x7f80u : 0x7c00u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // (a place's numbers have 32 bits, which the launch has seen to)
  const uint32_t pairs = 2 * p.kv_heads, stride = TW == 1 ? gridDim.x * kTeamWarps : gridDim.x;
  uint32_t team = TW == 1 ? blockIdx.x * kTeamWarps + warp : blockIdx.x;
  auto page_of = [&](int s, int& slot) {  // -1: skipped
    const int page = s < 0 ? -1 : s / p.page_size;
    slot = s < 0 ? -1 : s - page * p.page_size;
    return page < p.num_pages ? page : -1;
  };
  auto slot_at = [&](int64_t row) { return row >= 0 && row < p.count ? p.dst[row] : -1; };
  // A team's head and tensor, and its first row. Its slots are read, and its rows sent for to L2, while the one before works.
  int64_t row0;
  int pair, held_slot, slot_before;
  auto send_for = [&]() {
    const uint32_t rows = team / pairs;
    row0 = (int64_t)rows * p.group;
    pair = (int)(team - rows * pairs);
    if (row0 >= p.count) return;
    held_slot = slot_at(row0 + lane);
    slot_before = slot_at(row0 - 1);
    if (lane < p.group && row0 + lane < p.count) {
      const int head = pair >> 1;
      const T* row = pair & 1 ? static_cast<const T*>(p.v_src) + head * p.v_shead + (row0 + lane) * p.v_row
                              : static_cast<const T*>(p.k_src) + head * p.k_shead + (row0 + lane) * p.k_row;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(row));
      if (p.dim > 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + p.dim - 1));
    }
  };
  // lanes a row: a power of two, sixteen columns each
  const int ch = p.dim / 16, bits = ch > 4 ? 3 : ch > 2 ? 2 : ch > 1 ? 1 : 0;
  const int per = (32 >> bits) * TW;                            // rows a load of the team
  const int at = (TW == 1 ? 0 : warp * (32 >> bits)) + (lane >> bits), c = (lane & ((1 << bits) - 1)) * 16;
  const bool live = c < p.dim;
  const int step = TW == 1 ? lane : threadIdx.x;
  int turn = 0;
  send_for();
  while (row0 < p.count) {
    const int64_t base = row0;
    const int head = pair >> 1;
    const bool is_v = pair & 1;
    const T* src = static_cast<const T*>(is_v ? p.v_src : p.k_src) + head * (is_v ? p.v_shead : p.k_shead);
    const int64_t src_row = is_v ? p.v_row : p.k_row, dst_slot = is_v ? p.v_slot : p.k_slot;
    int my_slot, unused;
    const int mine = page_of(held_slot, my_slot);
    int before = page_of(slot_before, unused);
    team += stride;
    send_for();
    // (group <= 32: a lane looks at a row)
    const int above = __shfl_up_sync(0xffffffffu, mine, 1);
    if (lane > 0) before = above;
    unsigned starts = __ballot_sync(0xffffffffu, lane < p.group && mine >= 0 && mine != before);
    const unsigned same = __ballot_sync(0xffffffffu, mine >= 0 && mine == before);
    const unsigned firsts = __ballot_sync(0xffffffffu, my_slot == 0);
    uint8_t* pool = static_cast<uint8_t*>(is_v ? p.v : p.k) + head * (is_v ? p.v_head : p.k_head);
    const int64_t dst_page = is_v ? p.v_page : p.k_page;
    float* scales = is_v ? p.v_scale + head * p.vs_head : p.k_scale + head * p.ks_head;
    const int64_t scale_page = is_v ? p.vs_page : p.ks_page;
    const int64_t src_step = per * src_row;
    for (; starts; starts &= starts - 1) {
      const int s = __ffs(starts) - 1, page = __shfl_sync(0xffffffffu, mine, s);
      const int64_t first = base + s;
      int n = __ffs(~((same >> s) >> 1));  // rows of the run among the 32
      bool begins = (firsts >> s & (n >= 32 ? 0xffffffffu : (1u << n) - 1u)) != 0;  // slot 0 of the page is among the rows
      if (s + n > 31) {                    // up to the last of them: it may go on
        n = 32 - s;
        for (;;) {
          int slot;
          const int next = page_of(slot_at(first + n + lane), slot);
          const unsigned other = ~__ballot_sync(0xffffffffu, next == page);
          const int more = other ? __ffs(other) - 1 : 32;
          begins |= __any_sync(0xffffffffu, lane < more && slot == 0);
          n += more;
          if (other) break;
        }
      }
      float* scale_at = scales + page * scale_page;
      const float old = *scale_at;
      uint4 x[kHeld][2];
      const T* from = src + (first + at) * src_row + c;
      auto load = [&](int r0) {
        const T* q = from + r0 * src_row;
#pragma unroll
        for (int u = 0; u < kHeld; ++u, q += src_step) {
          x[u][0] = x[u][1] = make_uint4(0u, 0u, 0u, 0u);
          if (r0 + u * per + at < n && live) {
            x[u][0] = load16(q, 0);
            x[u][1] = load16(q, 8);
          }
        }
      };
      const bool held = n <= kHeld * per;
      // the largest magnitude as 16 bits, whose order is that of the values; without what is not finite if asked for
      auto largest = [&](bool finite) -> uint32_t {
        uint32_t top = 0;
        for (int r0 = 0; r0 < n; r0 += kHeld * per) {
          if (!held) load(r0);
#pragma unroll
          for (int u = 0; u < kHeld; ++u) {
            const uint32_t w[8] = {x[u][0].x, x[u][0].y, x[u][0].z, x[u][0].w, x[u][1].x, x[u][1].y, x[u][1].z, x[u][1].w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              uint32_t a = w[i] & 0x7fff7fffu;
              if (finite) {
                if ((a & 0xffffu) >= kInf) a &= 0xffff0000u;
                if (a >> 16 >= kInf) a &= 0xffffu;
              }
              top = max_u16x2(top, a);
            }
          }
        }
        top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
        if (TW > 1) {
          if (lane == 0) tops[turn & 1][warp] = top;
          __syncthreads();
#pragma unroll
          for (int i = 0; i < kTeamWarps; ++i) top = max(top, tops[turn & 1][i]);
          ++turn;
        }
        return top;
      };
      if (held) load(0);
      uint32_t top = largest(false);
      const bool infinite = top >= kInf;
      if (infinite) top = largest(true);
      const float need = pow2_scale(Elem<T>::unpack(top).x), scale = begins ? need : fmaxf(old, need);
      uint8_t* to = pool + page * dst_page;
      if (TW > 1) __syncthreads();  // everybody has read the scale
      else __syncwarp();
      if (!begins && !(old >= scale)) {
        const float by = old / scale;
        const int chunks = p.dim / 16;
        for (int i = step; i < p.page_size * chunks; i += 32 * TW) {
          uint4* q = reinterpret_cast<uint4*>(to + (int64_t)(i / chunks) * dst_slot + i % chunks * 16);
          uint4 v = *q;
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[k] & 0xffffu), __NV_E4M3);
            const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[k] >> 16), __NV_E4M3);
            const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
            w[k] = pack_e4m3x2(a.x * by, a.y * by) | pack_e4m3x2(b.x * by, b.y * by) << 16;
          }
          *q = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (TW > 1) __syncthreads();
        else __syncwarp();
      }
      if (step == 0) *scale_at = scale;
      // a power of two is multiplied with its inverse, which is exact; any other scale, which a caller brought, divides
      const bool pow2 = (__float_as_uint(scale) & 0x7fffffu) == 0;
      const float inv = 1.f / scale;
      auto write = [&](auto exact) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
          const int r = u * per + at;
          const int slot = __shfl_sync(0xffffffffu, my_slot, (s + r) & 31);
          if (r < n && live) *reinterpret_cast<uint4*>(to + slot * dst_slot + c) = quantized<T, decltype(exact)::value>(x[u], scale, inv);
        }
      };
      if (held && s + n <= 32 && pow2 && !infinite) {
        write(std::true_type{});
        continue;
      }
#pragma unroll 1
      for (int r0 = 0; r0 < n; r0 += kHeld * per) {
        if (!held) load(r0);
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
          const int r = r0 + u * per + at;
          if (r >= n || !live) continue;
          if (infinite) {  // to NaN: the conversion would make the largest value of an infinity
            uint32_t* w = &x[u][0].x;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if ((w[i] & 0x7fffu) == kInf) w[i] |= 1u;
              if ((w[i] >> 16 & 0x7fffu) == kInf) w[i] |= 0x10000u;
            }
          }
          const int slot = p.dst[first + r] - page * p.page_size;
          *reinterpret_cast<uint4*>(to + slot * dst_slot + c) = pow2 ? quantized<T, true>(x[u], scale, inv) : quantized<T, false>(x[u], scale, inv);
        }
      }
    }
  }
}

template <typename T>
cudaError_t launch_e4m3(PageMoveParams p, cudaStream_t st) {
  // A block a run where runs may be long: pages of 64 slots and rows for two of them. 16384 rows of prompts, 8 heads, D = 128, us, with
  // a warp and with a block: pages of 48 27.3 and 36.5, of 64 34.2 and 28.9, of 256 46.9 and 33.9; 1024 rows, pages of 256 28.5
  // and 13.1; one row of each of 64 sequences, whatever their pages, 3.3 and 4.8.
  const bool block = p.page_size >= 64 && p.count >= 2 * (int64_t)p.page_size;
  const int64_t pairs = 2 * p.kv_heads;
  // one row a team while all teams are on the GPU at once, up to a page's rows where there are many (8 heads, D = 128, us, with this room and
  // with that of 16 blocks an SM, at which teams of one row took up to three turns: 512 rows of a prompt, pages of 16, 4.1 and 5.4, pages
  // of 64 4.7 and 5.4; one row of each of 512 sequences, pages of 16, 7.3 and 8.3)
  const int64_t room = 148 * kTeamBlocks * (block ? 1 : kTeamWarps);
  p.group = (int)std::min<int64_t>(std::max<int64_t>((p.count * pairs + room - 1) / room, 1), std::min(p.page_size, 32));
  const int64_t teams = (p.count + p.group - 1) / p.group * pairs, blocks = block ? teams : (teams + kTeamWarps - 1) / kTeamWarps;
  if (teams > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const unsigned grid = (unsigned)std::min<int64_t>(blocks, 148 * kTeamBlocks);
  if (block) append_e4m3_kernel<T, kTeamWarps><<<grid, 32 * kTeamWarps, 0, st>>>(p);
  else append_e4m3_kernel<T, 1><<<grid, 32 * kTeamWarps, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t append_pages_e4m3(PageMoveParams p, bool bf16, cudaStream_t st) {
  return bf16 ? launch_e4m3<__nv_bfloat16>(p, st) : launch_e4m3<__half>(p, st);
}
// bytes move two at a time: sizes and strides are multiples of 16 of them
cudaError_t copy_pages_e4m3(PageMoveParams p, cudaStream_t st) {
  for (int64_t* s : {&p.k_page, &p.k_head, &p.k_slot, &p.v_page, &p.v_head, &p.v_slot}) *s /= 2;
  p.dim /= 2;
  return launch<true, true>(p, st);
}

cudaError_t append_pages(const PageMoveParams& p, cudaStream_t st) { return launch<false>(p, st); }
cudaError_t copy_pages(const PageMoveParams& p, cudaStream_t st) { return launch<true>(p, st); }

}  // namespace vmb
