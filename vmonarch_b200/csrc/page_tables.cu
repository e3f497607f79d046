// The book of a paged cache on the GPU: which pages hold a sequence's tokens, and which are free.
//
// Free pages are a stack, free_pages[0 .. num_free). Sequence b of length n holds ceil(n / page_size) pages, in order, in its
// row of the table.
//   reserve   sequence b is to hold c_b more tokens. The new pages of all sequences, in order, come off the stack one by one:
//             the j-th is free_pages[num_free - 1 - j]. Row i of the packed new tokens (all of sequence 0's, then 1's ...) gets
//             the slot page * page_size + position % page_size of its token; rows past the last token -1.
//   truncate  sequence b keeps its first k_b tokens. Pages beyond them go back in the opposite order, so that a truncate
//             undoes a reserve.
// A call that cannot be done (too few free pages, a table row too narrow, more tokens than rows) changes nothing, says so in
// `failed` and gives the slots -1, which the appending kernels skip.
//
// The work is a prefix sum over the sequences, a few bytes a token, and bound by latency: the sums are one block's (each
// thread takes neighbouring sequences), which goes on to the rows or pages by itself where they are few; where they are more, the
// eight blocks of a cluster all form the sums and share the rest; otherwise the block leaves its sums to a second kernel that
// is launched early. Whole numbers, no atomics on them: the same book from run to run.
#include "common.cuh"
#include "launch.h"
#include "page_tables.h"

namespace vmb {
namespace {

constexpr int kThreads = 1024;
// Most sequences of a call in one block or one cluster, and rows (or table entries / 16, of which a call returns few). us in one
// block, in a cluster and with a second kernel, reserve: 64 sequences of one new token each 2.1, 4.5 and 5.7, 256 of four 4.5, 4.7 and
// 5.9, 1024 of four 9.5, 6.7 and 8.2, 8 of 1024 9.5, 5.0 and 4.6, 64 of 1024 64, 6.8 and 5.2, where the second launch costs the host
// 2.5, 128 of 1024 134, 10.3 and 5.7; truncate, all of their pages: 2.6, 3.7 and 4.9, 3.0, 3.9 and 5.6, 4.6, 5.4 and 7.0, 4.0, 3.9
// and 4.0, 19, 4.1 and 4.8, 39, 4.3 and 5.3.
constexpr int kOneBatch = 1024;
constexpr int kBlockRows = 2048;
constexpr int kClusterRows = 65536;
constexpr int kClusterBlocks = 8;
// Rows, and table entries, up to which no workspace is asked for, though a cluster's calls do not read it.
constexpr int kOneRows = 4096, kOneEntries = 65536;
// Table entries up to which one block does a truncate: the whole table may go back, 64 entries a thread.
constexpr int kBlockEntries = 65536;

enum { kNoPages = 1, kTooWide = 2, kTooMany = 4, kOverfull = 8 };

// Pages of `a` tokens; a and b below 2^31, so that their sum stays in 32 bits (a 64-bit division costs more than all else here).
__device__ __forceinline__ int ceil_div(int a, int b) { return (int)(((uint32_t)a + (uint32_t)b - 1u) / (uint32_t)b); }

// What the sums of a call say of each sequence: its length before, the rows and pages before it; and of the call.
struct Plan {
  int *len, *rows, *pages, *call;  // [batch], [batch + 1], [batch + 1]; call: done (1) or not, free pages before
};
__device__ __forceinline__ Plan plan_at(int32_t* at, int batch) {
  return Plan{at, at + batch, at + 2 * batch + 1, at + 3 * batch + 2};
}

// Exclusive sums of two values over the block's threads, and their totals.
struct Sums {
  int64_t a, b, total_a, total_b;
};
__device__ __forceinline__ Sums block_sums(int64_t a, int64_t b) {
  __shared__ int64_t warp_a[33], warp_b[33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  int64_t ia = a, ib = b;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, ia, s), y = __shfl_up_sync(0xffffffffu, ib, s);
    if (lane >= s) ia += x, ib += y;
  }
  if (lane == 31) warp_a[warp] = ia, warp_b[warp] = ib;
  __syncthreads();
  if (warp == 0) {
    int64_t x = lane < warps ? warp_a[lane] : 0, y = lane < warps ? warp_b[lane] : 0;
    const int64_t x0 = x, y0 = y;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, x, s), v = __shfl_up_sync(0xffffffffu, y, s);
      if (lane >= s) x += u, y += v;
    }
    warp_a[lane] = x - x0, warp_b[lane] = y - y0;
    if (lane == 31) warp_a[32] = x, warp_b[32] = y;
  }
  __syncthreads();
  return Sums{warp_a[warp] + ia - a, warp_b[warp] + ib - b, warp_a[32], warp_b[32]};
}

// The last sequence whose first number is at most x: before[seq] <= x < before[seq + 1].
__device__ __forceinline__ int sequence_of(const int* before, int batch, int64_t x) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (before[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// R neighbouring rows from `row` on, then those `step` further on: one search and, inside a page, one look for R of them.
template <int R>
__device__ __forceinline__ void write_slots(const BookParams& p, const Plan& plan, int64_t row, int64_t step) {
  const bool done = plan.call[0] != 0;
  const int top = plan.call[1] - 1, last = plan.rows[p.batch];
  for (; row < p.total; row += step) {
    int slots[R];
    int seq = -1, next = 0, page = 0, in = 0, i = 0;  // of the row before; `next`: where its sequence ends
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t r = row + k;
      slots[k] = -1;
      if (!done || r >= last) continue;
      bool look = true;
      if (seq >= 0 && r < next) {
        look = ++in == p.page_size;
        if (look) in = 0, ++i;
      } else {
        if (seq < 0) seq = sequence_of(plan.rows, p.batch, r);
        else
          while (plan.rows[seq + 1] <= r) ++seq;
        next = plan.rows[seq + 1];
        const int at = plan.len[seq] + (int)(r - plan.rows[seq]);
        i = at / p.page_size;
        in = at - i * p.page_size;
      }
      if (look) {
        const int have = ceil_div(plan.len[seq], p.page_size);
        int32_t* entry = p.table + seq * p.stride + i;
        page = i < have ? *entry : p.free_pages[top - (plan.pages[seq] + i - have)];
        if (in == 0) *entry = page;  // (a page's first token is new if the page is)
      }
      if ((unsigned)page < (unsigned)p.num_pages) slots[k] = page * p.page_size + in;
    }
    if (R == 4 && row + R <= p.total && (reinterpret_cast<uintptr_t>(p.slots) & 15) == 0) {
      *reinterpret_cast<int4*>(p.slots + row) = make_int4(slots[0], slots[1 % R], slots[2 % R], slots[3 % R]);
    } else {
#pragma unroll
      for (int k = 0; k < R; ++k)
        if (row + k < p.total) p.slots[row + k] = slots[k];
    }
  }
}
// The pages beyond the sequences' new lengths, from the x-th on in steps of `step`.
__device__ __forceinline__ void return_pages(const BookParams& p, const Plan& plan, int64_t x, int64_t step) {
  const int number = plan.pages[p.batch], top = plan.call[1] + number - 1;
  for (; x < number; x += step) {
    const int b = sequence_of(plan.pages, p.batch, x);
    // (the last of them is the last that the sequence held)
    const int held = ceil_div(plan.len[b], p.page_size);
    p.free_pages[top - x] = p.table[b * p.stride + held - (plan.pages[b + 1] - (int)x)];
  }
}

// Where the rest of a call is done: by a kernel of its own, by the block that has the sums, or by the blocks of a cluster, which
// all form the sums.
enum Rest { kNext, kBlock, kCluster };

// RESERVE: counts -> sums, else lengths to keep -> sums.
template <bool RESERVE, Rest REST>
__device__ __forceinline__ void keep_book(const BookParams& p) {
  __shared__ int32_t plan_sh[REST != kNext ? 3 * kOneBatch + 4 : 1];
  const Plan plan = plan_at(REST != kNext ? plan_sh : p.plan, p.batch);
  if (REST == kNext) let_next_kernel_start();
  const int per = (p.batch + blockDim.x - 1) / blockDim.x;
  const int b0 = min((int)threadIdx.x * per, p.batch), b1 = min(b0 + per, p.batch);
  const int64_t room = min((int64_t)p.width * p.page_size, (int64_t)0x7fffffff - 64);  // (what the attention takes)
  int64_t rows = 0, pages = 0;
  int bad = 0;
  // tokens before and behind a call
  auto lengths = [&](int b, int64_t& len, int64_t& next) {
    len = p.lengths[b];
    const int64_t want = p.want[b];
    next = RESERVE ? len + want : max((int64_t)0, min(len, want));
    if (len < 0 || (RESERVE && want < 0)) bad |= kTooMany, next = len = max(len, (int64_t)0);
    if (max(len, next) > room) bad |= kTooWide, next = len = min(len, room);
  };
  auto difference = [&](int len, int next) {
    const int pages = ceil_div(next, p.page_size) - ceil_div(len, p.page_size);
    return RESERVE ? pages : -pages;
  };
  for (int b = b0; b < b1; ++b) {
    int64_t len, next;
    lengths(b, len, next);
    rows += RESERVE ? next - len : 0;
    pages += difference((int)len, (int)next);
  }
  const int free_before = max(0, min(*p.num_free, p.num_pages));
  const Sums s = block_sums(rows, pages);
  if (RESERVE && s.total_b > free_before) bad |= kNoPages;
  if (RESERVE && s.total_a > p.total) bad |= kTooMany;
  if (!RESERVE && free_before + s.total_b > p.num_pages) bad |= kOverfull;
  // (every thread has read the number of free pages)
  bad = (__syncthreads_or(bad & kNoPages) ? kNoPages : 0) | (__syncthreads_or(bad & kTooWide) ? kTooWide : 0) |
        (__syncthreads_or(bad & kTooMany) ? kTooMany : 0) | (__syncthreads_or(bad & kOverfull) ? kOverfull : 0);
  if (threadIdx.x == 0) {
    plan.call[0] = bad == 0;
    plan.call[1] = free_before;
    if (bad && p.failed && blockIdx.x == 0) *p.failed |= bad;
    if (!bad && REST != kCluster) *p.num_free = free_before + (int)(RESERVE ? -s.total_b : s.total_b);
  }
  if (!bad) {
    rows = s.a;
    pages = s.b;
    for (int b = b0; b < b1; ++b) {
      int64_t len, next;
      lengths(b, len, next);
      plan.len[b] = (int)len;
      plan.rows[b] = (int)rows;
      plan.pages[b] = (int)pages;
      rows += RESERVE ? next - len : 0;
      pages += difference((int)len, (int)next);
      if (REST != kCluster) p.lengths[b] = (int)next;
    }
    if (threadIdx.x == 0) plan.rows[p.batch] = (int)s.total_a, plan.pages[p.batch] = (int)s.total_b;
  }
  if (REST == kCluster) {  // every block has read the book before one of them writes it
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (blockIdx.x == 0 && !bad) {
      if (threadIdx.x == 0) *p.num_free = free_before + (int)(RESERVE ? -s.total_b : s.total_b);
      for (int b = b0; b < b1; ++b) {
        int64_t len, next;
        lengths(b, len, next);
        p.lengths[b] = (int)next;
      }
    }
  }
  if (REST == kNext) return;
  __syncthreads();
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
  if (RESERVE) {
    constexpr int R = REST == kBlock ? 1 : 4;
    write_slots<R>(p, plan, R * at, R * step);
  } else if (!bad) {
    return_pages(p, plan, at, step);
  }
}
template <bool RESERVE, Rest REST>
__global__ void __launch_bounds__(kThreads) book_kernel(const __grid_constant__ BookParams p) { keep_book<RESERVE, REST>(p); }
template <bool RESERVE>
__global__ void __cluster_dims__(kClusterBlocks, 1, 1) __launch_bounds__(kThreads) book_cluster_kernel(const __grid_constant__ BookParams p) {
  keep_book<RESERVE, kCluster>(p);
}

__global__ void __launch_bounds__(256) slots_kernel(const __grid_constant__ BookParams p) {
  wait_for_kernel_before();
  let_next_kernel_start();
  write_slots<4>(p, plan_at(p.plan, p.batch), ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, (int64_t)gridDim.x * 1024);
}
__global__ void __launch_bounds__(256) return_kernel(const __grid_constant__ BookParams p) {
  wait_for_kernel_before();
  let_next_kernel_start();
  const Plan plan = plan_at(p.plan, p.batch);
  if (plan.call[0]) return_pages(p, plan, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

// threads of the first kernel: a sequence, and where it does them a row, each, if that many fit
int threads_for(int64_t n) { return (int)(n >= kThreads ? kThreads : n <= 128 ? 128 : (n + 31) / 32 * 32); }

}  // namespace

int64_t book_plan_ints(int64_t batch) { return 3 * batch + 4; }

bool reserve_needs_workspace(const BookParams& p) { return p.batch > kOneBatch || p.total > kOneRows; }
bool truncate_needs_workspace(const BookParams& p) { return p.batch > kOneBatch || (int64_t)p.batch * p.width > kOneEntries; }
bool reserve_in_one(const BookParams& p) { return p.batch <= kOneBatch && p.total <= kClusterRows; }
bool truncate_in_one(const BookParams& p) { return p.batch <= kOneBatch && (int64_t)p.batch * p.width <= 16 * kClusterRows; }

cudaError_t reserve_pages(const BookParams& p, cudaStream_t st) {
  if (reserve_in_one(p)) {
    if (p.total <= kBlockRows) book_kernel<true, kBlock><<<1, threads_for(p.total > p.batch ? p.total : p.batch), 0, st>>>(p);
    else book_cluster_kernel<true><<<kClusterBlocks, kThreads, 0, st>>>(p);
    return cudaGetLastError();
  }
  book_kernel<true, kNext><<<1, threads_for(p.batch), 0, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.total == 0) return e;
  const int64_t blocks = (p.total + 1023) / 1024;
  return launch_early(slots_kernel, blocks < 148 * 8 ? blocks : 148 * 8, 256, 0, st, p);
}

cudaError_t truncate_pages(const BookParams& p, cudaStream_t st) {
  if (truncate_in_one(p)) {
    if ((int64_t)p.batch * p.width <= kBlockEntries) book_kernel<false, kBlock><<<1, threads_for(p.batch), 0, st>>>(p);
    else book_cluster_kernel<false><<<kClusterBlocks, kThreads, 0, st>>>(p);
    return cudaGetLastError();
  }
  book_kernel<false, kNext><<<1, threads_for(p.batch), 0, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.width == 0) return e;  // (rows of no entries hold no pages)
  // (as many pages as the table has entries may go back, but hardly ever do)
  const int64_t blocks = ((int64_t)p.batch * p.width + 255) / 256;
  return launch_early(return_kernel, blocks < 148 * 8 ? blocks : 148 * 8, 256, 0, st, p);
}

}  // namespace vmb
