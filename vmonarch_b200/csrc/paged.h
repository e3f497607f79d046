// Parameter blocks of the paged-cache kernels (paged_decode.cu, pages.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace vmb {

struct PagedParams {
  const void *q, *k, *v;
  void* o;
  float* lse;              // [batch][heads] natural logarithm, or NULL
  const int32_t* table;    // [batch][table_stride] page ids
  const int32_t* lengths;  // [batch]
  int64_t q_row, q_head, o_row, o_head;                      // strides, elements
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;
  int64_t table_stride;
  int batch, heads, kv_heads, dim, page_size, num_pages, max_len;
  float scale_log2;
  int window, sinks;       // window 0: none
  // pools of e4m3 values: value x scale[page][head]; NULL: 16-bit pools
  const float *k_scale, *v_scale;
  int64_t ks_page, ks_head, vs_page, vs_head;
  // set by paged_plan
  int group, nt, chunks, items, whole_items, box_rows, join_blocks;
  int per_sm;  // blocks of the 8-bit kernel that an SM holds
  int cols;  // columns that the kernels work on: 64 or 128
  uint32_t page_magic, page_shift;  // t / page_size = t * page_magic >> page_shift, t < 2^31
  int64_t blocks;
  float *part, *part_ml;
  int2* cuts;            // [batch][items]: the first and last block of an item that is cut, -1 of one that is not
  long long wait_limit;  // pipeline wait limit in cycles (0: the default ~2 s)
  int hold_loads;        // test of the timeout path: the first warp of a block issues no load
};

// Pages of [kv_heads][page_size][dim] elements, by strides.
struct PageMoveParams {
  const void *k_src, *v_src;
  void *k, *v;
  const int32_t *src, *dst;  // append: dst = slots, src unused
  int64_t k_row, k_shead, v_row, v_shead;                    // append: strides of the new rows
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;
  int64_t count;             // append: rows; copy: pages
  int kv_heads, dim, page_size, num_pages;
  float *k_scale, *v_scale;  // pools of e4m3 values: [page][head]
  int64_t ks_page, ks_head, vs_page, vs_head;
  // set by append_pages_e4m3: rows whose runs one team of warps takes
  int group;
};

void paged_plan(PagedParams& p);
int64_t paged_workspace(const PagedParams& p);
cudaError_t paged_decode(PagedParams p, void* workspace, bool bf16, cudaStream_t st);
// over e4m3 pools (p planned, with its partials' places): tiles of that many tokens
constexpr int kPagedTile8 = 128;
cudaError_t paged_decode8(const PagedParams& p, bool bf16, cudaStream_t st);
cudaError_t append_pages(const PageMoveParams& p, cudaStream_t st);
cudaError_t copy_pages(const PageMoveParams& p, cudaStream_t st);
cudaError_t append_pages_e4m3(PageMoveParams p, bool bf16, cudaStream_t st);
cudaError_t copy_pages_e4m3(PageMoveParams p, cudaStream_t st);

}  // namespace vmb
