// Parameter block of the kernels that keep the book of a paged cache (page_tables.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace vmb {

struct BookParams {
  int32_t *table, *lengths;   // [batch][stride], [batch]
  int32_t *free_pages;        // [num_pages], a stack of num_free pages
  int32_t *num_free, *failed; // failed: NULL allowed
  const int32_t* want;        // [batch]: reserve: tokens to come; truncate: tokens to keep
  int32_t* slots;             // reserve: [total]
  int64_t stride, total;
  int batch, width, num_pages, page_size;
  int32_t* plan;              // workspace of book_plan_ints(batch), or NULL where a call needs none
};

// Whether a call needs a workspace, and whether one kernel does its work.
bool reserve_needs_workspace(const BookParams& p);
bool truncate_needs_workspace(const BookParams& p);
bool reserve_in_one(const BookParams& p);
bool truncate_in_one(const BookParams& p);
int64_t book_plan_ints(int64_t batch);
cudaError_t reserve_pages(const BookParams& p, cudaStream_t st);
cudaError_t truncate_pages(const BookParams& p, cudaStream_t st);

}  // namespace vmb
