// extern "C" entry points of the paged cache (include/vmonarch_b200.h): argument validation and dispatch.
#include <algorithm>
#include <cmath>

#include "../../include/vmonarch_b200.h"
#include "common.cuh"
#include "launch.h"
#include "paged.h"

namespace {

using vmb::set_error;

int cuda_rc(cudaError_t e, const char* what) {
  return e == cudaSuccess ? VMB_OK : set_error(VMB_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool rows_ok(const vmb_rows& r) {
  return r.ptr && aligned16(r.ptr) && r.row >= 0 && r.head >= 0 && r.row % 8 == 0 && r.head % 8 == 0;
}
bool pages_ok(const vmb_pages& r) {
  return r.ptr && aligned16(r.ptr) && r.page >= 0 && r.head >= 0 && r.slot >= 0 && r.page % 8 == 0 && r.head % 8 == 0 &&
         r.slot % 8 == 0;
}

int check_pool(const char* what, int64_t num_pages, int kv_heads, int dim, int page_size) {
  if (dim < 8 || dim > 128 || dim % 8)
    return set_error(VMB_ENOTSUP, "%s: head dim %d is not a multiple of 8 up to 128", what, dim);
  if (kv_heads < 1 || page_size < 1 || num_pages < 1 || num_pages > 0x7fffffff ||
      (int64_t)page_size * kv_heads * dim > 0x7fffffff)
    return set_error(VMB_EINVAL, "%s: bad pool sizes", what);
  return VMB_OK;
}

int fill(const vmb_paged_args* a, vmb::PagedParams& p) {
  const char* what = "vmb_paged_attention";
  if (!a) return set_error(VMB_EINVAL, "%s: null args", what);
  if (a->dtype != VMB_DTYPE_BF16 && a->dtype != VMB_DTYPE_F16)
    return set_error(VMB_EINVAL, "%s: unknown dtype %d", what, a->dtype);
  int rc = check_pool(what, a->num_pages, a->kv_heads, a->dim, a->page_size);
  if (rc) return rc;
  if (a->heads < 1 || a->heads % a->kv_heads)
    return set_error(VMB_EINVAL, "%s: heads=%d is not a multiple of kv_heads=%d", what, a->heads, a->kv_heads);
  if (a->batch < 0 || a->batch > 0x7fffffff / a->heads || a->table_width < 0 || a->table_stride < a->table_width)
    return set_error(VMB_EINVAL, "%s: bad batch or table sizes", what);
  if (!(a->sm_scale >= 0.f) || !std::isfinite(a->sm_scale))
    return set_error(VMB_EINVAL, "%s: sm_scale must be finite and not negative", what);
  p.q = a->q.ptr; p.k = a->k.ptr; p.v = a->v.ptr; p.o = a->o.ptr;
  p.lse = a->lse;
  vmb::test_timeout(&p.wait_limit, &p.hold_loads);
  p.table = a->table;
  p.lengths = a->lengths;
  p.q_row = a->q.row; p.q_head = a->q.head; p.o_row = a->o.row; p.o_head = a->o.head;
  p.k_page = a->k.page; p.k_head = a->k.head; p.k_slot = a->k.slot;
  p.v_page = a->v.page; p.v_head = a->v.head; p.v_slot = a->v.slot;
  p.table_stride = a->table_stride;
  p.batch = (int)a->batch;
  p.heads = a->heads; p.kv_heads = a->kv_heads; p.dim = a->dim; p.page_size = a->page_size;
  p.num_pages = (int)a->num_pages;
  // token positions are 32-bit, a tile past the last one included
  p.max_len = (int)std::min<int64_t>(a->table_width * a->page_size, 0x7fffffff - 64);
  p.scale_log2 = a->sm_scale * vmb::kLog2e;
  vmb::paged_plan(p);
  return VMB_OK;
}

int move_params(const char* what, const vmb_pages* k, const vmb_pages* v, const int32_t* dst, int64_t count,
                int64_t num_pages, int kv_heads, int dim, int page_size, vmb::PageMoveParams& p) {
  int rc = check_pool(what, num_pages, kv_heads, dim, page_size);
  if (rc) return rc;
  if (count < 0) return set_error(VMB_EINVAL, "%s: negative count", what);
  if (!k || !v || !dst || !pages_ok(*k) || !pages_ok(*v))
    return set_error(VMB_EINVAL, "%s: pools need 16-byte aligned rows, indices a buffer", what);
  p.k = k->ptr; p.v = v->ptr;
  p.k_page = k->page; p.k_head = k->head; p.k_slot = k->slot;
  p.v_page = v->page; p.v_head = v->head; p.v_slot = v->slot;
  p.dst = dst;
  p.count = count;
  p.kv_heads = kv_heads; p.dim = dim; p.page_size = page_size;
  p.num_pages = (int)num_pages;
  return VMB_OK;
}

}  // namespace

extern "C" {

int64_t vmb_paged_workspace_bytes(const vmb_paged_args* a) {
  vmb::PagedParams p{};
  if (fill(a, p) != VMB_OK) return -1;
  return p.batch == 0 ? 0 : vmb::paged_workspace(p);
}

int vmb_paged_attention(const vmb_paged_args* a, void* stream) {
  vmb::PagedParams p{};
  int rc = fill(a, p);
  if (rc) return rc;
  if (p.batch == 0) return VMB_OK;
  if (!rows_ok(a->q) || !rows_ok(a->o) || !pages_ok(a->k) || !pages_ok(a->v) || !a->lengths || (a->table_width > 0 && !a->table))
    return set_error(VMB_EINVAL, "vmb_paged_attention: tensors need 16-byte aligned rows");
  const int64_t need = vmb::paged_workspace(p);
  if (need > 0 && (!a->workspace || a->workspace_bytes < need || (reinterpret_cast<uintptr_t>(a->workspace) & 255)))
    return set_error(VMB_EINVAL, "vmb_paged_attention: a 256-byte aligned workspace of %lld bytes needed", (long long)need);
  vmb::count_launches(p.whole_items ? 1 : 2);
  return cuda_rc(vmb::paged_decode(p, a->workspace, a->dtype == VMB_DTYPE_BF16, static_cast<cudaStream_t>(stream)),
                 "vmb_paged_attention");
}

int vmb_append_pages(const vmb_rows* k_new, const vmb_rows* v_new, const vmb_pages* k, const vmb_pages* v,
                     const int32_t* slots, int64_t count, int64_t num_pages, int32_t kv_heads, int32_t dim,
                     int32_t page_size, void* stream) {
  vmb::PageMoveParams p{};
  if (count == 0) return VMB_OK;
  int rc = move_params("vmb_append_pages", k, v, slots, count, num_pages, kv_heads, dim, page_size, p);
  if (rc) return rc;
  if (!k_new || !v_new || !rows_ok(*k_new) || !rows_ok(*v_new))
    return set_error(VMB_EINVAL, "vmb_append_pages: new rows need 16-byte alignment");
  p.k_src = k_new->ptr; p.v_src = v_new->ptr;
  p.k_row = k_new->row; p.k_shead = k_new->head; p.v_row = v_new->row; p.v_shead = v_new->head;
  vmb::count_launches(1);
  return cuda_rc(vmb::append_pages(p, static_cast<cudaStream_t>(stream)), "vmb_append_pages");
}

int vmb_copy_pages(const vmb_pages* k, const vmb_pages* v, const int32_t* src, const int32_t* dst, int64_t count,
                   int64_t num_pages, int32_t kv_heads, int32_t dim, int32_t page_size, void* stream) {
  vmb::PageMoveParams p{};
  if (count == 0) return VMB_OK;
  int rc = move_params("vmb_copy_pages", k, v, dst, count, num_pages, kv_heads, dim, page_size, p);
  if (rc) return rc;
  if (!src) return set_error(VMB_EINVAL, "vmb_copy_pages: null source list");
  p.src = src;
  vmb::count_launches(1);
  return cuda_rc(vmb::copy_pages(p, static_cast<cudaStream_t>(stream)), "vmb_copy_pages");
}

}  // extern "C"
