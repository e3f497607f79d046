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
bool pages_ok(const vmb_pages& r, int step = 8) {
  return r.ptr && aligned16(r.ptr) && r.page >= 0 && r.head >= 0 && r.slot >= 0 && r.page % step == 0 && r.head % step == 0 &&
         r.slot % step == 0;
}
bool scales_ok(const vmb_page_scales& s) { return s.ptr && s.page >= 0 && s.head >= 0; }

int check_pool(const char* what, int64_t num_pages, int kv_heads, int dim, int page_size, bool e4m3 = false) {
  if (e4m3 && dim % 16)
    return set_error(VMB_ENOTSUP, "%s: head dim %d is not a multiple of 16, as e4m3 pools need", what, dim);
  if (dim < 8 || dim > 128 || dim % 8)
    return set_error(VMB_ENOTSUP, "%s: head dim %d is not a multiple of 8 up to 128", what, dim);
  if (kv_heads < 1 || page_size < 1 || num_pages < 1 || num_pages > 0x7fffffff ||
      (int64_t)page_size * kv_heads * dim > 0x7fffffff)
    return set_error(VMB_EINVAL, "%s: bad pool sizes", what);
  return VMB_OK;
}

int fill(const vmb_paged_args* a, const vmb_cache_args* c, vmb::PagedParams& p, const char* what) {
  if (!a) return set_error(VMB_EINVAL, "%s: null args", what);
  const bool e4m3 = c && c->k_scale.ptr;
  if (a->dtype != VMB_DTYPE_BF16 && a->dtype != VMB_DTYPE_F16)
    return set_error(VMB_EINVAL, "%s: unknown dtype %d", what, a->dtype);
  int rc = check_pool(what, a->num_pages, a->kv_heads, a->dim, a->page_size, e4m3);
  if (rc) return rc;
  if (c) {
    if (c->window < 0 || c->sinks < 0 || (c->sinks > 0 && c->window == 0))
      return set_error(VMB_EINVAL, "%s: windows and sinks are not negative, and sinks need a window", what);
    if ((c->k_scale.ptr || c->v_scale.ptr) && (!scales_ok(c->k_scale) || !scales_ok(c->v_scale)))
      return set_error(VMB_EINVAL, "%s: e4m3 pools need scales of keys and of values", what);
    p.window = c->window;
    p.sinks = c->sinks;
    p.k_scale = c->k_scale.ptr; p.ks_page = c->k_scale.page; p.ks_head = c->k_scale.head;
    p.v_scale = c->v_scale.ptr; p.vs_page = c->v_scale.page; p.vs_head = c->v_scale.head;
  }
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
  p.max_len = (int)std::min<int64_t>(a->table_width * a->page_size, 0x7fffffff - (e4m3 ? vmb::kPagedTile8 : 64));
  p.scale_log2 = a->sm_scale * vmb::kLog2e;
  vmb::paged_plan(p);
  return VMB_OK;
}

int move_params(const char* what, const vmb_pages* k, const vmb_pages* v, const int32_t* dst, int64_t count,
                int64_t num_pages, int kv_heads, int dim, int page_size, vmb::PageMoveParams& p, bool e4m3 = false) {
  int rc = check_pool(what, num_pages, kv_heads, dim, page_size, e4m3);
  if (rc) return rc;
  if (count < 0) return set_error(VMB_EINVAL, "%s: negative count", what);
  if (!k || !v || !dst || !pages_ok(*k, e4m3 ? 16 : 8) || !pages_ok(*v, e4m3 ? 16 : 8))
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

int scale_params(const char* what, const vmb_page_scales& k, const vmb_page_scales& v, vmb::PageMoveParams& p) {
  if (!scales_ok(k) || !scales_ok(v)) return set_error(VMB_EINVAL, "%s: e4m3 pools need scales", what);
  p.k_scale = k.ptr; p.ks_page = k.page; p.ks_head = k.head;
  p.v_scale = v.ptr; p.vs_page = v.page; p.vs_head = v.head;
  return VMB_OK;
}

int64_t attention_workspace(const vmb_paged_args* a, const vmb_cache_args* c, const char* what) {
  vmb::PagedParams p{};
  if (fill(a, c, p, what) != VMB_OK) return -1;
  return p.batch == 0 ? 0 : vmb::paged_workspace(p);
}

int attention(const vmb_paged_args* a, const vmb_cache_args* c, const char* what, void* stream) {
  vmb::PagedParams p{};
  int rc = fill(a, c, p, what);
  if (rc) return rc;
  if (p.batch == 0) return VMB_OK;
  const int step = p.k_scale ? 16 : 8;
  if (!rows_ok(a->q) || !rows_ok(a->o) || !pages_ok(a->k, step) || !pages_ok(a->v, step) || !a->lengths ||
      (a->table_width > 0 && !a->table))
    return set_error(VMB_EINVAL, "%s: tensors need 16-byte aligned rows", what);
  const int64_t need = vmb::paged_workspace(p);
  if (need > 0 && (!a->workspace || a->workspace_bytes < need || (reinterpret_cast<uintptr_t>(a->workspace) & 255)))
    return set_error(VMB_EINVAL, "%s: a 256-byte aligned workspace of %lld bytes needed", what, (long long)need);
  vmb::count_launches(p.whole_items ? 1 : 2);
  return cuda_rc(vmb::paged_decode(p, a->workspace, a->dtype == VMB_DTYPE_BF16, static_cast<cudaStream_t>(stream)), what);
}

}  // namespace

extern "C" {

int64_t vmb_paged_workspace_bytes(const vmb_paged_args* a) { return attention_workspace(a, nullptr, "vmb_paged_attention"); }

int vmb_paged_attention(const vmb_paged_args* a, void* stream) { return attention(a, nullptr, "vmb_paged_attention", stream); }

int64_t vmb_cache_workspace_bytes(const vmb_paged_args* a, const vmb_cache_args* c) {
  return attention_workspace(a, c, "vmb_cache_attention");
}

int vmb_cache_attention(const vmb_paged_args* a, const vmb_cache_args* c, void* stream) {
  return attention(a, c, "vmb_cache_attention", stream);
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

int vmb_append_pages_e4m3(const vmb_move_e4m3_args* a, void* stream) {
  const char* what = "vmb_append_pages_e4m3";
  vmb::PageMoveParams p{};
  if (!a) return set_error(VMB_EINVAL, "%s: null args", what);
  if (a->count == 0) return VMB_OK;
  if (a->dtype != VMB_DTYPE_BF16 && a->dtype != VMB_DTYPE_F16) return set_error(VMB_EINVAL, "%s: unknown dtype %d", what, a->dtype);
  int rc = move_params(what, &a->k, &a->v, a->dst, a->count, a->num_pages, a->kv_heads, a->dim, a->page_size, p, true);
  if (rc || (rc = scale_params(what, a->k_scale, a->v_scale, p))) return rc;
  if (!rows_ok(a->k_new) || !rows_ok(a->v_new)) return set_error(VMB_EINVAL, "%s: new rows need 16-byte alignment", what);
  p.k_src = a->k_new.ptr; p.v_src = a->v_new.ptr;
  p.k_row = a->k_new.row; p.k_shead = a->k_new.head; p.v_row = a->v_new.row; p.v_shead = a->v_new.head;
  vmb::count_launches(1);
  return cuda_rc(vmb::append_pages_e4m3(p, a->dtype == VMB_DTYPE_BF16, static_cast<cudaStream_t>(stream)), what);
}

int vmb_copy_pages_e4m3(const vmb_move_e4m3_args* a, void* stream) {
  const char* what = "vmb_copy_pages_e4m3";
  vmb::PageMoveParams p{};
  if (!a) return set_error(VMB_EINVAL, "%s: null args", what);
  if (a->count == 0) return VMB_OK;
  int rc = move_params(what, &a->k, &a->v, a->dst, a->count, a->num_pages, a->kv_heads, a->dim, a->page_size, p, true);
  if (rc || (rc = scale_params(what, a->k_scale, a->v_scale, p))) return rc;
  if (!a->src) return set_error(VMB_EINVAL, "%s: null source list", what);
  p.src = a->src;
  vmb::count_launches(1);
  return cuda_rc(vmb::copy_pages_e4m3(p, static_cast<cudaStream_t>(stream)), what);
}

}  // extern "C"
