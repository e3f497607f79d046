// extern "C" entry points of the page tables (include/vmonarch_b200.h): argument validation and dispatch.
#include "../../include/vmonarch_b200.h"
#include "launch.h"
#include "page_tables.h"

namespace {

using vmb::set_error;

int fill(const char* what, const vmb_page_book* a, const int32_t* want, vmb::BookParams& p) {
  if (!a) return set_error(VMB_EINVAL, "%s: null book", what);
  if (a->batch < 0 || a->batch > 0x3fffffff || a->table_width < 0 || a->table_width > 0x7fffffff || a->table_stride < a->table_width)
    return set_error(VMB_EINVAL, "%s: bad batch or table sizes", what);
  if (a->page_size < 1 || a->num_pages < 1 || a->num_pages > 0x7fffffff / a->page_size)
    return set_error(VMB_EINVAL, "%s: bad page sizes, or more than 2^31 - 1 slots", what);
  if (!a->free_pages || !a->num_free || (a->batch > 0 && (!a->lengths || !want)) || (a->batch > 0 && a->table_width > 0 && !a->table))
    return set_error(VMB_EINVAL, "%s: a tensor is missing", what);
  p.table = a->table; p.lengths = a->lengths; p.free_pages = a->free_pages; p.num_free = a->num_free; p.failed = a->failed;
  p.want = want;
  p.stride = a->table_stride;
  p.batch = (int)a->batch; p.width = (int)a->table_width; p.num_pages = (int)a->num_pages; p.page_size = a->page_size;
  return VMB_OK;
}

int workspace(const char* what, vmb::BookParams& p, bool needed, void* ws, int64_t bytes) {
  const int64_t need = !needed ? 0 : 4 * vmb::book_plan_ints(p.batch);
  if (need > 0 && (!ws || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 3)))
    return set_error(VMB_EINVAL, "%s: a workspace of %lld bytes needed", what, (long long)need);
  p.plan = static_cast<int32_t*>(ws);
  return VMB_OK;
}

int cuda_rc(cudaError_t e, const char* what) {
  return e == cudaSuccess ? VMB_OK : set_error(VMB_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}

}  // namespace

extern "C" {

int64_t vmb_page_book_workspace_bytes(const vmb_page_book* a) {
  return !a || a->batch < 0 || a->batch > 0x3fffffff ? -1 : 4 * vmb::book_plan_ints(a->batch);
}

int vmb_reserve_pages(const vmb_page_book* a, const int32_t* counts, int32_t* slots, int64_t total, void* ws, int64_t ws_bytes,
                      void* stream) {
  const char* what = "vmb_reserve_pages";
  vmb::BookParams p{};
  int rc = fill(what, a, counts, p);
  if (rc) return rc;
  if (total < 0 || total > 0x7fffffff || (total > 0 && !slots)) return set_error(VMB_EINVAL, "%s: bad number of rows, or no slots", what);
  p.slots = slots;
  p.total = total;
  if ((rc = workspace(what, p, vmb::reserve_needs_workspace(p), ws, ws_bytes))) return rc;
  vmb::count_launches(vmb::reserve_in_one(p) || total == 0 ? 1 : 2);
  return cuda_rc(vmb::reserve_pages(p, static_cast<cudaStream_t>(stream)), what);
}

int vmb_truncate_pages(const vmb_page_book* a, const int32_t* keep, void* ws, int64_t ws_bytes, void* stream) {
  const char* what = "vmb_truncate_pages";
  vmb::BookParams p{};
  int rc = fill(what, a, keep, p);
  if (rc || p.batch == 0) return rc;
  if ((rc = workspace(what, p, vmb::truncate_needs_workspace(p), ws, ws_bytes))) return rc;
  vmb::count_launches(vmb::truncate_in_one(p) || p.width == 0 ? 1 : 2);
  return cuda_rc(vmb::truncate_pages(p, static_cast<cudaStream_t>(stream)), what);
}

}  // extern "C"
