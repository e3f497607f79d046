// extern "C" entry points of the gated residual norm (include/vmonarch_b200.h): argument validation and
// dispatch.
#include <cmath>

#include "../../include/vmonarch_b200.h"
#include "gated_norm.h"
#include "launch.h"

namespace {

using vmb::set_error;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool matrix_ok(const vmb_matrix& m) { return aligned16(m.ptr) && m.row >= 0 && m.row <= 0x7fffffff && m.row % 8 == 0; }
int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

int fill(const vmb_gated_norm_args* a, const char* what, vmb::GatedNormParams& p) {
  if (!a) return set_error(VMB_EINVAL, "%s: null args", what);
  if (a->dtype != VMB_DTYPE_BF16 && a->dtype != VMB_DTYPE_F16)
    return set_error(VMB_EINVAL, "%s: unknown dtype %d", what, a->dtype);
  if (a->param_dtype != a->dtype && a->param_dtype != VMB_DTYPE_F32)
    return set_error(VMB_EINVAL, "%s: parameters must be of the rows' dtype or fp32", what);
  if (a->cols < 8 || a->cols > 8192 || a->cols % 8)
    return set_error(VMB_ENOTSUP, "%s: %d columns are not a multiple of 8 up to 8192", what, a->cols);
  if (a->rows < 0 || a->rows > 0x7fffffff || a->seqs < 1 || a->seqs > 65535 || (a->seqs > 1 && !a->seq_start))
    return set_error(VMB_EINVAL, "%s: bad rows or sequences", what);
  if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return set_error(VMB_EINVAL, "%s: eps must be finite and not negative", what);
  const void* ptrs[] = {a->x_new, a->h, a->gate, a->scale, a->shift, a->weight, a->post_weight, a->dx, a->dy,
                        a->dgate, a->dscale, a->dshift, a->dweight, a->dpost_weight};
  for (const void* q : ptrs)
    if (!aligned16(q)) return set_error(VMB_EINVAL, "%s: tensors must be 16-byte aligned", what);
  if (!matrix_ok(a->x) || !matrix_ok(a->y) || !matrix_ok(a->dx_new) || !matrix_ok(a->dh))
    return set_error(VMB_EINVAL, "%s: rows must be 16-byte aligned", what);
  if (a->rows > 0 && !a->y.ptr && (a->gate || a->post_weight)) return set_error(VMB_EINVAL, "%s: gate and post_weight need y", what);
  p.x = a->x.ptr; p.y = a->y.ptr; p.x_row = (int)a->x.row; p.y_row = (int)a->y.row;
  p.x_new = a->x_new; p.h = a->h;
  p.gate = a->gate; p.scale = a->scale; p.shift = a->shift; p.weight = a->weight; p.post_weight = a->post_weight;
  p.stats = a->stats;
  p.seq_start = a->seqs > 1 ? a->seq_start : nullptr;
  p.dx_new = a->dx_new.ptr; p.dx_new_row = (int)a->dx_new.row;
  p.dh = a->dh.ptr; p.dh_row = (int)a->dh.row;
  p.dx = a->dx; p.dy = a->dy;
  p.dgate = a->dgate; p.dscale = a->dscale; p.dshift = a->dshift; p.dweight = a->dweight; p.dpost_weight = a->dpost_weight;
  p.rows = a->rows; p.cols = a->cols; p.seqs = a->seqs; p.layer = a->layer ? 1 : 0;
  p.eps = a->eps;
  return VMB_OK;
}

bool wants_sums(const vmb::GatedNormParams& p) { return p.dgate || p.dscale || p.dshift || p.dweight || p.dpost_weight; }
int64_t part_bytes(const vmb::GatedNormParams& p) {
  return up256(((int64_t)vmb::gated_norm_blocks(p) + p.seqs) * 3 * p.cols * 4);
}

int cuda_rc(cudaError_t e, const char* what) {
  return e == cudaSuccess ? VMB_OK : set_error(VMB_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}

}  // namespace

extern "C" {

int vmb_gated_norm_fwd(const vmb_gated_norm_args* a, void* stream) {
  vmb::GatedNormParams p{};
  int rc = fill(a, "vmb_gated_norm_fwd", p);
  if (rc) return rc;
  if (p.rows == 0) return VMB_OK;
  if (!p.x || !p.h || (p.y && !p.x_new)) return set_error(VMB_EINVAL, "vmb_gated_norm_fwd: null tensor pointer");
  vmb::count_launches(1);
  return cuda_rc(vmb::gated_norm(p, a->dtype == VMB_DTYPE_BF16, a->param_dtype == VMB_DTYPE_F32, false,
                                 static_cast<cudaStream_t>(stream)), "vmb_gated_norm_fwd");
}

int64_t vmb_gated_norm_bwd_workspace_bytes(const vmb_gated_norm_args* a) {
  vmb::GatedNormParams p{};
  if (fill(a, "vmb_gated_norm_bwd", p) != VMB_OK) return -1;
  return wants_sums(p) ? part_bytes(p) + (p.seqs > 1 ? up256((int64_t)p.seqs * p.cols * 8) : 0) : 0;
}

int vmb_gated_norm_bwd(const vmb_gated_norm_args* a, void* stream) {
  vmb::GatedNormParams p{};
  int rc = fill(a, "vmb_gated_norm_bwd", p);
  if (rc) return rc;
  if (p.rows > 0 && (!p.x || !p.dx || !p.stats || (p.y && !p.dy)))
    return set_error(VMB_EINVAL, "vmb_gated_norm_bwd: null tensor pointer");
  const int64_t need = vmb_gated_norm_bwd_workspace_bytes(a);
  if (need > 0) {
    if (!a->workspace || a->workspace_bytes < need || (reinterpret_cast<uintptr_t>(a->workspace) & 255))
      return set_error(VMB_EINVAL, "vmb_gated_norm_bwd: a 256-byte aligned workspace of %lld bytes needed", (long long)need);
    p.part = static_cast<float*>(a->workspace);
    p.seq_part = p.part + part_bytes(p) / 4;
  }
  if (p.rows == 0 && !p.part) return VMB_OK;
  const bool weights = p.part && p.seqs > 1 && (p.dweight || p.dpost_weight);
  vmb::count_launches((p.rows > 0 ? 1 : 0) + (p.part ? 1 : 0) + (weights ? 1 : 0));
  return cuda_rc(vmb::gated_norm(p, a->dtype == VMB_DTYPE_BF16, a->param_dtype == VMB_DTYPE_F32, true,
                                 static_cast<cudaStream_t>(stream)), "vmb_gated_norm_bwd");
}

}  // extern "C"
