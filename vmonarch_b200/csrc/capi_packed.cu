// extern "C" entry points of the packed-sequence attention: argument validation, workspace carving
// and dispatch (include/vmonarch_b200.h).
#include <algorithm>
#include <cmath>

#include "../../include/vmonarch_b200.h"
#include "launch.h"
#include "packed.h"

static_assert(sizeof(vmb_packed_unit) == sizeof(vmb::PackedUnit), "unit layouts agree");

namespace {

using vmb::set_error;

int64_t up256(int64_t x);
// Partial tiles of split units: [parts][heads][rows][64 or 128] fp32, or with dim 0 a (max, sum) pair a row.
int64_t part_bytes(int64_t parts, int64_t heads, int rows, int dim) {
  return up256(parts * heads * rows * (dim == 0 ? 2 : dim > 64 ? 128 : 64) * 4);
}

int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

int cuda_rc(cudaError_t e, const char* what) {
  return e == cudaSuccess ? VMB_OK : set_error(VMB_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}

// A view the kernels can address: 16-byte aligned base, rows and heads at non-negative multiples of 16 bytes.
bool rows_ok(const vmb_rows& r) {
  return r.ptr && (reinterpret_cast<uintptr_t>(r.ptr) & 15) == 0 && r.row >= 0 && r.head >= 0 && r.row % 8 == 0 &&
         r.head % 8 == 0;
}
vmb::View view(const vmb_rows& r) { return vmb::View{r.row, r.head, 0, 0}; }

bool list_ok(const vmb_packed_list& l) {
  return l.n_units >= 0 && l.n_joins >= 0 && l.n_parts >= 0 && (l.n_units == 0 || l.units) &&
         (l.n_joins == 0 || l.joins);
}

int check(const vmb_packed_args* a, const char* what, bool bwd) {
  if (!a) return set_error(VMB_EINVAL, "%s: null args", what);
  if (a->dtype != VMB_DTYPE_BF16 && a->dtype != VMB_DTYPE_F16)
    return set_error(VMB_EINVAL, "%s: unknown dtype %d", what, a->dtype);
  if (a->q_total < 0 || a->k_total < 0 || a->q_total > 0x7fffffff || a->k_total > 0x7fffffff || a->stat_rows < 0 ||
      (bwd && a->stat_rows > 0x7fffffff))
    return set_error(VMB_EINVAL, "%s: bad row counts", what);
  if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads)
    return set_error(VMB_EINVAL, "%s: heads=%d is not a multiple of kv_heads=%d", what, a->heads, a->kv_heads);
  if (a->dim < 8 || a->dim > 128 || a->dim % 8)
    return set_error(VMB_ENOTSUP, "%s: head dim %d is not a multiple of 8 up to 128", what, a->dim);
  if (!(a->sm_scale >= 0.f) || !std::isfinite(a->sm_scale))
    return set_error(VMB_EINVAL, "%s: sm_scale must be finite and not negative", what);
  if (!list_ok(a->units) || !list_ok(a->q_units) || !list_ok(a->kv_units))
    return set_error(VMB_EINVAL, "%s: malformed unit list", what);
  if (a->q_total > 0 && (!rows_ok(a->q) || !rows_ok(a->o) || (a->o_low.ptr && !rows_ok(a->o_low))))
    return set_error(VMB_EINVAL, "%s: q, o and o_low need 16-byte aligned rows", what);
  if (a->k_total > 0 && (!rows_ok(a->k) || !rows_ok(a->v)))
    return set_error(VMB_EINVAL, "%s: k and v need 16-byte aligned rows", what);
  if (bwd) {
    if (a->q_total > 0 && (!rows_ok(a->dout) || !rows_ok(a->dq) || !a->o_low.ptr || !a->lse))
      return set_error(VMB_EINVAL, "%s: dout and dq need 16-byte aligned rows, o_low and lse a buffer", what);
    if (a->k_total > 0 && (!rows_ok(a->dk) || !rows_ok(a->dv)))
      return set_error(VMB_EINVAL, "%s: dk and dv need 16-byte aligned rows", what);
  }
  return VMB_OK;
}

int workspace(const vmb_packed_args* a, const char* what, int64_t need) {
  if (need > 0 && (!a->workspace || a->workspace_bytes < need || (reinterpret_cast<uintptr_t>(a->workspace) & 255)))
    return set_error(VMB_EINVAL, "%s: a 256-byte aligned workspace of %lld bytes needed", what, (long long)need);
  return VMB_OK;
}

// Heads whose keys and values are walked together: as many as keep
// about 48 MB between them, so that the blocks in flight share them in L2 (126 MB on B200).
int head_chunk(int64_t bytes_per_head, int heads) {
  const int64_t n = (int64_t(48) << 20) / std::max<int64_t>(bytes_per_head, 1);
  return (int)std::max<int64_t>(1, std::min<int64_t>(n, heads));
}

// Statistics of a backward: three planes of rows, a value per 128 rows and head, 128 per 128 rows and key head.
int64_t plane_bytes(const vmb_packed_args* a) { return up256(3 * a->heads * a->stat_rows * 4); }
int64_t tile_bytes(const vmb_packed_args* a) { return up256(a->heads * (a->stat_rows / 128) * 4); }
int64_t stat_bytes(const vmb_packed_args* a) {
  return plane_bytes(a) + tile_bytes(a) + up256(a->kv_heads * (a->stat_rows / 128) * 128 * 4);
}

vmb::PackedParams params(const vmb_packed_args* a) {
  vmb::PackedParams p{};
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.group = a->heads / a->kv_heads;
  p.dim = a->dim;
  p.causal = a->causal ? 1 : 0;
  p.q_total = a->q_total;
  p.k_total = a->k_total;
  p.stat_rows = a->stat_rows;
  p.sm_scale = a->sm_scale;
  p.q = a->q.ptr; p.k = a->k.ptr; p.v = a->v.ptr; p.o = a->o.ptr; p.o_low = a->o_low.ptr;
  p.dout = a->dout.ptr; p.dq = a->dq.ptr; p.dk = a->dk.ptr; p.dv = a->dv.ptr;
  p.lse = a->lse;
  vmb::test_timeout(&p.wait_limit, &p.hold_loads);
  p.qv = view(a->q); p.kv = view(a->k); p.vv = view(a->v); p.ov = view(a->o); p.olv = view(a->o_low);
  p.dov = view(a->dout); p.dqv = view(a->dq); p.dkv = view(a->dk); p.dvv = view(a->dv);
  return p;
}

}  // namespace

extern "C" {

int64_t vmb_packed_fwd_workspace_bytes(const vmb_packed_args* a) {
  if (!a || a->heads < 1 || a->units.n_parts < 0 || a->dim > 128) return -1;
  return part_bytes(a->units.n_parts, a->heads, 256, a->dim) + part_bytes(a->units.n_parts, a->heads, 256, 0);
}

int vmb_packed_fwd(const vmb_packed_args* a, void* stream) {
  int rc = check(a, "vmb_packed_fwd", false);
  if (rc) return rc;
  if (a->units.n_units == 0) return VMB_OK;
  vmb::PackedParams p = params(a);
  p.units = reinterpret_cast<const vmb::PackedUnit*>(a->units.units);
  p.n_units = a->units.n_units;
  p.head_chunk = std::min(a->heads, p.group * head_chunk(4 * a->k_total * a->dim, a->kv_heads));
  if ((rc = workspace(a, "vmb_packed_fwd", vmb_packed_fwd_workspace_bytes(a)))) return rc;
  if (a->units.n_parts > 0) {
    p.joins = a->units.joins;
    p.n_joins = a->units.n_joins;
    p.part = static_cast<float*>(a->workspace);
    p.part_ml = p.part + part_bytes(a->units.n_parts, a->heads, 256, a->dim) / 4;
  }
  vmb::count_launches(p.n_joins > 0 ? 2 : 1);
  return cuda_rc(vmb::packed_fwd(p, a->dtype == VMB_DTYPE_BF16, static_cast<cudaStream_t>(stream)), "vmb_packed_fwd");
}

int64_t vmb_packed_bwd_workspace_bytes(const vmb_packed_args* a) {
  if (!a || a->heads < 1 || a->kv_heads < 1 || a->stat_rows < 0 || a->q_units.n_parts < 0 || a->kv_units.n_parts < 0) return -1;
  return stat_bytes(a) + part_bytes(a->q_units.n_parts, a->heads, 128, a->dim) +
         part_bytes(a->kv_units.n_parts, 2 * a->kv_heads, 128, a->dim);
}

int vmb_packed_bwd(const vmb_packed_args* a, void* stream) {
  int rc = check(a, "vmb_packed_bwd", true);
  if (rc) return rc;
  if (a->q_units.n_units == 0 && a->kv_units.n_units == 0) return VMB_OK;
  if ((rc = workspace(a, "vmb_packed_bwd", vmb_packed_bwd_workspace_bytes(a)))) return rc;
  vmb::PackedParams dq = params(a), kv = dq;
  dq.stats = kv.stats = static_cast<float*>(a->workspace);
  dq.tile_scale = kv.tile_scale = dq.stats + plane_bytes(a) / 4;
  dq.centre = kv.centre = dq.tile_scale + tile_bytes(a) / 4;
  dq.units = reinterpret_cast<const vmb::PackedUnit*>(a->q_units.units);
  dq.n_units = a->q_units.n_units;
  dq.head_chunk = std::min(a->heads, dq.group * head_chunk(4 * a->k_total * a->dim, a->kv_heads));
  kv.units = reinterpret_cast<const vmb::PackedUnit*>(a->kv_units.units);
  kv.n_units = a->kv_units.n_units;
  kv.head_chunk = a->kv_heads;  // all of them: units of a second chunk would start too late to end evenly
  dq.joins = a->q_units.joins;
  dq.n_joins = a->q_units.n_parts > 0 ? a->q_units.n_joins : 0;
  dq.part = dq.stats + stat_bytes(a) / 4;
  kv.joins = a->kv_units.joins;
  kv.n_joins = a->kv_units.n_parts > 0 ? a->kv_units.n_joins : 0;
  kv.part = dq.part + part_bytes(a->q_units.n_parts, a->heads, 128, a->dim) / 4;
  vmb::count_launches((dq.n_units > 0 ? 2 : 0) + (kv.n_units > 0 ? 1 : 0) + (dq.n_joins > 0) + (kv.n_joins > 0));
  return cuda_rc(vmb::packed_bwd(dq, kv, a->dtype == VMB_DTYPE_BF16, static_cast<cudaStream_t>(stream)),
                 "vmb_packed_bwd");
}

}  // extern "C"
