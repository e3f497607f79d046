"""ctypes binding of the C ABI declared in ``include/vmonarch_b200.h``.

The library is the in-tree ``libvmonarch_b200.so`` built by :mod:`vmonarch_b200.build`. There is
no fallback: if the library is missing or fails to load, importing the package raises, and every
op raises if its inputs are not CUDA tensors.
"""
from __future__ import annotations

import ctypes
import os
from pathlib import Path

import torch
from torch.autograd import forward_ad

LIB_PATH = Path(os.environ.get("VMONARCH_B200_LIB", Path(__file__).resolve().parent / "libvmonarch_b200.so"))

VMB_DTYPE_BF16 = 0
VMB_DTYPE_F16 = 1
VMB_DTYPE_F32 = 2  # parameters of vmb_gated_norm only
VMB_OK = 0
_ERRNAMES = {1: "EINVAL", 2: "ENOTSUP", 3: "ECUDA"}

c_i64 = ctypes.c_int64
c_i32 = ctypes.c_int32
c_vp = ctypes.c_void_p
c_fp = ctypes.POINTER(ctypes.c_float)


ABI_VERSION = 7  # VMB_ABI_VERSION of include/vmonarch_b200.h that these structures mirror


class View(ctypes.Structure):
    """vmb_view: element (s, r, c) at c + r*row + (s % n1)*s1 + (s / n1 % n2)*s2 + (s / (n1 n2))*s3."""
    _fields_ = [("row", c_i64), ("s1", c_i64), ("s2", c_i64), ("s3", c_i64)]


class FeaLayout(ctypes.Structure):
    _fields_ = [("n1", c_i64), ("n2", c_i64)] + [(n, View) for n in (
        "q", "k", "v", "v2", "o", "dout", "grad_q", "grad_k", "grad_v", "grad_v2", "fin_q", "fin_k", "fin_v",
        "fin_v2")]


class LstepLayout(ctypes.Structure):
    _fields_ = [("n1", c_i64)] + [(n, View) for n in ("q", "out", "u", "z", "du", "dz", "dq", "dout")]


class FeaFwdArgs(ctypes.Structure):
    _fields_ = [
        ("q", c_vp), ("q_bs", c_i64),
        ("k", c_vp), ("k_bs", c_i64),
        ("v", c_vp), ("v_bs", c_i64),
        ("v2", c_vp), ("v2_bs", c_i64),
        ("o", c_vp), ("o_bs", c_i64),
        ("lse", c_vp), ("ent", c_vp),
        ("batch", c_i64), ("n_q", c_i64), ("n_kv", c_i64),
        ("d", c_i32), ("dv", c_i32), ("dv1", c_i32), ("dtype", c_i32),
        ("sm_scale", ctypes.c_float),
        ("workspace", c_vp), ("workspace_bytes", c_i64),
        ("layout", ctypes.POINTER(FeaLayout)),
        ("qkv_e4m3", c_i32),
    ]


class FeaBwdArgs(ctypes.Structure):
    _fields_ = [
        ("q", c_vp), ("q_bs", c_i64),
        ("k", c_vp), ("k_bs", c_i64),
        ("v", c_vp), ("v_bs", c_i64),
        ("v2", c_vp), ("v2_bs", c_i64),
        ("o", c_vp), ("o_bs", c_i64),
        ("dout", c_vp), ("do_bs", c_i64),
        ("lse", c_vp), ("ent", c_vp), ("dent", c_vp),
        ("grad_q", c_vp), ("grad_q_bs", c_i64),
        ("grad_k", c_vp), ("grad_k_bs", c_i64),
        ("grad_v", c_vp), ("grad_v_bs", c_i64),
        ("grad_v2", c_vp), ("grad_v2_bs", c_i64),
        ("workspace", c_vp), ("workspace_bytes", c_i64),
        ("batch", c_i64), ("n_q", c_i64), ("n_kv", c_i64),
        ("d", c_i32), ("dv", c_i32), ("dv1", c_i32), ("dtype", c_i32),
        ("grad_mode", c_i32), ("v_is_k", c_i32),
        ("sm_scale", ctypes.c_float),
        ("delta", c_vp),
        ("deterministic", c_i32),
        ("fin_q", c_vp), ("fin_q_bs", c_i64),
        ("fin_k", c_vp), ("fin_k_bs", c_i64),
        ("fin_v", c_vp), ("fin_v_bs", c_i64),
        ("fin_v2", c_vp), ("fin_v2_bs", c_i64),
        ("layout", ctypes.POINTER(FeaLayout)),
    ]


class LstepArgs(ctypes.Structure):
    _fields_ = [
        ("q", c_vp), ("out", c_vp), ("ent", c_vp),
        ("u", c_vp), ("z", c_vp),
        ("du", c_vp), ("dz", c_vp),
        ("dq", c_vp), ("dout", c_vp),
        ("bh", c_i64), ("m", c_i64), ("b", c_i64),
        ("d", c_i32), ("dw", c_i32), ("dtype", c_i32), ("last", c_i32),
        ("skip_rows", c_i64),
        ("scale", ctypes.c_float), ("min_col_mass", ctypes.c_float),
        ("dq_store", c_i32),
        ("delta_out", c_vp),
        ("layout", ctypes.POINTER(LstepLayout)),
    ]


class PackedList(ctypes.Structure):
    _fields_ = [("units", c_vp), ("joins", c_vp), ("n_units", c_i32), ("n_joins", c_i32), ("n_parts", c_i32),
                ("reserved", c_i32)]


class Rows(ctypes.Structure):
    """vmb_rows: a (rows, heads, dim) tensor with contiguous columns."""
    _fields_ = [("ptr", c_vp), ("row", c_i64), ("head", c_i64)]


class PackedArgs(ctypes.Structure):
    _fields_ = [(n, Rows) for n in ("q", "k", "v", "o", "dout", "dq", "dk", "dv", "o_low")] + [
        ("lse", c_vp),
        ("q_total", c_i64), ("k_total", c_i64), ("stat_rows", c_i64),
        ("heads", c_i32), ("kv_heads", c_i32), ("dim", c_i32), ("dtype", c_i32), ("causal", c_i32),
        ("sm_scale", ctypes.c_float),
        ("units", PackedList), ("q_units", PackedList), ("kv_units", PackedList),
        ("workspace", c_vp), ("workspace_bytes", c_i64),
    ]


class Pages(ctypes.Structure):
    """vmb_pages: a (pages, kv_heads, page_size, dim) pool with contiguous columns."""
    _fields_ = [("ptr", c_vp), ("page", c_i64), ("head", c_i64), ("slot", c_i64)]


class PagedArgs(ctypes.Structure):
    _fields_ = [
        ("q", Rows), ("o", Rows), ("k", Pages), ("v", Pages),
        ("table", c_vp), ("lengths", c_vp), ("lse", c_vp),
        ("batch", c_i64), ("table_stride", c_i64), ("table_width", c_i64), ("num_pages", c_i64),
        ("heads", c_i32), ("kv_heads", c_i32), ("dim", c_i32), ("page_size", c_i32), ("dtype", c_i32),
        ("sm_scale", ctypes.c_float),
        ("workspace", c_vp), ("workspace_bytes", c_i64),
    ]


class PageScales(ctypes.Structure):
    """vmb_page_scales: a (pages, kv_heads) tensor of float32."""
    _fields_ = [("ptr", c_vp), ("page", c_i64), ("head", c_i64)]


class CacheArgs(ctypes.Structure):
    _fields_ = [("k_scale", PageScales), ("v_scale", PageScales), ("window", c_i32), ("sinks", c_i32)]


class MoveE4m3Args(ctypes.Structure):
    _fields_ = [("k_new", Rows), ("v_new", Rows), ("k", Pages), ("v", Pages), ("k_scale", PageScales), ("v_scale", PageScales),
                ("src", c_vp), ("dst", c_vp), ("count", c_i64), ("num_pages", c_i64),
                ("kv_heads", c_i32), ("dim", c_i32), ("page_size", c_i32), ("dtype", c_i32)]


class PageBook(ctypes.Structure):
    _fields_ = [("table", c_vp), ("lengths", c_vp), ("free_pages", c_vp), ("num_free", c_vp), ("failed", c_vp),
                ("table_stride", c_i64), ("batch", c_i64), ("table_width", c_i64), ("num_pages", c_i64), ("page_size", c_i32)]


class Matrix(ctypes.Structure):
    """vmb_matrix: a (rows, cols) tensor with contiguous columns."""
    _fields_ = [("ptr", c_vp), ("row", c_i64)]


class GatedNormArgs(ctypes.Structure):
    _fields_ = [
        ("x", Matrix), ("y", Matrix), ("x_new", c_vp), ("h", c_vp),
        ("gate", c_vp), ("scale", c_vp), ("shift", c_vp), ("weight", c_vp), ("post_weight", c_vp),
        ("stats", c_vp), ("seq_start", c_vp),
        ("dx_new", Matrix), ("dh", Matrix), ("dx", c_vp), ("dy", c_vp),
        ("dgate", c_vp), ("dscale", c_vp), ("dshift", c_vp), ("dweight", c_vp), ("dpost_weight", c_vp),
        ("rows", c_i64),
        ("cols", c_i32), ("seqs", c_i32), ("dtype", c_i32), ("param_dtype", c_i32), ("layer", c_i32),
        ("eps", ctypes.c_float),
        ("workspace", c_vp), ("workspace_bytes", c_i64),
    ]


#: every symbol include/vmonarch_b200.h declares, with its ctypes signature
SIGNATURES = {
    "vmb_abi_version": (ctypes.c_int, []),
    "vmb_last_error": (ctypes.c_char_p, []),
    "vmb_kernel_launches": (ctypes.c_uint64, []),
    "vmb_test_pipeline_timeout": (ctypes.c_int, [c_i64, c_i32]),
    "vmb_device_status": (ctypes.c_int, [c_vp, ctypes.POINTER(ctypes.c_int32)]),
    "vmb_fea_fwd_workspace_bytes": (c_i64, [ctypes.POINTER(FeaFwdArgs)]),
    "vmb_fea_fwd": (ctypes.c_int, [ctypes.POINTER(FeaFwdArgs), c_vp]),
    "vmb_fea_bwd_workspace_bytes": (c_i64, [ctypes.POINTER(FeaBwdArgs)]),
    "vmb_fea_bwd_min_workspace_bytes": (c_i64, [ctypes.POINTER(FeaBwdArgs)]),
    "vmb_fea_bwd": (ctypes.c_int, [ctypes.POINTER(FeaBwdArgs), c_vp]),
    "vmb_fea_bwd_noalloc": (ctypes.c_int, [ctypes.POINTER(FeaBwdArgs), c_vp]),
    "vmb_lstep_fwd": (ctypes.c_int, [ctypes.POINTER(LstepArgs), c_vp]),
    "vmb_lstep_bwd": (ctypes.c_int, [ctypes.POINTER(LstepArgs), c_vp]),
    "vmb_cast_f32": (ctypes.c_int, [c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_i32, c_vp]),
    "vmb_cast_f32_view": (ctypes.c_int, [c_vp, ctypes.POINTER(View), c_vp, ctypes.POINTER(View), c_i64, c_i64, c_i64,
                                         c_i64, c_i64, c_i32, c_vp]),
    "vmb_quant_e4m3": (ctypes.c_int, [c_vp, ctypes.POINTER(View), c_vp, ctypes.POINTER(View), c_i64, c_i64, c_i64,
                                      c_i64, c_i64, c_i32, ctypes.c_float, c_vp]),
    "vmb_packed_fwd_workspace_bytes": (c_i64, [ctypes.POINTER(PackedArgs)]),
    "vmb_packed_bwd_workspace_bytes": (c_i64, [ctypes.POINTER(PackedArgs)]),
    "vmb_packed_fwd": (ctypes.c_int, [ctypes.POINTER(PackedArgs), c_vp]),
    "vmb_packed_bwd": (ctypes.c_int, [ctypes.POINTER(PackedArgs), c_vp]),
    "vmb_packed_window_fwd": (ctypes.c_int, [ctypes.POINTER(PackedArgs), c_i32, c_i32, c_vp]),
    "vmb_packed_window_bwd": (ctypes.c_int, [ctypes.POINTER(PackedArgs), c_i32, c_i32, c_vp]),
    "vmb_gated_norm_bwd_workspace_bytes": (c_i64, [ctypes.POINTER(GatedNormArgs)]),
    "vmb_gated_norm_fwd": (ctypes.c_int, [ctypes.POINTER(GatedNormArgs), c_vp]),
    "vmb_gated_norm_bwd": (ctypes.c_int, [ctypes.POINTER(GatedNormArgs), c_vp]),
    "vmb_paged_workspace_bytes": (c_i64, [ctypes.POINTER(PagedArgs)]),
    "vmb_paged_attention": (ctypes.c_int, [ctypes.POINTER(PagedArgs), c_vp]),
    "vmb_page_book_workspace_bytes": (c_i64, [ctypes.POINTER(PageBook)]),
    "vmb_reserve_pages": (ctypes.c_int, [ctypes.POINTER(PageBook), c_vp, c_vp, c_i64, c_vp, c_i64, c_vp]),
    "vmb_truncate_pages": (ctypes.c_int, [ctypes.POINTER(PageBook), c_vp, c_vp, c_i64, c_vp]),
    "vmb_cache_workspace_bytes": (c_i64, [ctypes.POINTER(PagedArgs), ctypes.POINTER(CacheArgs)]),
    "vmb_cache_attention": (ctypes.c_int, [ctypes.POINTER(PagedArgs), ctypes.POINTER(CacheArgs), c_vp]),
    "vmb_append_pages_e4m3": (ctypes.c_int, [ctypes.POINTER(MoveE4m3Args), c_vp]),
    "vmb_copy_pages_e4m3": (ctypes.c_int, [ctypes.POINTER(MoveE4m3Args), c_vp]),
    "vmb_append_pages": (ctypes.c_int, [ctypes.POINTER(Rows), ctypes.POINTER(Rows), ctypes.POINTER(Pages),
                                        ctypes.POINTER(Pages), c_vp, c_i64, c_i64, c_i32, c_i32, c_i32, c_vp]),
    "vmb_copy_pages": (ctypes.c_int, [ctypes.POINTER(Pages), ctypes.POINTER(Pages), c_vp, c_vp, c_i64, c_i64, c_i32,
                                      c_i32, c_i32, c_vp]),
}


def _load() -> ctypes.CDLL:
    if not LIB_PATH.exists():
        raise ImportError(
            f"vmonarch_b200: CUDA library {LIB_PATH} is missing; build it with `python vmonarch_b200/build.py`")
    lib = ctypes.CDLL(str(LIB_PATH))
    lib.vmb_abi_version.restype = ctypes.c_int
    if lib.vmb_abi_version() != ABI_VERSION:
        raise ImportError(f"vmonarch_b200: {LIB_PATH} has ABI version {lib.vmb_abi_version()}, the binding expects "
                          f"{ABI_VERSION}; rebuild it with `python vmonarch_b200/build.py`")
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name, None)
        if fn is None:  # calls are added without a new ABI version
            raise ImportError(f"vmonarch_b200: {LIB_PATH} does not have {name}; rebuild it with `python vmonarch_b200/build.py`")
        fn.restype = res
        fn.argtypes = args
    return lib


lib = _load()


class VMonarchError(RuntimeError):
    """Raised when a C-ABI call returns an error code."""


def check(rc: int, what: str) -> None:
    if rc != VMB_OK:
        msg = lib.vmb_last_error().decode(errors="replace")
        raise VMonarchError(f"{what} failed ({_ERRNAMES.get(rc, rc)}): {msg}")


def dtype_code(dt: torch.dtype) -> int:
    if dt == torch.bfloat16:
        return VMB_DTYPE_BF16
    if dt == torch.float16:
        return VMB_DTYPE_F16
    raise AssertionError(f"unsupported dtype {dt}")


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def device_status(device: torch.device) -> int:
    """OR of the pipeline-timeout codes recorded by the kernels since the last call (0 = none)."""
    out = ctypes.c_int32(0)
    launch("vmb_device_status", lambda stream: lib.vmb_device_status(stream, ctypes.byref(out)), device)
    return out.value


def stream_ptr(device: torch.device) -> int:
    return raw_stream(device.index if device.index is not None else torch.cuda.current_device())


#: handle of a device's current stream, by device index (torch.cuda.current_stream builds a Stream object around it)
raw_stream = torch._C._cuda_getCurrentRawStream
#: index of the current device
current_device = torch._C._cuda_getDevice


def launch(what: str, fn, device: torch.device, *args) -> None:
    """Calls a C entry with `args` and the current stream of `device`, which is made the current device for the call
    where it is not: the entries set up and launch kernels on the current device, and a stream handle alone does not
    name one (every device's default stream has the handle 0)."""
    index = device.index
    if index == current_device():
        rc = fn(*args, raw_stream(index))
    else:
        with torch.cuda.device(current_device() if index is None else index):
            rc = fn(*args, raw_stream(current_device()))
    if rc:
        check(rc, what)


def derived(needed: bool) -> bool:
    """Whether a call goes through its autograd function: an input requires a gradient (`needed`), or a level of
    forward-mode derivatives is open, whose dual tensors the function refuses."""
    return forward_ad._current_level >= 0 or needed and torch.is_grad_enabled()


def once_differentiable(backward):
    """torch's decorator of that name, whose bookkeeping is left out while no graph of the gradients is recorded."""
    recorded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return (recorded if torch.is_grad_enabled() else backward)(ctx, *grads)
    return run
