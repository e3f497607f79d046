"""The C ABI of the packed, paged and gated-norm calls: structures agree with their ctypes mirrors, and bad
arguments are refused before any CUDA work."""
import ctypes
import subprocess
import tempfile
from pathlib import Path

import pytest

from vmonarch_b200 import _native as N

HEADER = Path(__file__).resolve().parent.parent / "include" / "vmonarch_b200.h"
STRUCTS = {"vmb_packed_list": N.PackedList, "vmb_rows": N.Rows, "vmb_packed_args": N.PackedArgs, "vmb_pages": N.Pages,
           "vmb_paged_args": N.PagedArgs, "vmb_matrix": N.Matrix, "vmb_gated_norm_args": N.GatedNormArgs}


def test_struct_layouts_match_c_header():
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {",
             'printf("%zu\\n", sizeof(vmb_packed_unit));']
    for cname, pytype in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        lines += [f'printf("%zu\\n", offsetof({cname}, {field}));' for field, _ in pytype._fields_]
    with tempfile.TemporaryDirectory() as tmp:
        src, exe = Path(tmp) / "layout.c", Path(tmp) / "layout"
        src.write_text("\n".join(lines + ["return 0; }"]))
        subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", str(src), "-o", str(exe)], check=True)
        out = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = [48]
    for pytype in STRUCTS.values():
        want.append(ctypes.sizeof(pytype))
        want += [getattr(pytype, f).offset for f, _ in pytype._fields_]
    assert out == want


def packed(**over):
    a = N.PackedArgs()
    for name in ("q", "k", "v", "o", "dout", "dq", "dk", "dv", "o_low"):
        setattr(a, name, N.Rows(256, 256, 64))
    a.lse = 256
    a.q_total = a.k_total = a.stat_rows = 128
    a.heads, a.kv_heads, a.dim, a.dtype, a.sm_scale = 4, 2, 64, N.VMB_DTYPE_BF16, 0.125
    a.units = a.q_units = a.kv_units = N.PackedList(256, None, 1, 0, 0, 0)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over, code", [
    (dict(dtype=2), 1), (dict(dim=20), 2), (dict(dim=136), 2), (dict(dim=0), 2), (dict(heads=3), 1), (dict(kv_heads=0), 1),
    (dict(q_total=-1), 1), (dict(sm_scale=-1.0), 1), (dict(sm_scale=float("nan")), 1), (dict(q=N.Rows(None, 256, 64)), 1),
    (dict(k=N.Rows(8, 256, 64)), 1), (dict(v=N.Rows(256, 257, 64)), 1), (dict(o=N.Rows(256, 256, -64)), 1),
    (dict(units=N.PackedList(None, None, 1, 0, 0, 0)), 1), (dict(units=N.PackedList(256, None, -1, 0, 0, 0)), 1),
])
def test_packed_refusals(over, code):
    for fn in (N.lib.vmb_packed_fwd, N.lib.vmb_packed_bwd):
        assert fn(ctypes.byref(packed(**over)), None) == code
        assert N.lib.vmb_last_error()
    assert N.lib.vmb_packed_fwd(None, None) == N.lib.vmb_packed_bwd(None, None) == 1


@pytest.mark.parametrize("over", [dict(dout=N.Rows(None, 0, 0)), dict(dk=N.Rows(4, 256, 64)), dict(lse=None),
                                  dict(o_low=N.Rows(None, 0, 0)), dict(workspace=None), dict(workspace=257, workspace_bytes=1 << 30)])
def test_packed_backward_refusals(over):
    assert N.lib.vmb_packed_bwd(ctypes.byref(packed(**over)), None) == 1


def test_empty_calls_launch_nothing():
    before = N.lib.vmb_kernel_launches()
    none = N.PackedList(None, None, 0, 0, 0, 0)
    assert N.lib.vmb_packed_fwd(ctypes.byref(packed(units=none)), None) == 0
    assert N.lib.vmb_packed_bwd(ctypes.byref(packed(q_units=none, kv_units=none)), None) == 0
    assert N.lib.vmb_paged_attention(ctypes.byref(paged(batch=0)), None) == 0
    assert N.lib.vmb_gated_norm_fwd(ctypes.byref(gated(rows=0)), None) == 0
    assert N.lib.vmb_kernel_launches() == before


def paged(**over):
    a = N.PagedArgs()
    a.q = a.o = N.Rows(256, 256, 64)
    a.k = a.v = N.Pages(256, 2048, 1024, 64)
    a.table = a.lengths = a.workspace = 256
    a.workspace_bytes = 0
    a.batch, a.table_stride, a.table_width, a.num_pages = 2, 64, 64, 100
    a.heads, a.kv_heads, a.dim, a.page_size, a.dtype, a.sm_scale = 4, 2, 64, 16, N.VMB_DTYPE_F16, 0.125
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over, code", [
    (dict(dtype=2), 1), (dict(dim=12), 2), (dict(dim=256), 2), (dict(heads=5), 1), (dict(kv_heads=0), 1), (dict(page_size=0), 1),
    (dict(num_pages=-1), 1), (dict(num_pages=0), 1), (dict(batch=-1), 1), (dict(table_stride=3), 1), (dict(sm_scale=float("inf")), 1),
    (dict(q=N.Rows(8, 256, 64)), 1), (dict(k=N.Pages(256, 2048, 1024, 63)), 1), (dict(lengths=None), 1), (dict(table=None), 1),
    (dict(), 1),  # tables this wide need a workspace
])
def test_paged_refusals(over, code):
    assert N.lib.vmb_paged_attention(ctypes.byref(paged(**over)), None) == code


def test_paged_workspace():
    assert N.lib.vmb_paged_workspace_bytes(None) == -1
    assert N.lib.vmb_paged_workspace_bytes(ctypes.byref(paged(dim=12))) == -1
    assert N.lib.vmb_paged_workspace_bytes(ctypes.byref(paged())) > 0
    assert N.lib.vmb_paged_workspace_bytes(ctypes.byref(paged(table_width=8))) == 0  # items of one block


def test_move_refusals():
    rows, pages, bad = N.Rows(256, 128, 64), N.Pages(256, 2048, 1024, 64), N.Pages(8, 2048, 1024, 64)
    app = lambda k=rows, p=pages, slots=256, n=4, num=100, d=64, ps=16: N.lib.vmb_append_pages(  # noqa: E731
        ctypes.byref(k), ctypes.byref(k), ctypes.byref(p), ctypes.byref(p), slots, n, num, 2, d, ps, None)
    cpy = lambda p=pages, src=256, dst=256, n=4, num=100, d=64, ps=16: N.lib.vmb_copy_pages(  # noqa: E731
        ctypes.byref(p), ctypes.byref(p), src, dst, n, num, 2, d, ps, None)
    assert app(k=N.Rows(256, 100, 64)) == app(p=bad) == app(slots=None) == app(n=-1) == app(num=-1) == app(ps=0) == 1
    assert cpy(p=bad) == cpy(src=None) == cpy(dst=None) == cpy(n=-1) == cpy(ps=-1) == 1
    assert app(d=20) == cpy(d=20) == 2
    assert app(n=0) == cpy(n=0) == 0


def gated(**over):
    a = N.GatedNormArgs()
    a.x = a.y = a.dx_new = a.dh = N.Matrix(256, 64)
    for name in ("x_new", "h", "gate", "scale", "shift", "weight", "post_weight", "stats", "seq_start", "dx", "dy", "dgate"):
        setattr(a, name, 256)
    a.rows, a.cols, a.seqs, a.eps = 10, 64, 2, 1e-6
    a.dtype = a.param_dtype = N.VMB_DTYPE_BF16
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over, code", [
    (dict(dtype=2), 1), (dict(param_dtype=1), 1), (dict(cols=60), 2), (dict(cols=8200), 2), (dict(cols=0), 2), (dict(rows=-1), 1),
    (dict(seqs=0), 1), (dict(seqs=70000), 1), (dict(seq_start=None), 1), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1),
    (dict(x=N.Matrix(256, 65)), 1), (dict(x=N.Matrix(8, 64)), 1), (dict(x=N.Matrix(None, 64)), 1), (dict(gate=8), 1),
    (dict(y=N.Matrix(None, 0)), 1),
])
def test_gated_norm_refusals(over, code):
    for fn in (N.lib.vmb_gated_norm_fwd, N.lib.vmb_gated_norm_bwd):
        assert fn(ctypes.byref(gated(**over)), None) == code
    if "x" not in over or over["x"].ptr:
        assert N.lib.vmb_gated_norm_bwd_workspace_bytes(ctypes.byref(gated(**over))) == -1
    assert N.lib.vmb_gated_norm_fwd(ctypes.byref(gated(h=None)), None) == 1
    assert N.lib.vmb_gated_norm_bwd(ctypes.byref(gated(stats=None)), None) == 1
    assert N.lib.vmb_gated_norm_bwd(ctypes.byref(gated()), None) == 1  # no workspace
