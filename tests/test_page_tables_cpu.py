"""The page tables' and the 8-bit cache's refusals, structures and host book, without a GPU."""
import ctypes
import subprocess
import tempfile
from pathlib import Path

import pytest
import torch

from test_ops_capi import HEADER
from vmonarch_b200 import PagedKVCache, PageTables, append_pages, copy_pages, paged_attention, reserve_pages, truncate_pages
from vmonarch_b200 import _native as N

STRUCTS = {"vmb_page_scales": N.PageScales, "vmb_cache_args": N.CacheArgs, "vmb_page_book": N.PageBook,
           "vmb_move_e4m3_args": N.MoveE4m3Args}
E4M3 = torch.float8_e4m3fn


def test_struct_layouts_match_c_header():
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {"]
    want = []
    for cname, pytype in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        lines += [f'printf("%zu\\n", offsetof({cname}, {field}));' for field, _ in pytype._fields_]
        want.append(ctypes.sizeof(pytype))
        want += [getattr(pytype, f).offset for f, _ in pytype._fields_]
    with tempfile.TemporaryDirectory() as tmp:
        src, exe = Path(tmp) / "layout.c", Path(tmp) / "layout"
        src.write_text("\n".join(lines + ["return 0; }"]))
        subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", str(src), "-o", str(exe)], check=True)
        assert [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()] == want


def book(**over):
    b = N.PageBook(256, 256, 256, 256, None, 8, 4, 8, 100, 16)
    for k, v in over.items():
        setattr(b, k, v)
    return ctypes.byref(b)


@pytest.mark.parametrize("over", [
    dict(batch=-1), dict(batch=2 ** 31), dict(table_width=-1), dict(table_stride=7), dict(page_size=0), dict(num_pages=0),
    dict(num_pages=2 ** 27), dict(table=None), dict(lengths=None), dict(free_pages=None), dict(num_free=None),
])
def test_book_refusals(over):
    assert N.lib.vmb_reserve_pages(book(**over), 256, 256, 10, None, 0, None) == 1 and N.lib.vmb_last_error()
    assert N.lib.vmb_truncate_pages(book(**over), 256, None, 0, None) == 1 and N.lib.vmb_last_error()


def test_book_calls_refuse_bad_rows_and_workspaces():
    for args in ((None, 256, 256, 10, None, 0), (book(), None, 256, 10, None, 0), (book(), 256, None, 10, None, 0),
                 (book(), 256, 256, -1, None, 0), (book(), 256, 256, 2 ** 31, None, 0), (book(), 256, 256, 5000, None, 0),
                 (book(batch=2000), 256, 256, 10, 256, 100), (book(batch=2000), 256, 256, 10, 258, 10 ** 6)):
        assert N.lib.vmb_reserve_pages(*args, None) == 1
    for args in ((None, 256, None, 0), (book(), None, None, 0), (book(batch=2000), 256, None, 0),
                 (book(table_width=20000, table_stride=20000), 256, None, 0)):
        assert N.lib.vmb_truncate_pages(*args, None) == 1
    assert N.lib.vmb_page_book_workspace_bytes(None) == N.lib.vmb_page_book_workspace_bytes(book(batch=-1)) == -1
    assert N.lib.vmb_page_book_workspace_bytes(book(batch=1000)) >= 12000
    assert N.lib.vmb_truncate_pages(book(batch=0), None, None, 0, None) == 0


def paged(**over):
    a = N.PagedArgs()
    a.q = a.o = N.Rows(256, 256, 64)
    a.k = a.v = N.Pages(256, 4096, 1024, 64)
    a.table = a.lengths = 256
    a.batch, a.table_stride, a.table_width, a.num_pages = 2, 4, 4, 10
    a.heads, a.kv_heads, a.dim, a.page_size, a.dtype, a.sm_scale = 4, 2, 64, 16, 0, 0.125
    for k, v in over.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("args, cache, code", [
    ({}, dict(window=-1), 1), ({}, dict(window=4, sinks=-1), 1), ({}, dict(sinks=3), 1),
    ({}, dict(k_scale=N.PageScales(256, 2, 1)), 1), ({}, dict(v_scale=N.PageScales(256, 2, 1)), 1),
    ({}, dict(k_scale=N.PageScales(256, -2, 1), v_scale=N.PageScales(256, 2, 1)), 1),
    (dict(dim=40), dict(k_scale=N.PageScales(256, 2, 1), v_scale=N.PageScales(256, 2, 1)), 2),
    (dict(k=N.Pages(256, 4096, 1024, 72)), dict(k_scale=N.PageScales(256, 2, 1), v_scale=N.PageScales(256, 2, 1)), 1),
    (dict(dtype=2), {}, 1), (dict(heads=3), {}, 1), (dict(lengths=None), dict(window=4), 1),
])
def test_cache_attention_refusals(args, cache, code):
    c = N.CacheArgs()
    for k, v in cache.items():
        setattr(c, k, v)
    assert N.lib.vmb_cache_attention(paged(**args), ctypes.byref(c), None) == code and N.lib.vmb_last_error()


def move8(**over):
    r, p, s = N.Rows(256, 128, 64), N.Pages(256, 2048, 1024, 64), N.PageScales(256, 2, 1)
    a = N.MoveE4m3Args(r, r, p, p, s, s, 256, 256, 3, 10, 2, 64, 16, 0)
    for k, v in over.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_e4m3_move_refusals():
    both = [(dict(k=N.Pages(256, 2048, 1024, 72)), 1), (dict(v=N.Pages(264, 2048, 1024, 64)), 1), (dict(k_scale=N.PageScales(None, 2, 1)), 1),
            (dict(v_scale=N.PageScales(256, -1, 1)), 1), (dict(dst=None), 1), (dict(count=-1), 1), (dict(num_pages=0), 1),
            (dict(dim=40), 2), (dict(dim=144), 2)]
    for over, code in both + [(dict(k_new=N.Rows(8, 128, 64)), 1), (dict(v_new=N.Rows(None, 128, 64)), 1), (dict(dtype=2), 1)]:
        assert N.lib.vmb_append_pages_e4m3(move8(**over), None) == code and N.lib.vmb_last_error()
    for over, code in both + [(dict(src=None), 1)]:
        assert N.lib.vmb_copy_pages_e4m3(move8(**over), None) == code and N.lib.vmb_last_error()
    assert N.lib.vmb_append_pages_e4m3(None, None) == N.lib.vmb_copy_pages_e4m3(None, None) == 1
    assert N.lib.vmb_append_pages_e4m3(move8(count=0), None) == N.lib.vmb_copy_pages_e4m3(move8(count=0), None) == 0


def test_page_tables_start_empty():
    t = PageTables(10, 4, 3, 5, pages=[7, 2, 9], device="cpu")
    assert t.free_pages.tolist()[:3] == [9, 7, 2] and t.num_free.tolist() == [3] and t.lengths.tolist() == [0, 0, 0]
    assert tuple(t.table.shape) == (3, 5)
    t.check()
    t.failed.fill_(5)
    with pytest.raises(MemoryError, match="not enough free pages, more tokens"):
        t.check()
    t.check()
    for bad in (dict(num_pages=0), dict(page_size=0), dict(batch=0), dict(width=0), dict(num_pages=2 ** 30), dict(pages=[1, 1]),
                dict(pages=[10]), dict(pages=[-1])):
        with pytest.raises(AssertionError):
            PageTables(**{**dict(num_pages=10, page_size=4, batch=3, width=5, device="cpu"), **bad})


def test_pages_handed_to_tables_on_the_device():
    cache = PagedKVCache(10, 4, 1, 16, dtype=E4M3, device="cpu")
    a = cache.add()
    cache.reserve([a], [9])
    t = cache.page_tables(2, 3, 4)
    assert cache.num_free == 3 and sorted(t.free_pages[:4].tolist()) == [3, 4, 5, 6]
    cache.reserve([a], [12])
    assert sorted(cache.pages(a)) == [0, 1, 2, 7, 8, 9]
    with pytest.raises(MemoryError):
        cache.page_tables(2, 3, 1)
    with pytest.raises(AssertionError, match="moved"):
        cache.compact()
    for other in (PageTables(10, 4, 2, 3, device="cpu"), object()):
        with pytest.raises(AssertionError, match="taken back"):
            cache.take_back(other)


def test_8_bit_pools_refuse():
    with pytest.raises(AssertionError, match="multiple of 16"):
        PagedKVCache(4, 8, 1, 24, dtype=E4M3, device="cpu")
    cache = PagedKVCache(4, 8, 2, 32, layers=3, dtype=E4M3, device="cpu")
    assert cache.k_scale.shape == cache.v_scale.shape == (3, 4, 2) and not cache.k_scale.any() and cache.k.dtype == E4M3
    assert PagedKVCache(4, 8, 2, 32, device="cpu").k_scale is None
    k, s = cache.k[0], cache.k_scale[0]
    rows, i = torch.zeros(1, 2, 32, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for kw in ({}, dict(k_scale=s), dict(k_scale=s, v_scale=s.double()), dict(k_scale=s, v_scale=s[:1])):
        with pytest.raises(AssertionError, match="scale"):
            paged_attention(rows, k, k, i[None], i, **kw)
        with pytest.raises(AssertionError, match="scale"):
            append_pages(rows, rows, k, k, i, **kw)
        with pytest.raises(AssertionError, match="scale"):
            copy_pages(k, k, i, i, **kw)
    with pytest.raises(AssertionError, match="scale"):
        paged_attention(rows, k.to(torch.bfloat16), k.to(torch.bfloat16), i[None], i, k_scale=s, v_scale=s)
    with pytest.raises(AssertionError, match="CUDA"):
        paged_attention(rows, k, k, i[None], i, k_scale=s, v_scale=s)
    for call in (reserve_pages, truncate_pages):
        kw = dict(total=1) if call is reserve_pages else {}
        with pytest.raises(AssertionError, match="CUDA"):
            call(i[None], i.clone(), i.clone(), i.clone(), i.clone(), page_size=4, **kw)
