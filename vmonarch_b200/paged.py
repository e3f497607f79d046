"""A paged key / value cache, and attention of one new token per sequence over it (no reference
counterpart).

The pool of a layer is a pair of tensors (num_pages, Hk, page_size, D). A sequence's tokens fill pages
listed in its row of a page table: token t lies in slot t % page_size of page table[b, t // page_size].
:func:`append_pages`, :func:`copy_pages` and :func:`paged_attention` work on such tensors, wherever they come
from; :class:`PagedKVCache` holds the pools of a model's layers and keeps the book of their pages.
"""
from __future__ import annotations

import ctypes
import struct

import numpy as np
import torch

from . import _native as N
from .kernel import SUPPORTED_DTYPES
from .packed import MAX_DIM, _place


def _pages(t, n, h, ps, d):
    """vmb_pages of a pool (n pages, h heads, ps slots, d columns), which the kernels address in place."""
    ptr, (page, head, slot, col) = t.data_ptr(), t.stride()
    if n == 1 or h == 1 or ps == 1:  # such strides do not count
        page, head, slot = page if n > 1 else 0, head if h > 1 else 0, slot if ps > 1 else 0
    assert col == 1 or d == 1, "pools need contiguous columns"
    assert not ptr & 15 and page >= 0 and head >= 0 and slot >= 0 and not (page | head | slot) & 7, \
        "pools need 16-byte aligned rows"
    return ptr, page, head, slot


def _check_pools(k_pages, v_pages):
    """(pages, heads, page size, dim, dtype, device) of a pair of pools."""
    shape, dtype, device = k_pages.shape, k_pages.dtype, k_pages.device
    assert len(shape) == 4 and v_pages.shape == shape, "pools must be (num_pages, Hk, page_size, D)"
    assert dtype in SUPPORTED_DTYPES and v_pages.dtype == dtype, f"unsupported dtype {dtype}"
    n, h, ps, d = shape
    assert 8 <= d <= MAX_DIM and d % 8 == 0, f"head dim {d} is not a multiple of 8 up to {MAX_DIM}"
    assert n >= 1 and h >= 1 and ps >= 1, "pools need at least one page, head and slot"
    assert k_pages.is_cuda and v_pages.device == device, "pools must be on one CUDA device"
    return n, h, ps, d, dtype, device


def _check_index(t, name, dim, device):
    assert t.dtype == torch.int32 and t.dim() == dim and t.device == device, \
        f"{name} must be int32, {dim}-dimensional and on the pools' device"


def paged_attention(q, k_pages, v_pages, page_table, lengths, *, sm_scale=None, return_lse=False):
    """
    Attention of one new token per sequence over a paged cache (inference: carries no gradient).

    Args:
        q: (B, H, D), bf16 or fp16, D a multiple of 8 up to 128
        k_pages, v_pages: (num_pages, Hk, page_size, D), the same dtype, H a multiple of Hk; any strides
            with contiguous columns and 16-byte aligned rows, any page size
        page_table: (B, width) int32, the pages of each sequence; entries past its length are not read.
            A page id outside the pool reads as zeros.
        lengths: (B,) int32, the tokens each sequence has cached, the new one's among them if it is to
            see itself; at most width * page_size count
        sm_scale: softmax scale, not negative; defaults to 1 / sqrt(D)
        return_lse: also return the log of each softmax's sum
    Returns:
        o: (B, H, D); 0 for a sequence of length 0
        lse (with return_lse): (B, H) float32, natural logarithm, -inf for a sequence of length 0
    Table and lengths stay on the device: the call does not wait for it and can be captured in a CUDA
    graph whose replays see other lengths.
    """
    num, hk, page_size, d, dtype, device = _check_pools(k_pages, v_pages)
    shape = q.shape
    assert len(shape) == 3 and q.dtype == dtype and shape[2] == d and q.device == device, \
        "q must be (B, H, D) with the pools' D, dtype and device"
    b, h, _ = shape
    assert h >= 1 and h % hk == 0, "H must be a multiple of Hk"
    _check_index(page_table, "page_table", 2, device)
    _check_index(lengths, "lengths", 1, device)
    rows, width = page_table.shape
    assert rows == b and lengths.size(0) == b, "page_table and lengths must have a row per sequence"
    sm_scale = d ** -0.5 if sm_scale is None else float(sm_scale)
    assert 0 <= sm_scale < float("inf"), "sm_scale must be finite and not negative"
    q, *qr = _place(q)
    stride, col = page_table.stride()
    if width > 1 and col != 1 or b > 1 and stride < width:
        page_table, stride = page_table.contiguous(), width
    lengths = lengths.contiguous()
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((b, h), dtype=torch.float32, device=device) if return_lse else None
    if b:
        a = N.PagedArgs()
        _PAGED.pack_into(a, 0, *qr, o.data_ptr(), h * d, d, *_pages(k_pages, num, hk, page_size, d), *_pages(v_pages, num, hk, page_size, d), page_table.data_ptr(),
                         lengths.data_ptr(), lse.data_ptr() if return_lse else 0, b, stride if b > 1 else width, width, num,
                         h, hk, d, page_size, N.dtype_code(dtype), sm_scale)
        size = N.lib.vmb_paged_workspace_bytes(ctypes.byref(a))
        if size > 0:
            ws = torch.empty(size, dtype=torch.uint8, device=device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), size
        N.launch("vmb_paged_attention", N.lib.vmb_paged_attention, device, ctypes.byref(a))
    return (o, lse) if return_lse else o


# vmb_paged_args up to its workspace
_PAGED = struct.Struct("21q5if")
assert _PAGED.size == N.PagedArgs.workspace.offset


def append_pages(k, v, k_pages, v_pages, slots):
    """
    Writes new rows into their slots of a pool, in place.

    Args:
        k, v: (T, Hk, D), the pools' dtype
        k_pages, v_pages: (num_pages, Hk, page_size, D)
        slots: (T,) int32, page * page_size + slot of each row. Slots outside the pool (negative ones, as
            padding) are skipped; no slot may be named twice.
    """
    num, hk, page_size, d, dtype, device = _check_pools(k_pages, v_pages)
    assert k.dim() == 3 and v.shape == k.shape and k.shape[1:] == (hk, d), "k and v must be (T, Hk, D) with the pools' Hk and D"
    assert k.dtype == dtype and v.dtype == dtype, "k and v must have the pools' dtype"
    assert k.device == device and v.device == device, "k and v must be on the pools' device"
    _check_index(slots, "slots", 1, device)
    n = k.size(0)
    assert slots.size(0) == n, "slots must name one slot per row"
    assert num * page_size < 2 ** 31, "slots are 32-bit: the pool has too many"
    if n == 0:
        return
    k, *kr = _place(k)
    v, *vr = _place(v)
    slots = slots.contiguous()
    pool = num, hk, page_size, d
    N.launch("vmb_append_pages", N.lib.vmb_append_pages, device, N.Rows(*kr), N.Rows(*vr), N.Pages(*_pages(k_pages, *pool)),
             N.Pages(*_pages(v_pages, *pool)), slots.data_ptr(), n, num, hk, d, page_size)


def copy_pages(k_pages, v_pages, src, dst):
    """
    Copies page src[i] to page dst[i] of both pools, in place.

    Args:
        k_pages, v_pages: (num_pages, Hk, page_size, D)
        src, dst: (n,) int32 page ids. Pairs with a page outside the pool are skipped; no destination may be
            another pair's source or destination.
    """
    num, hk, page_size, d, dtype, device = _check_pools(k_pages, v_pages)
    _check_index(src, "src", 1, device)
    _check_index(dst, "dst", 1, device)
    n = src.size(0)
    assert dst.size(0) == n, "src and dst must have the same length"
    if n == 0:
        return
    src, dst = src.contiguous(), dst.contiguous()
    pool = num, hk, page_size, d
    N.launch("vmb_copy_pages", N.lib.vmb_copy_pages, device, N.Pages(*_pages(k_pages, *pool)),
             N.Pages(*_pages(v_pages, *pool)), src.data_ptr(), dst.data_ptr(), n, num, hk, d, page_size)


class PagedKVCache:
    """
    The pools of a model's layers and the book of their pages.

    Sequences are known by the integers that :meth:`add` and :meth:`fork` return. The book lives on the host
    and is one for all layers; the tensors that a step needs (:meth:`reserve`, :meth:`tables`) are made
    from it once a step. Forked sequences share their pages, which are counted; a shared page is copied
    when one of its owners is about to write into it.

    Args:
        num_pages, page_size: size of each layer's pools
        kv_heads, head_dim: of the keys and values; head_dim a multiple of 8 up to 128
        layers: number of layers
        dtype, device: of the pools
    """

    def __init__(self, num_pages, page_size, kv_heads, head_dim, *, layers=1, dtype=torch.bfloat16, device="cuda"):
        assert num_pages >= 1 and page_size >= 1 and kv_heads >= 1 and layers >= 1, "sizes must be positive"
        assert num_pages * page_size < 2 ** 31, "slots are 32-bit: fewer pages or smaller ones"
        assert dtype in SUPPORTED_DTYPES, f"unsupported dtype {dtype}"
        assert 8 <= head_dim <= MAX_DIM and head_dim % 8 == 0, f"head dim {head_dim} is not a multiple of 8 up to {MAX_DIM}"
        self.page_size, self.num_pages = page_size, num_pages
        shape = (layers, num_pages, kv_heads, page_size, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.device = self.k.device
        self._free = list(range(num_pages - 1, -1, -1))  # taken from the end: low pages first
        self._owners = [0] * num_pages
        self._pages, self._length = {}, {}
        self._next = 0

    @property
    def num_free(self) -> int:
        """Pages that no sequence holds."""
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._length[seq]

    def pages(self, seq: int) -> list[int]:
        return list(self._pages[seq])

    def add(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._length[seq] = [], 0
        return seq

    def fork(self, seq: int) -> int:
        """A new sequence with the tokens of `seq`, whose pages it shares."""
        new = self.add()
        self._pages[new], self._length[new] = list(self._pages[seq]), self._length[seq]
        for page in self._pages[seq]:
            self._owners[page] += 1
        return new

    def free(self, seq: int) -> None:
        """Gives up a sequence; pages that no other one shares become free."""
        for page in self._pages.pop(seq):
            self._owners[page] -= 1
            if self._owners[page] == 0:
                self._free.append(page)
        del self._length[seq]

    def _ints(self, values):
        return torch.from_numpy(np.asarray(values, dtype=np.int32)).to(self.device)

    def _copy(self, src, dst):
        if src:
            src, dst = self._ints(src), self._ints(dst)
            for k, v in zip(self.k, self.v):
                copy_pages(k, v, src, dst)

    def reserve(self, seqs, counts) -> torch.Tensor:
        """
        Room for counts[i] more tokens of sequence seqs[i]: their slots, (sum(counts),) int32, for
        :meth:`write` in every layer. Pages shared with other sequences that are written into are copied
        first. Raises MemoryError, with nothing changed, when there are not enough free pages.
        """
        seqs, counts = list(seqs), [int(c) for c in counts]
        assert len(seqs) == len(counts) and len(set(seqs)) == len(seqs), "one count per sequence, each named once"
        assert all(c >= 0 for c in counts), "counts must not be negative"
        ps, owners = self.page_size, {}
        shared, need = [], 0
        for seq, n in zip(seqs, counts):
            have, length = self._pages[seq], self._length[seq]
            need += -(-(length + n) // ps) - len(have)
            if n and length % ps:
                page = have[-1]
                left = owners.setdefault(page, self._owners[page])
                if left > 1:
                    owners[page] -= 1  # the last owner that writes keeps it
                    shared.append(seq)
                    need += 1
        if need > len(self._free):
            raise MemoryError(f"paged cache: {need} pages needed, {len(self._free)} of {self.num_pages} free")
        src, dst = [], []
        for seq in shared:
            old, new = self._pages[seq][-1], self._take()
            self._owners[old] -= 1
            self._pages[seq][-1] = new
            src.append(old)
            dst.append(new)
        self._copy(src, dst)
        slots = []
        for seq, n in zip(seqs, counts):
            have, length = self._pages[seq], self._length[seq]
            while len(have) * ps < length + n:
                have.append(self._take())
            at = np.arange(length, length + n)
            slots.append(np.asarray(have, dtype=np.int64)[at // ps] * ps + at % ps if n else at)
            self._length[seq] = length + n
        return self._ints(np.concatenate(slots) if slots else [])

    def _take(self) -> int:
        page = self._free.pop()
        self._owners[page] = 1
        return page

    def write(self, layer: int, k, v, slots) -> None:
        """Rows k, v (T, Hk, D) of one layer into the slots that :meth:`reserve` gave."""
        append_pages(k, v, self.k[layer], self.v[layer], slots)

    def tables(self, seqs):
        """(page table, lengths) of the sequences, for :meth:`attend` in every layer."""
        rows = [self._pages[s] for s in seqs]
        table = np.zeros((len(rows), max([len(r) for r in rows], default=0)), dtype=np.int32)
        for i, r in enumerate(rows):
            table[i, :len(r)] = r
        return self._ints(table), self._ints([self._length[s] for s in seqs])

    def attend(self, layer: int, q, table, lengths, *, sm_scale=None):
        """:func:`paged_attention` of one token per sequence over a layer's pool."""
        return paged_attention(q, self.k[layer], self.v[layer], table, lengths, sm_scale=sm_scale)

    def compact(self) -> int:
        """Moves the pages in use to the lowest ids (tables made before are void) and returns how many
        are in use. The pools' tails can then be left out of a copy or a snapshot."""
        used = [p for p in range(self.num_pages) if self._owners[p]]
        n = len(used)
        holes = [p for p in range(n) if not self._owners[p]]
        movers = [p for p in used if p >= n]
        self._copy(movers, holes)
        new = dict(zip(movers, holes))
        for pages in self._pages.values():
            pages[:] = [new.get(p, p) for p in pages]
        for old, at in new.items():
            self._owners[at], self._owners[old] = self._owners[old], 0
        self._free = list(range(self.num_pages - 1, n - 1, -1))
        return n
