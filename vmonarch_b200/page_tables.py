"""Page tables, slot maps and the stack of free pages of a paged cache, kept on the GPU (no reference counterpart).

:class:`PagedKVCache` keeps its book on the host and copies tables and slots to the device for every step. Here the book is
tensors: a step that knows its sequences' new tokens as a tensor of counts takes pages, fills the tables and gets the slots
without the host, and can be captured in a CUDA graph together with what reads them.
"""
from __future__ import annotations

import ctypes
import operator
import struct

import torch

from . import _native as N

#: what `failed` says, by its bits
_FAILURES = {1: "not enough free pages", 2: "a sequence is longer than its row of the page table holds",
             4: "more tokens than rows, or a negative length or count", 8: "more pages returned than there are"}


def _book(page_table, lengths, want, free_pages, num_free, page_size, failed):
    """vmb_page_book of the tensors, and their device."""
    device, int32 = page_table.device, torch.int32
    assert page_table.dtype == int32 and page_table.dim() == 2, "page_table must be int32 and 2-dimensional"
    batch, width = page_table.shape
    assert lengths.dtype == int32 and lengths.device == device and lengths.shape == (batch,), \
        "lengths must be int32, an entry per row of the page table and on its device"
    assert want.dtype == int32 and want.device == device and want.shape == (batch,), \
        "counts, or lengths to keep, must be int32, an entry per row of the page table and on its device"
    assert free_pages.dtype == int32 and free_pages.device == device and free_pages.dim() == 1, \
        "free_pages must be int32, 1-dimensional and on the page table's device"
    assert num_free.dtype == int32 and num_free.device == device and num_free.shape == (1,), \
        "num_free must be one int32 on the page table's device"
    stride, col = page_table.stride()
    assert width <= 1 or col == 1 and (batch <= 1 or stride >= width), "the page table's rows must be contiguous and apart"
    num_pages, page_size = free_pages.size(0), operator.index(page_size)
    assert page_size >= 1 and num_pages >= 1, "page_size and free_pages must not be empty"
    assert num_pages * page_size < 2 ** 31, "slots are 32-bit: the pool has too many"
    assert lengths.is_contiguous() and free_pages.is_contiguous(), "lengths and free_pages are written in place and must be contiguous"
    if failed is not None:
        assert failed.dtype == int32 and failed.device == device and failed.numel() == 1, "failed must be one int32 on the same device"
    assert page_table.is_cuda, "the book must be on a CUDA device"
    book = N.PageBook()
    _BOOK.pack_into(book, 0, page_table.data_ptr(), lengths.data_ptr(), free_pages.data_ptr(), num_free.data_ptr(),
                    0 if failed is None else failed.data_ptr(), stride if batch > 1 else width, batch, width, num_pages, page_size)
    return book, device, batch, width


# vmb_page_book
_BOOK = struct.Struct("9qi")
assert _BOOK.size <= ctypes.sizeof(N.PageBook)


def _workspace(book, device):
    size = N.lib.vmb_page_book_workspace_bytes(ctypes.byref(book))
    return torch.empty(size, dtype=torch.uint8, device=device), size


def reserve_pages(page_table, lengths, counts, free_pages, num_free, *, page_size, total, failed=None):
    """
    Room for counts[b] more tokens of every sequence: takes pages for them, in place, and returns their slots.

    Args:
        page_table: (B, width) int32; row b names the pages of sequence b, the first ceil(lengths[b] / page_size) of which
            are in use. The entries of new pages are written.
        lengths: (B,) int32, the tokens that each sequence holds; counts are added
        counts: (B,) int32, not negative
        free_pages: (num_pages,) int32, a stack of which the first num_free pages are free
        num_free: (1,) int32; the pages taken, from the stack's end, are subtracted
        page_size: slots of a page
        total: rows of the packed new tokens, at least the sum of counts
        failed: (1,) int32, into which the bit of what went wrong is added: 1 not enough free pages, 2 a sequence would be
            longer than its row of the table holds, 4 more tokens than `total`, or a negative length or count
    Returns:
        slots: (total,) int32, page * page_size + slot of every new token, sequence after sequence, as
            :func:`append_pages` takes them; -1 in the rows past the last one
    A call that cannot be done changes nothing but `failed`, and its slots are -1. Nothing waits for the device. Pages have
    one owner here: forks and their shared pages are :class:`PagedKVCache`'s.
    """
    book, device, batch, _ = _book(page_table, lengths, counts, free_pages, num_free, page_size, failed)
    total = operator.index(total)
    assert 0 <= total < 2 ** 31, "total must be a number of rows"
    counts = counts.contiguous()
    slots = torch.empty(total, dtype=torch.int32, device=device)
    ws, size = (None, 0) if batch <= 1024 and total <= 4096 else _workspace(book, device)
    N.launch("vmb_reserve_pages", N.lib.vmb_reserve_pages, device, ctypes.byref(book), counts.data_ptr(), slots.data_ptr(), total,
             N.ptr(ws), size)
    return slots


def truncate_pages(page_table, lengths, keep, free_pages, num_free, *, page_size, failed=None):
    """
    Cuts every sequence back to its first keep[b] tokens, in place (0 gives it up, its length or more leaves it as it is), and
    returns the pages beyond them to the stack, so that it undoes a :func:`reserve_pages` of as many tokens. Entries of the table
    beyond a length are left as they are.

    Args: as of :func:`reserve_pages`, with keep (B,) int32, negative for 0. failed: 2 a length is more than its row of the
        table holds, 4 a negative length, 8 more pages than free_pages has room for, which cannot be unless one was returned
        twice. Such a call changes nothing else.
    """
    book, device, batch, width = _book(page_table, lengths, keep, free_pages, num_free, page_size, failed)
    if not batch:
        return
    keep = keep.contiguous()
    ws, size = (None, 0) if batch <= 1024 and batch * width <= 65536 else _workspace(book, device)
    N.launch("vmb_truncate_pages", N.lib.vmb_truncate_pages, device, ctypes.byref(book), keep.data_ptr(), N.ptr(ws), size)


class PageTables:
    """
    The book of a paged cache on the GPU: tables and lengths of `batch` sequences, empty at first, and the stack of free pages.

    Args:
        num_pages, page_size: of the pools
        batch: sequences
        width: entries of a table row: a sequence holds at most width * page_size tokens
        pages: the pages that are free (default: all); low ones are taken first
        device: of the tensors

    `table` and `lengths` are what :func:`paged_attention` takes. :meth:`PagedKVCache.page_tables` makes one over a cache's pools.
    """

    def __init__(self, num_pages, page_size, batch, width, *, pages=None, device="cuda"):
        assert num_pages >= 1 and page_size >= 1 and batch >= 1 and width >= 1, "sizes must be positive"
        assert num_pages * page_size < 2 ** 31, "slots are 32-bit: fewer pages or smaller ones"
        pages = list(range(num_pages)) if pages is None else sorted(pages)
        assert len(set(pages)) == len(pages) and all(0 <= p < num_pages for p in pages), "pages must be different ones of the pool"
        self.page_size = page_size
        self.table = torch.zeros((batch, width), dtype=torch.int32, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        stack = torch.zeros(num_pages, dtype=torch.int32)
        stack[:len(pages)] = torch.tensor(pages[::-1], dtype=torch.int32)
        self.free_pages = stack.to(device)
        self.num_free = torch.tensor([len(pages)], dtype=torch.int32).to(device)
        self.failed = torch.zeros(1, dtype=torch.int32, device=device)

    def reserve(self, counts, total):
        """Slots of counts[b] more tokens of every sequence: :func:`reserve_pages`."""
        return reserve_pages(self.table, self.lengths, counts, self.free_pages, self.num_free, page_size=self.page_size,
                             total=total, failed=self.failed)

    def truncate(self, keep):
        """Cuts the sequences back to keep[b] tokens: :func:`truncate_pages`."""
        truncate_pages(self.table, self.lengths, keep, self.free_pages, self.num_free, page_size=self.page_size, failed=self.failed)

    def check(self):
        """Raises MemoryError if a call since the last check could not be done. Waits for the device."""
        bits = int(self.failed)
        if bits:
            self.failed.zero_()
            raise MemoryError("page tables: " + ", ".join(text for bit, text in _FAILURES.items() if bits & bit))
