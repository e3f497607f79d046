"""The book of a paged cache on the GPU: calls at the ends of what it allows."""
import pytest
import torch

from vmonarch_b200 import PagedKVCache, reserve_pages, truncate_pages
from vmonarch_b200 import _native as N

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_taken_back_after_a_reserve_that_failed():
    """Too few pages, a sequence too long for its row, too few rows: none of it was done, and every page is free once afterwards."""
    cache = PagedKVCache(20, 4, 1, 16, device="cuda")
    kept = cache.add()
    cache.reserve([kept], [10])
    tables = cache.page_tables(3, 6, 9)
    tables.reserve(ints([5, 0, 9]), 14)
    for counts, total in (([12, 12, 13], 37), ([20, 0, 0], 20), ([1, 1, 1], 2)):
        assert (tables.reserve(ints(counts), total) == -1).all()
    assert int(tables.failed) == 7 and tables.lengths.tolist() == [5, 0, 9]
    cache.take_back(tables)
    assert cache.num_free == 17 and sorted(cache._free + cache.pages(kept)) == list(range(20))
    assert not tables.num_free.any() and not tables.lengths.any()
    with pytest.raises(AssertionError, match="taken back"):
        cache.take_back(tables)
    assert cache.compact() == 3


def test_a_loan_stays_where_its_truncation_fails():
    cache = PagedKVCache(20, 4, 1, 16, device="cuda")
    tables = cache.page_tables(3, 6, 9)
    tables.reserve(ints([5, 0, 9]), 14)
    tables.lengths[1] = 25  # what no call of its own leaves
    for _ in range(2):
        with pytest.raises(MemoryError, match="longer"):
            cache.take_back(tables)
        assert cache.num_free == 11 and tables.lengths.tolist() == [5, 25, 9] and tables.num_free.tolist() == [4]
        with pytest.raises(AssertionError, match="moved"):
            cache.compact()
    tables.lengths[1] = 0
    cache.take_back(tables)
    assert sorted(cache._free) == list(range(20)) and cache.compact() == 0


@pytest.mark.parametrize("batch", [3, 1024, 1025, 2000])
def test_tables_without_entries(batch):
    """Rows of no entries: nothing is held, so there is nothing to return, and no token can be taken."""
    table = torch.empty(batch, 0, dtype=torch.int32, device="cuda")
    lengths, free, num, failed = ints([0] * batch), ints([3, 2, 1, 0]), ints([4]), ints([0])
    book = dict(page_size=4, failed=failed)
    before = N.lib.vmb_kernel_launches()
    truncate_pages(table, lengths, ints([0] * batch), free, num, **book)
    truncate_pages(table, lengths, ints([5, -1] * (batch // 2) + [0] * (batch % 2)), free, num, **book)
    assert N.lib.vmb_kernel_launches() == before + 2
    assert reserve_pages(table, lengths, ints([0] * batch), free, num, total=6, **book).tolist() == [-1] * 6
    assert not failed.any()
    assert (reserve_pages(table, lengths, ints([1] * batch), free, num, total=batch, **book) == -1).all() and int(failed) & 2
    assert not lengths.any() and num.tolist() == [4] and free.tolist() == [3, 2, 1, 0]
