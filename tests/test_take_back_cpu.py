"""Pages that a PageTables holds go back to the cache's book whatever its earlier calls could not do, without a GPU: the
truncation is a plain one over the same tensors."""
import pytest
import torch

from vmonarch_b200 import PagedKVCache, PageTables


def plain_truncate(self, keep):
    """truncate_pages' rule: a call that cannot be done sets its bit and changes nothing else."""
    width, ps = self.table.size(1), self.page_size
    if (self.lengths < 0).any() or (self.lengths > width * ps).any():
        self.failed |= 4 if (self.lengths < 0).any() else 2
        return
    for b in reversed(range(len(self.lengths))):
        for i in reversed(range(-(-int(keep[b]) // ps), -(-int(self.lengths[b]) // ps))):
            self.free_pages[int(self.num_free)] = self.table[b, i]
            self.num_free += 1
        self.lengths[b] = keep[b]


@pytest.fixture
def lent(monkeypatch):
    monkeypatch.setattr(PageTables, "truncate", plain_truncate)
    cache = PagedKVCache(10, 4, 1, 16, device="cpu")
    seq = cache.add()
    cache.reserve([seq], [9])
    tables = cache.page_tables(2, 3, 4)
    # as a reserve of nine tokens leaves them
    tables.table[0] = torch.tensor([3, 4, 5])
    tables.lengths[0] = 9
    tables.num_free.fill_(1)
    return cache, tables


def everything_free(cache):
    assert cache.num_free == 7 and sorted(cache._free) == list(range(3, 10))
    assert cache.compact() == 3


@pytest.mark.parametrize("bits", [0, 1, 2, 4, 7])
def test_after_calls_that_could_not_be_done(lent, bits):
    cache, tables = lent
    tables.failed.fill_(bits)
    cache.take_back(tables)
    assert not tables.num_free.any() and not tables.lengths.any()
    with pytest.raises(AssertionError, match="taken back"):
        cache.take_back(tables)
    everything_free(cache)


@pytest.mark.parametrize("length", [-1, 13])
def test_a_truncation_that_cannot_be_done_leaves_the_loan(lent, length):
    cache, tables = lent
    tables.lengths[1] = length
    for _ in range(2):
        with pytest.raises(MemoryError):
            cache.take_back(tables)
        assert cache.num_free == 3 and tables.num_free.tolist() == [1] and tables.lengths.tolist() == [9, length]
        with pytest.raises(AssertionError, match="moved"):
            cache.compact()
    tables.lengths[1] = 0
    cache.take_back(tables)
    everything_free(cache)
