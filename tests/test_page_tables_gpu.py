"""Page tables and slot maps kept on the GPU: equal, number for number, to a book kept in Python."""
import random

import pytest
import torch

from vmonarch_b200 import PagedKVCache, PageTables, append_pages, paged_attention, reserve_pages, truncate_pages
from window_reference import window_reference

pytestmark = pytest.mark.gpu


class Book:
    """The same rules, one sequence and page at a time."""

    def __init__(self, pages, page_size, batch, width):
        self.free, self.ps, self.width = sorted(pages, reverse=True), page_size, width
        self.table, self.lengths = [[] for _ in range(batch)], [0] * batch

    def reserve(self, counts, total):
        need = sum(-(-(n + c) // self.ps) - -(-n // self.ps) for n, c in zip(self.lengths, counts))
        bad = (need > len(self.free)) | 2 * any(n + c > self.width * self.ps for n, c in zip(self.lengths, counts)) | 4 * (sum(counts) > total)
        if bad:
            return [-1] * total, bad
        slots = []
        for b, c in enumerate(counts):
            for _ in range(c):
                if self.lengths[b] % self.ps == 0:
                    self.table[b].append(self.free.pop())
                slots.append(self.table[b][-1] * self.ps + self.lengths[b] % self.ps)
                self.lengths[b] += 1
        return slots + [-1] * (total - len(slots)), 0

    def truncate(self, keep):
        back = []
        for b, k in enumerate(keep):
            self.lengths[b] = max(0, min(self.lengths[b], k))
            used = -(-self.lengths[b] // self.ps)
            back += self.table[b][used:]
            del self.table[b][used:]
        self.free += back[::-1]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def same(tables, book):
    assert tables.lengths.tolist() == book.lengths and int(tables.num_free) == len(book.free)
    assert tables.free_pages[:len(book.free)].tolist() == book.free
    for row, want in zip(tables.table.tolist(), book.table):
        assert row[:len(want)] == want


@pytest.mark.parametrize("batch, width, page, pool, most", [
    (1, 1, 1, 1, 1), (3, 5, 4, 12, 9), (64, 40, 16, 700, 70), (300, 9, 7, 1500, 30), (1024, 30, 8, 9000, 40), (1025, 6, 16, 3000, 30),
    (3000, 50, 3, 50000, 60), (5, 20000, 2, 60000, 20000), (2, 3000, 16, 5000, 40000),
])
def test_random_lives(batch, width, page, pool, most):
    """Counts and cuts at random, some of which cannot be done: one block's calls and those with a second kernel."""
    rng = random.Random(batch)
    mine = rng.sample(range(pool), max(1, pool * 9 // 10))
    tables, book = PageTables(pool, page, batch, width, pages=mine), Book(mine, page, batch, width)
    for turn in range(30):
        if rng.random() < 0.6:
            share = rng.random()
            counts = [rng.randint(0, most) if rng.random() < share else 0 for _ in range(batch)]
            room = [width * page - n for n in book.lengths]
            if rng.random() < 0.8:
                counts = [min(c, r) for c, r in zip(counts, room)]
            total = sum(counts) + rng.choice([0, 0, 1, 300]) - (rng.random() < 0.1 and sum(counts) > 0)
            want, bad = book.reserve(counts, total)
            assert tables.reserve(ints(counts), total).tolist() == want
            if bad:
                with pytest.raises(MemoryError):
                    tables.check()
        else:
            low = rng.choice([-1, 0, 0.5, 0.9])
            keep = [int(n * (1 if rng.random() < 0.3 else rng.uniform(max(low, 0), 1))) if low >= 0 else rng.randint(-2, 2) for n in book.lengths]
            book.truncate(keep)
            tables.truncate(ints(keep))
        same(tables, book)
        tables.check()


@pytest.mark.parametrize("batch, page", [(70, 16), (1100, 5)])
def test_truncate_undoes_reserve(batch, page):
    rng = random.Random(1)
    tables = PageTables(20000, page, batch, 30)
    first = [rng.randint(0, 10 * page) for _ in range(batch)]
    tables.reserve(ints(first), sum(first))
    before = [t.clone() for t in (tables.lengths, tables.free_pages, tables.num_free)]
    more = [rng.randint(0, 10 * page) for _ in range(batch)]
    slots = tables.reserve(ints(more), sum(more))
    tables.truncate(ints(first))
    for t, b in zip((tables.lengths, tables.free_pages, tables.num_free), before):
        assert torch.equal(t, b)
    assert torch.equal(tables.reserve(ints(more), sum(more)), slots)
    tables.check()


@pytest.mark.parametrize("batch, width, page, most", [
    (1024, 70, 16, 60), (1024, 257, 16, 64), (1024, 257, 16, 70), (3, 40000, 1, 17000), (64, 1100, 7, 1024), (1, 70000, 1, 65536), (2, 33, 64, 2049),
])
def test_captured_exchanges(batch, width, page, most):
    """Sequences given up or cut back and others admitted, captured together: one block's, a cluster's and two kernels' calls."""
    rng = random.Random(width)
    pool = batch * width
    mine = rng.sample(range(pool), pool - 5)
    tables, book = PageTables(pool, page, batch, width, pages=mine), Book(mine, page, batch, width)
    keep, counts, total = ints([0] * batch), ints([0] * batch), batch * most
    slots = [None]

    def step():
        tables.truncate(keep)
        slots[0] = tables.reserve(counts, total)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(6):
        left = [0 if rng.random() < 0.7 else rng.randint(0, n) for n in book.lengths]
        if turn == 3:
            left = list(book.lengths)
        more = [min(rng.choice([0, 1, rng.randint(0, most), most]), width * page - n) for n in left]
        if turn == 4:
            more[rng.randrange(batch)] = width * page + 1  # cannot be done: slots of -1, the book as the cut left it
        keep.copy_(ints(left))
        counts.copy_(ints(more))
        book.truncate(left)
        want, bad = book.reserve(more, total)
        graph.replay()
        assert torch.equal(slots[0], ints(want))
        assert (int(tables.failed) != 0) == bool(bad)
        tables.failed.zero_()
        same(tables, book)


def test_what_cannot_be_done_changes_nothing():
    tables = PageTables(10, 4, 3, 3)
    tables.reserve(ints([4, 5, 0]), 9)
    state = [t.clone() for t in (tables.table, tables.lengths, tables.free_pages, tables.num_free)]
    for counts, total, bit in (([0, 8, 0], 8, 2), ([12, 0, 0], 12, 2), ([8, 7, 12], 26, 4), ([1, -1, 0], 5, 4), ([2 ** 31 - 1] * 3, 5, 7)):
        slots = tables.reserve(ints(counts), total)
        assert (slots == -1).all() and len(slots) == total
        assert int(tables.failed) & bit and int(tables.failed) & ~7 == 0
        tables.failed.zero_()
        for t, s in zip((tables.table, tables.lengths, tables.free_pages, tables.num_free), state):
            assert torch.equal(t, s)
    tables.num_free.fill_(9)  # as after returning pages twice: no room for the three that are in use
    tables.truncate(ints([0, 0, 0]))
    with pytest.raises(MemoryError, match="returned"):
        tables.check()
    assert tables.lengths.tolist() == [4, 5, 0] and int(tables.num_free) == 9
    tables.num_free.copy_(state[3])
    tables.lengths[0] = 400
    for call in (lambda: tables.reserve(ints([0, 0, 1]), 1), lambda: tables.truncate(ints([0, 0, 0]))):
        call()
        with pytest.raises(MemoryError, match="longer"):
            tables.check()
    tables.lengths[0] = -4
    for call in (lambda: tables.reserve(ints([0, 0, 1]), 1), lambda: tables.truncate(ints([0, 0, 0]))):
        call()
        with pytest.raises(MemoryError, match="negative"):
            tables.check()


def test_views_and_empty_calls():
    """A table that is part of a wider one, counts that are a column of a matrix, no rows, no sequences."""
    wide = torch.full((3, 10), -5, dtype=torch.int32, device="cuda")
    lengths, free, num = ints([0, 0, 0]), ints([3, 2, 1, 0]), ints([4])
    counts = ints([[5, 9], [0, 9], [3, 9]])[:, 0]
    slots = reserve_pages(wide[:, 2:6], lengths, counts, free, num, page_size=4, total=10)
    assert slots.tolist() == [0, 1, 2, 3, 4, 8, 9, 10, -1, -1]
    assert wide.tolist() == [[-5, -5, 0, 1] + [-5] * 6, [-5] * 10, [-5, -5, 2] + [-5] * 7]
    assert reserve_pages(wide[:, 2:6], lengths, ints([0, 0, 0]), free, num, page_size=4, total=0).tolist() == []
    truncate_pages(wide[:, 2:6], lengths, ints([[4, 1], [0, 1], [9, 1]])[:, 0], free, num, page_size=4)
    assert lengths.tolist() == [4, 0, 3] and num.tolist() == [2] and free.tolist()[:2] == [3, 1]
    none = torch.empty(0, 4, dtype=torch.int32, device="cuda")
    assert reserve_pages(none, ints([]), ints([]), free, num, page_size=4, total=3).tolist() == [-1] * 3
    truncate_pages(none, ints([]), ints([]), free, num, page_size=4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("window, sinks", [(None, 0), (20, 3)])
def test_captured_decoding(window, sinks, dtype):
    """Steps that take pages, write their token and attend, captured once: replayed, every step sees what it should, beside a
    sequence of the host's book, and after a cut of drafted tokens."""
    h, hk, d, batch, page = 4, 2, 64, 3, 8
    cache = PagedKVCache(60, page, hk, d, layers=1, dtype=dtype)
    kept = cache.add()
    cache.reserve([kept], [30])  # the host's own pages
    tables = cache.page_tables(batch, 10)
    assert cache.num_free == 0 and int(tables.num_free) == 56
    with pytest.raises(AssertionError):
        cache.compact()
    g = torch.Generator(device="cuda").manual_seed(0)
    q = torch.zeros(batch, h, d, device="cuda", dtype=torch.bfloat16)
    k, v = (torch.zeros(batch, hk, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    counts, keep = ints([0, 0, 0]), ints([0, 0, 0])

    def step():
        tables.truncate(keep)
        slots = tables.reserve(counts, batch + 1)
        cache.write(0, k, v, slots[:batch])
        return cache.attend(0, q, tables.table, tables.lengths, window=window, sinks=sinks)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    ks, vs = [[] for _ in range(batch)], [[] for _ in range(batch)]
    for t in range(50):
        q.normal_(generator=g)
        k.normal_(generator=g)
        v.normal_(generator=g)
        keep.copy_(ints([len(ks[0]), max(0, len(ks[1]) - (t % 7 == 0) * 2), len(ks[2]) if t != 31 else 0]))
        counts.copy_(ints([1, 1, 1]))
        for b, n in enumerate(keep.tolist()):
            del ks[b][n:], vs[b][n:]
            ks[b].append(k[b].double())
            vs[b].append(v[b].double())
        graph.replay()
        lens = [len(x) for x in ks]
        assert tables.lengths.tolist() == lens
        kk, vv = torch.stack(sum(ks, [])), torch.stack(sum(vs, []))
        if dtype == torch.float8_e4m3fn:  # what the cache holds; test_cache8_gpu.py says how far that may be off
            held = []
            for pool, s in ((cache.k[0], cache.k_scale[0]), (cache.v[0], cache.v_scale[0])):
                values = pool.view(torch.uint8).view(dtype).double() * s[..., None, None].double()
                held.append(torch.cat([values[tables.table[b].long()].transpose(1, 2).reshape(-1, hk, d)[:n] for b, n in enumerate(lens)]))
            for a, b in zip((kk, vv), held):
                assert (a - b).abs().max() <= 0.07 * a.abs().max()
            kk, vv = held
        ref = window_reference(q.double(), kk, vv, [1] * batch, lens, window or 10 ** 9, sinks, d ** -0.5)[0]
        for b in range(batch):
            assert (out[b].double() - ref[b]).norm() <= 2 * 2.0 ** -8 * ref[b].norm()
    tables.check()
    # every page belongs to one owner
    pages = [p for b, n in enumerate(lens) for p in tables.table[b, :-(-n // page)].tolist()]
    pages += tables.free_pages[:int(tables.num_free)].tolist() + cache.pages(kept)
    assert sorted(pages) == list(range(60))
    cache.take_back(tables)
    assert cache.num_free == 56 and int(tables.num_free) == 0 and cache.compact() == 4
    cache.reserve([cache.add()], [56 * page])
    with pytest.raises(AssertionError):
        cache.take_back(tables)


def test_other_streams_and_devices():
    tables = PageTables(100, 4, 8, 10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = tables.reserve(ints([3] * 8), 24)
    side.synchronize()
    assert a.tolist() == [4 * b + i for b in range(8) for i in range(3)]


def test_slots_of_a_whole_pool():
    """Every slot of a pool is given once; a batch of long sequences writes through them."""
    page, pool, batch = 16, 9000, 40
    tables = PageTables(pool, page, batch, pool // batch)
    counts = [pool // batch * page] * batch
    slots = tables.reserve(ints(counts), sum(counts))
    assert torch.equal(slots.sort()[0], torch.arange(pool * page, dtype=torch.int32, device="cuda")) and int(tables.num_free) == 0
    kp = torch.zeros(pool, 1, page, 8, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    rows = torch.randn(len(slots), 1, 8, device="cuda").to(torch.bfloat16)
    append_pages(rows, rows, kp, vp, slots)
    o = paged_attention(rows[:batch], kp, vp, tables.table, torch.ones_like(tables.lengths))
    assert torch.equal(o, rows[::counts[0]])
    tables.check()


def test_refusals():
    t = PageTables(10, 4, 3, 3)
    ok = dict(page_table=t.table, lengths=t.lengths, counts=ints([0] * 3), free_pages=t.free_pages, num_free=t.num_free, page_size=4, total=3)
    for bad in (dict(page_table=t.table.long()), dict(lengths=t.lengths[:2]), dict(counts=ints([0] * 2)), dict(counts=ints([0] * 3).long()),
                dict(lengths=t.lengths.cpu()), dict(num_free=t.free_pages), dict(page_size=0), dict(total=-1), dict(total=2 ** 31),
                dict(page_table=t.table.t()), dict(lengths=ints([0] * 6)[::2]), dict(free_pages=ints([0] * 6)[::2]),
                dict(page_size=2 ** 30), dict(free_pages=t.free_pages[:0]), dict(failed=ints([0, 0]))):
        with pytest.raises(AssertionError):
            reserve_pages(**{**ok, **bad})
