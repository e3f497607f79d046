"""The book of a paged cache on the host, with the page copies replaced by torch indexing, and the
refusals of the paged calls."""
import random

import pytest
import torch

import vmonarch_b200.paged as paged
from vmonarch_b200 import PagedKVCache, append_pages, copy_pages, paged_attention


@pytest.fixture(autouse=True)
def host_moves(monkeypatch):
    def copy(k, v, src, dst):
        assert not set(src.tolist()) & set(dst.tolist()) and len(set(dst.tolist())) == len(dst)
        k[dst.long()], v[dst.long()] = k[src.long()], v[src.long()]

    def append(k, v, kp, vp, slots):
        assert len(set(slots.tolist())) == len(slots)
        page, at = slots.long() // kp.size(2), slots.long() % kp.size(2)
        kp[page, :, at], vp[page, :, at] = k, v

    monkeypatch.setattr(paged, "copy_pages", copy)
    monkeypatch.setattr(paged, "append_pages", append)


def contents(cache, layer, seq):
    """The keys of a sequence, in order."""
    table, lengths = cache.tables([seq])
    n = int(lengths[0])
    at = torch.arange(n)
    return cache.k[layer, table[0].long()[at // cache.page_size], :, at % cache.page_size] if n else \
        torch.zeros(0, cache.k.size(2), cache.k.size(4), dtype=cache.k.dtype)


@pytest.mark.parametrize("page_size", [1, 3, 8])
def test_random_lives(page_size):
    """Add, append, fork, free and compact at random: every sequence keeps its own tokens."""
    rng = random.Random(page_size)
    cache = PagedKVCache(40, page_size, 1, 8, layers=2, device="cpu")
    truth, stamp = {}, 0
    for _ in range(400):
        act = rng.random()
        if act < 0.2 or not truth:
            truth[cache.add()] = []
        elif act < 0.65:
            seqs = rng.sample(sorted(truth), rng.randint(1, len(truth)))
            counts = [rng.randint(0, 2 * page_size) for _ in seqs]
            before = cache.num_free, {s: cache.pages(s) for s in truth}
            try:
                slots = cache.reserve(seqs, counts)
            except MemoryError:
                assert (cache.num_free, {s: cache.pages(s) for s in truth}) == before
                continue
            vals = torch.arange(stamp, stamp + sum(counts)) % 251
            stamp += sum(counts)
            rows = vals.to(cache.k.dtype)[:, None, None].expand(-1, 1, 8)
            for layer in range(2):
                cache.write(layer, rows + layer, rows, slots)
            pos = 0
            for s, c in zip(seqs, counts):
                truth[s] += vals[pos:pos + c].tolist()
                pos += c
        elif act < 0.8:
            s = rng.choice(sorted(truth))
            truth[cache.fork(s)] = list(truth[s])
        elif act < 0.95:
            s = rng.choice(sorted(truth))
            cache.free(s)
            del truth[s]
        else:
            used = cache.compact()
            assert used == cache.num_pages - cache.num_free
            assert all(p < used for s in truth for p in cache.pages(s))
        held = {p for s in truth for p in cache.pages(s)}
        assert len(held) == cache.num_pages - cache.num_free
        for s, want in truth.items():
            assert cache.length(s) == len(want) and len(cache.pages(s)) == -(-len(want) // page_size)
            for layer in range(2):
                got = contents(cache, layer, s)[:, 0, 0].float()
                want_l = (torch.tensor(want, dtype=torch.float32).to(cache.k.dtype) + layer).float()
                assert torch.equal(got, want_l)


def test_forks_write_apart():
    cache = PagedKVCache(8, 4, 1, 8, device="cpu")
    a = cache.add()
    cache.reserve([a], [6])
    b = cache.fork(a)
    assert cache.pages(a) == cache.pages(b) and cache.num_free == 6
    cache.reserve([a, b], [1, 1])  # one of them leaves the shared half-full page, the other keeps it
    assert cache.pages(a)[0] == cache.pages(b)[0] and cache.pages(a)[1] != cache.pages(b)[1]
    assert cache.num_free == 5
    cache.free(a)
    cache.free(b)
    assert cache.num_free == 8


def test_cache_refusals():
    for bad in (dict(num_pages=0), dict(page_size=0), dict(kv_heads=0), dict(head_dim=20), dict(head_dim=136),
                dict(layers=0), dict(dtype=torch.float32), dict(num_pages=2 ** 28)):
        with pytest.raises(AssertionError):
            PagedKVCache(**{**dict(num_pages=4, page_size=8, kv_heads=1, head_dim=8, device="cpu"), **bad})
    cache = PagedKVCache(4, 8, 1, 8, device="cpu")
    s = cache.add()
    with pytest.raises(AssertionError):
        cache.reserve([s, s], [1, 1])
    with pytest.raises(AssertionError):
        cache.reserve([s], [-1])
    with pytest.raises(MemoryError):
        cache.reserve([s], [33])


def test_calls_refuse_host_tensors():
    k = torch.zeros(4, 1, 8, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(AssertionError, match="CUDA"):
        paged_attention(torch.zeros(1, 2, 64, dtype=torch.bfloat16), k, k, i[None], i)
    with pytest.raises(AssertionError, match="CUDA"):
        append_pages(k[0].transpose(0, 1), k[0].transpose(0, 1), k, k, i)
    with pytest.raises(AssertionError, match="CUDA"):
        copy_pages(k, k, i, i)
