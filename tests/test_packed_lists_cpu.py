"""The device copies of a PackedSequences' work lists, which the kernels get by their addresses: whoever makes them first
and on whatever thread, the lists that calls name are the ones that are kept."""
import threading

import pytest
import torch

from vmonarch_b200 import PackedSequences
from vmonarch_b200 import _native as N
import vmonarch_b200.packed as packed

KEYS = [(False, True, 0.125, torch.bfloat16, 4, 2, 64), (True, True, 0.125, torch.bfloat16, 4, 2, 64)]


def held_spans(seqs):
    """(first byte, end) of every list that the object keeps."""
    lists = [hit[1] for hit in seqs._cache.values() if isinstance(hit[0], N.PackedList)]
    return [(t.data_ptr(), t.data_ptr() + t.nbytes) for t in lists]


def named_lists(template):
    a = N.PackedArgs.from_buffer_copy(template)
    return [x for x in (a.units, a.q_units, a.kv_units) if x.n_units]


def together(n, fn):
    """fn() of n threads that meet before it; their results."""
    gate, out, threads = threading.Barrier(n), [None] * n, []

    def run(i):
        gate.wait()
        out[i] = fn()
    for i in range(n):
        threads.append(threading.Thread(target=run, args=(i,)))
        threads[-1].start()
    for t in threads:
        t.join()
    return out


@pytest.fixture
def slow_copies(monkeypatch):
    """The copy to the device lets another thread in, as a copy that gives up the interpreter does: up to two threads
    that make the same list are both in here before either goes on."""
    met = threading.Barrier(2)
    plain = torch.from_numpy

    def from_numpy(a):
        try:
            met.wait(0.2)
        except threading.BrokenBarrierError:
            met.reset()
        return plain(a)
    monkeypatch.setattr(packed.torch, "from_numpy", from_numpy)


@pytest.mark.parametrize("key", KEYS)
def test_calls_of_two_threads_name_the_kept_lists(slow_copies, key):
    for _ in range(3):
        seqs = PackedSequences([300, 5, 1000], device="cpu")
        for entry in (*together(2, lambda: seqs._template(key)), seqs._template(key)):
            lists = named_lists(entry[0])
            assert len(lists) == (2 if key[0] else 1)
            for x in lists:
                assert any(a <= x.units and x.units + 48 * x.n_units <= b for a, b in held_spans(seqs))


def test_starts_of_two_threads_are_the_kept_ones(slow_copies):
    seqs = PackedSequences([300, 5, 1000], device="cpu")
    a, b = together(2, lambda: seqs._starts().data_ptr())
    assert a == b == seqs._starts().data_ptr()


@pytest.mark.parametrize("key", KEYS)
def test_a_template_keeps_the_lists_it_names(key):
    """Even if the object's own entry for a list went away, the arguments that name it would still hold it."""
    seqs = PackedSequences([300, 5, 1000], device="cpu")
    entry = seqs._template(key)
    spans = [(t.data_ptr(), t.data_ptr() + t.nbytes) for t in entry[2]]
    for x in named_lists(entry[0]):
        assert (x.units, x.units + 48 * x.n_units + 8 * x.n_joins) in spans
