"""Calls on a stream other than the one on which a PackedSequences' device lists were allocated: the allocator is told,
so that it does not give the lists' memory to others before that stream is done with them."""
from types import SimpleNamespace

import pytest
import torch

from vmonarch_b200 import PackedSequences
from vmonarch_b200 import _native as N
import vmonarch_b200.gated_norm as gated_norm
import vmonarch_b200.packed as packed


class Listed(torch.Tensor):
    """A tensor that notes on which streams it was recorded."""

    def record_stream(self, stream):
        self.__dict__.setdefault("recorded", []).append(stream)


@pytest.fixture
def streams(monkeypatch):
    """A current stream that a test sets (`streams.now`), and no launches."""
    s = SimpleNamespace(now=7)
    monkeypatch.setattr(PackedSequences, "_stream", lambda seqs: s.now, raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: s.now)
    monkeypatch.setattr(N, "launch", lambda *a: None)
    plain = torch.from_numpy
    monkeypatch.setattr(packed.torch, "from_numpy", lambda a: plain(a.copy()).as_subclass(Listed))
    return s


def recorded(t):
    return t.__dict__.get("recorded", [])


def lists(seqs):
    """Every kept list by its kind, and the sequences' starts."""
    return {k[0]: v[1] for k, v in seqs._cache.items() if isinstance(k, tuple) and len(k) == 4} | \
        {k: v for k, v in seqs._cache.items() if k == "starts"}


def attention(seqs, backward):
    q, k, v = (torch.zeros(seqs.total_q, 2, 64, dtype=torch.bfloat16) for _ in range(3))
    key = (False, True, 0.125, q.dtype, 2, 2, 64)
    aux = torch.zeros(seqs.total_q * 2 * (128 + 4), dtype=torch.uint8)
    o = packed._forward(q, k, v, seqs, key, q.device, aux=aux)[3]
    if backward:
        packed._PackedAttention.backward(SimpleNamespace(saved_tensors=(q, k, v, o, aux), meta=(seqs, key)), o)


def norm(seqs, backward):
    x, w = torch.zeros(seqs.total_q, 64, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    sizes = (seqs.total_q, 64, seqs.num_sequences, N.VMB_DTYPE_BF16, N.VMB_DTYPE_BF16, False, 1e-6)
    params, stats = (None, None, None, w, None), torch.zeros(3 * seqs.total_q)
    gated_norm._forward(x, x, params, seqs, sizes, stats)
    if backward:
        gated_norm._GatedNorm.backward(SimpleNamespace(saved_tensors=(x, x, stats, *params), meta=(seqs, sizes),
                                                       needs_input_grad=(True, True, False, False) + (False,) * 5), x, x)


@pytest.mark.parametrize("call, kinds", [(attention, {"fwd", "dq", "kv"}), (norm, {"starts"})])
def test_lists_are_recorded_on_other_streams_alone(streams, call, kinds):
    seqs = PackedSequences([30, 5], device="cpu")
    call(seqs, True)
    assert set(lists(seqs)) == kinds and not any(map(recorded, lists(seqs).values()))
    streams.now = 9
    call(seqs, True)
    for name, t in lists(seqs).items():
        assert 9 in recorded(t), name
    before = {n: len(recorded(t)) for n, t in lists(seqs).items()}
    streams.now = 7
    call(seqs, True)
    assert before == {n: len(recorded(t)) for n, t in lists(seqs).items()}


def test_lists_made_on_several_streams(streams):
    """A forward on one stream, its backward on a second, both again on a third."""
    seqs = PackedSequences([30, 5], device="cpu")
    attention(seqs, False)
    streams.now = 9
    attention(seqs, True)
    assert 9 in recorded(lists(seqs)["fwd"])
    streams.now = 7
    attention(seqs, True)
    assert 7 in recorded(lists(seqs)["dq"]) and 7 in recorded(lists(seqs)["kv"])
    streams.now = 11
    attention(seqs, True)
    assert all(11 in recorded(t) for t in lists(seqs).values())
