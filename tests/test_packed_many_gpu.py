"""More work items than SMs: blocks go on to items that other blocks were to start (their rings and barriers run on from
item to item), several chunks of heads follow one another, and units of every kind meet.

An item's arithmetic does not depend on its neighbours, so outputs, statistics and dQ of a batch have the bits that each
sequence has alone, where every item has an SM of its own (no unit here is long enough to be cut in these). All outputs
are held to the definition in 64 bits with the bounds that test_packed_gpu.py derives."""
import random

import pytest
import torch

from packed_reference import packed_reference
from test_packed_gpu import U, grads, make, rel
from vmonarch_b200 import PackedSequences, packed_attention

pytestmark = pytest.mark.gpu
SMS = 148


def check(ql, kl, causal, h, hk, d, dtype):
    q, k, v, do = make(ql, kl, h, hk, d, dtype)
    seqs = PackedSequences(ql, kl)
    got = grads(lambda *x: packed_attention(*x, seqs, causal=causal), (q, k, v), do)
    with torch.no_grad():
        o, lse = packed_attention(q, k, v, seqs, causal=causal, return_lse=True)
    assert torch.equal(o, got[0])
    q0 = k0 = 0
    for nq, nk in zip(ql, kl):
        if nq:
            mine = [q[q0:q0 + nq], k[k0:k0 + nk], v[k0:k0 + nk]]
            one = PackedSequences([nq], [nk])
            alone = grads(lambda *x: packed_attention(*x, one, causal=causal), mine, do[q0:q0 + nq])
            with torch.no_grad():
                one_lse = packed_attention(*mine, one, causal=causal, return_lse=True)[1]
            assert one._list("fwd", causal, h, h // hk).n_units * h <= SMS and one._list("dq", causal, h, h // hk).n_parts == 0
            where = f"{nq} queries, {nk} keys at row {q0}"
            assert torch.equal(got[0][q0:q0 + nq], alone[0]), where
            assert torch.equal(lse[:, q0:q0 + nq], one_lse), where
            assert torch.equal(got[1][q0:q0 + nq], alone[1]), where
        q0, k0 = q0 + nq, k0 + nk
    want = grads(lambda *x: packed_reference(*x, ql, kl, causal, d ** -0.5)[0], [t.double() for t in (q, k, v)], do)
    for x, ref, bound in zip(got, want, (2, 4, 4, 4)):
        assert rel(x, ref) <= bound * U[dtype]
    return seqs._list("fwd", causal, h, h // hk).n_units * h


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [128, 64, 40])
@pytest.mark.parametrize("causal", [True, False])
def test_many_sequences_of_all_lengths(causal, d, dtype):
    """Hundreds of items of no to six tiles; units whose first 128 queries, or all, see no key among them."""
    rng = random.Random(d)
    edges = [0, 1, 2, 5, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 300, 384, 511, 513, 700]
    ql = [rng.choice(edges) for _ in range(60)]
    kl = [n if rng.random() < 0.5 else rng.choice(edges) for n in ql]
    assert check(ql, kl, causal, 8, 2, d, dtype) > 3 * SMS


@pytest.mark.parametrize("causal", [True, False])
def test_chunks_of_heads(causal):
    """More than 48 MB of keys and values: the query heads run in chunks of eight and six."""
    rng = random.Random(1)
    ql = [rng.randrange(300, 700) for _ in range(42)]
    assert sum(ql) * 128 * 4 * 7 > 48 << 20 and sum(ql) * 128 * 4 * 4 < 48 << 20
    assert check(ql, ql, causal, 14, 7, 128, torch.bfloat16) > 6 * SMS


@pytest.mark.parametrize("n", [1, 200])
def test_one_item_more_than_sms(n):
    """149 items: the last is taken over by whichever block is done first."""
    assert check([n] * (SMS + 1), [n] * (SMS + 1), True, 1, 1, 64, torch.bfloat16) == SMS + 1
