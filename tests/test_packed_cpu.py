"""Packed sequences on the host: the work lists cover every query, key and visible pair exactly once,
and calls that the operator does not take are refused before any CUDA work."""
import numpy as np
import pytest
import torch

from vmonarch_b200 import PackedSequences, packed_attention

LENS = [([130], None), ([1, 0, 300, 7], None), ([1, 5, 257, 128, 513], [0, 200, 31, 128, 600]),
        ([5, 200, 300, 700], [9, 100, 1, 900]), ([2], [5000]), ([5000], [2]), ([0, 0], [3, 0]), ([64] * 9, None)]


def units(seqs, kind, causal, heads, group):
    """A kernel's unit list as the device holds it (the lists live on the sequences' device)."""
    seqs._list(kind, causal, heads, group)
    info, dev = seqs._cache[(kind, causal, heads, group)]
    u, joins = dev.numpy()[:12 * info.n_units].reshape(-1, 12), dev.numpy()[12 * info.n_units:].reshape(-1, 2)
    assert len(joins) == info.n_joins and (not len(joins) or info.joins == info.units + 48 * info.n_units)
    # pieces of cut units: consecutive parts and ranges, each unit joined once; reported as one
    parts, whole = [], [x for x in u if x[7] < 0]
    for first, n in joins:
        mine = sorted((x for x in u if u[first][7] <= x[7] < u[first][7] + n), key=lambda x: x[7])
        assert len(mine) == n > 1 and all((x[[0, 1, 2, 3, 4, 8]] == mine[0][[0, 1, 2, 3, 4, 8]]).all() for x in mine)
        assert all(a[6] == b[5] and a[6] > a[5] for a, b in zip(mine, mine[1:]))
        parts += [x[7] for x in mine]
        one = mine[0].copy()
        one[6], one[7] = mine[-1][6], -1
        whole.append(one)
    assert sorted(parts) == list(range(info.n_parts))
    return np.array(whole).reshape(-1, 12)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ql, kl", LENS)
def test_query_units_cover_rows_and_visible_keys(ql, kl, causal):
    seqs = PackedSequences(ql, kl, device="cpu")
    kl = ql if kl is None else kl
    q_start, k_start = np.cumsum([0] + ql), np.cumsum([0] + kl)
    stat = np.cumsum([0] + [-(-n // 128) * 128 for n in ql])
    for kind, rows in (("fwd", 256), ("dq", 128)):
        seen = np.zeros(sum(ql), int)
        for q_row, q_valid, k_row, k_valid, vis0, begin, end, part, stat_row, *_ in units(seqs, kind, causal, 2, 1):
            s = np.searchsorted(q_start, q_row, side="right") - 1
            first = q_row - q_start[s]
            assert 1 <= q_valid <= rows and first % rows == 0 and first + q_valid <= ql[s]
            assert (k_row, k_valid) == (k_start[s], kl[s]) and part == -1 and begin == 0
            assert stat_row == stat[s] + first
            seen[q_row:q_row + q_valid] += 1
            limits = [min(max(kl[s] - ql[s] + first + r + 1, 0), kl[s]) if causal else kl[s] for r in range(q_valid)]
            assert [min(max(vis0 + r if causal else k_valid, 0), k_valid) for r in range(q_valid)] == limits
            assert end == -(-max(limits) // 128)
        assert (seen == 1).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ql, kl", LENS)
def test_key_units_cover_keys_and_the_queries_that_see_them(ql, kl, causal):
    group = 3
    seqs = PackedSequences(ql, kl, device="cpu")
    kl = ql if kl is None else kl
    q_start, k_start = np.cumsum([0] + ql), np.cumsum([0] + kl)
    seen = np.zeros(sum(kl), int)
    for q_row, q_valid, k_row, k_valid, vis0, begin, end, part, stat_row, *_ in units(seqs, "kv", causal, 6, group):
        s = np.searchsorted(k_start, k_row, side="right") - 1
        first = k_row - k_start[s]
        assert 1 <= k_valid <= 128 and first % 128 == 0 and (q_row, q_valid) == (q_start[s], ql[s])
        seen[k_row:k_row + k_valid] += 1
        t0 = max(vis0, 0) // 64
        tiles = [t for t in range(-(-ql[s] // 64)) if any(
            not causal or first <= kl[s] - ql[s] + q for q in range(64 * t, min(64 * t + 64, ql[s])))]
        assert begin == 0 and end == group * len(tiles)
        assert tiles == list(range(t0, t0 + len(tiles)))
        if causal:
            for r in range(k_valid):
                assert [q for q in range(ql[s]) if q >= vis0 + r] == \
                    [q for q in range(ql[s]) if first + r <= kl[s] - ql[s] + q]
    assert (seen == 1).all()


def test_longest_work_first_and_cut_where_the_sms_finish_sooner():
    """Pieces are never below half the least worth a piece, and a cut list is done before the uncut one, its join
    included; large lists hold no unit much above the SMs' fair share."""
    from vmonarch_b200.packed import _JOIN, _JOINED, _LEAST, _MANY, _PIECE, _SETUP, _span
    for lens in ([5, 900, 40, 333], [30000], [8000, 100], [200] * 60, [3677], [130]):
        for kind in ("fwd", "dq", "kv"):
            for heads, group in ((2, 2), (40, 5), (1, 1)):
                seqs = PackedSequences(lens, device="cpu")
                info = seqs._list(kind, True, heads, group)
                u = seqs._cache[(kind, True, heads, group)][1].numpy()[:12 * info.n_units].reshape(-1, 12)
                work, part = u[:, 6] - u[:, 5], u[:, 7] >= 0
                assert (np.diff(work) <= 0).all()
                blocks = heads // group if kind == "kv" else heads
                whole = seqs._key_units(True, group) if kind == "kv" else seqs._query_units(256 if kind == "fwd" else 128, True)
                if part.any():
                    assert work[part].min() >= _LEAST[kind] // 2
                    after = _span(np.sort(-work - _PIECE * part), blocks, _SETUP[kind]) + _JOIN + part.sum() * blocks // _JOINED
                    assert after < _span(np.sort(-whole[:, 6]), blocks, _SETUP[kind])
                if len(whole) * blocks > _MANY:
                    assert work.max() <= max(_LEAST[kind], -(-int(work.sum()) * blocks // 148)) * 5 // 4 + 1


@pytest.mark.parametrize("bad", [dict(lengths=[]), dict(lengths=[3, -1]), dict(lengths=[3], kv_lengths=[1, 2]),
                                 dict(lengths=[2 ** 31])])
def test_sequences_refuse_bad_lengths(bad):
    with pytest.raises(AssertionError):
        PackedSequences(device="cpu", **bad)


def test_lengths_from_a_tensor():
    seqs = PackedSequences(torch.tensor([3, 4], dtype=torch.int32), device="cpu")
    assert seqs.total_q == seqs.total_k == 7 and seqs.num_sequences == 2


def rows(t=7, h=4, d=64, dtype=torch.bfloat16):
    return torch.zeros(t, h, d, dtype=dtype)


@pytest.mark.parametrize("args, kw, why", [
    ((rows(dtype=torch.float32), rows(dtype=torch.float32), rows(dtype=torch.float32)), {}, "dtype"),
    ((rows(), rows(), rows(dtype=torch.float16)), {}, "dtype"),
    ((rows(d=132), rows(d=132), rows(d=132)), {}, "head dim"),
    ((rows(d=136), rows(d=136), rows(d=136)), {}, "head dim"),
    ((rows(d=20), rows(d=20), rows(d=20)), {}, "head dim"),
    ((rows(), rows(h=3), rows(h=3)), {}, "multiple of Hk"),
    ((rows(), rows(d=32), rows(d=32)), {}, "total_q"),
    ((rows(), rows(), rows(t=6)), {}, "total_q"),
    ((rows()[0], rows(), rows()), {}, "total_q"),
    ((rows(), rows(), rows()), {}, "CUDA"),
])
def test_refusals(args, kw, why):
    with pytest.raises(AssertionError, match=why):
        packed_attention(*args, PackedSequences([7], device="cpu"), **kw)
