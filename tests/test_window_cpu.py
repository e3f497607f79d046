"""Attention with a window on the host: its work lists cover every visible pair once and leave out what no query of a unit
sees, and calls that the operator does not take are refused before any CUDA work."""
import ctypes

import numpy as np
import pytest
import torch

from test_ops_capi import packed
from test_packed_cpu import LENS, rows, units
from vmonarch_b200 import PackedSequences, packed_attention
from vmonarch_b200 import _native as N
from window_reference import visible

MASKS = [(1, 0), (1, 1), (5, 0), (64, 3), (100, 129), (128, 0), (129, 128), (200, 300), (1000, 7), (3, 2000), (2 ** 30 - 1024, 0)]


def seen(ql, kl, mask):
    return [visible(a, b, *mask).numpy() for a, b in zip(ql, kl)]


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("ql, kl", LENS)
def test_query_units_walk_the_visible_tiles(ql, kl, mask):
    seqs = PackedSequences(ql, kl, device="cpu")
    kl = ql if kl is None else kl
    window, sinks = mask
    q_start, vis = np.cumsum([0] + ql), seen(ql, kl, mask)
    for kind, rows_ in (("fwd", 256), ("dq", 128)):
        count = np.zeros(sum(ql), int)
        for q_row, q_valid, _, k_valid, vis0, begin, end, part, _, _, lone, extra in units(seqs, kind, mask, 2, 1):
            s = np.searchsorted(q_start, q_row, side="right") - 1
            first = q_row - q_start[s]
            count[q_row:q_row + q_valid] += 1
            assert begin == 0 and part == -1 and 1 <= q_valid <= rows_
            tiles = [x if x < lone else x + extra for x in range(end)]
            assert len(set(tiles)) == len(tiles) and all(128 * x < k_valid for x in tiles)
            mine = vis[s][first:first + q_valid]
            want = [x for x in range(-(-kl[s] // 128)) if mine[:, 128 * x:128 * x + 128].any()]
            assert set(want) <= set(tiles)
            # beyond them: whole tiles between the unit's first key in sight and its last
            assert len(tiles) <= len(want) + 1 + (sinks > 0)
        assert (count == 1).all()


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("ql, kl", LENS)
def test_key_units_walk_the_queries_that_see_them(ql, kl, mask):
    group = 3
    seqs = PackedSequences(ql, kl, device="cpu")
    kl = ql if kl is None else kl
    k_start, vis = np.cumsum([0] + kl), seen(ql, kl, mask)
    count = np.zeros(sum(kl), int)
    for q_row, q_valid, k_row, k_valid, vis0, begin, end, part, _, _, lone, extra in units(seqs, "kv", mask, 6, group):
        s = np.searchsorted(k_start, k_row, side="right") - 1
        first = k_row - k_start[s]
        count[k_row:k_row + k_valid] += 1
        assert extra == min(max(mask[1] - first, 0), k_valid)
        mine = vis[s][:, first:first + k_valid]
        tiles = [t for t in range(-(-ql[s] // 64)) if mine[64 * t:64 * t + 64].any()]
        t0 = max(vis0, 0) // 64
        assert begin == 0 and end % group == 0 and tiles == list(range(t0, t0 + end // group))
        # the kernel's own count of a head's tiles
        q_end = q_valid if extra else max(min(q_valid, vis0 + k_valid - 1 + mask[0]), 0)
        assert end // group == max(-(-q_end // 64) - t0, 0)
        # its masks: rows c_lo <= query < c_hi, and the queries without a gradient of their scores
        for r in range(k_valid):
            hi = q_valid if r < extra else min(q_valid, vis0 + r + mask[0])
            assert np.array_equal(mine[:, r], (np.arange(ql[s]) >= vis0 + r) & (np.arange(ql[s]) < hi))
        assert np.array_equal(np.arange(ql[s]) >= lone, vis[s].sum(1) > 1)
    assert (count == 1).all()


def test_pieces_of_windowed_units():
    """Cut units keep their skipped tiles; units() checks that the pieces of each are consecutive."""
    for mask in ((5000, 300), (20000, 4)):
        seqs = PackedSequences([30000], device="cpu")
        for kind, heads, group in (("fwd", 1, 1), ("dq", 1, 1), ("kv", 2, 2)):
            whole = seqs._key_units(mask, group) if kind == "kv" else seqs._query_units(256 if kind == "fwd" else 128, mask)
            got = units(seqs, kind, mask, heads, group)
            assert sorted(got[:, 6]) == sorted(whole[:, 6]) and sorted(got[:, 11]) == sorted(whole[:, 11])


def test_a_window_as_long_as_the_sequences_lists_the_causal_units():
    seqs = PackedSequences([300, 5, 900], [300, 40, 1000], device="cpu")
    for kind in ("fwd", "dq", "kv"):  # (of few heads the forward's units are smaller)
        assert np.array_equal(units(seqs, kind, (1000, 0), 40, 1), units(seqs, kind, True, 40, 1))
    most = {kind: [units(seqs, kind, mask, 2, 1)[:, 1].max() for mask in ((1000, 0), True)] for kind in ("fwd", "dq")}
    assert most == {"fwd": [128, 256], "dq": [128, 128]}


@pytest.mark.parametrize("kw, why", [
    (dict(window=4), "causal"), (dict(window=0, causal=True), "at least 1"), (dict(window=-3, causal=True), "at least 1"),
    (dict(window=4, sinks=-1, causal=True), "negative"), (dict(sinks=4, causal=True), "sinks need a window"),
    (dict(window=4, causal=True), "CUDA"),
])
def test_refusals(kw, why):
    with pytest.raises(AssertionError, match=why):
        packed_attention(rows(), rows(), rows(), PackedSequences([7], device="cpu"), **kw)
    with pytest.raises(TypeError):
        packed_attention(rows(), rows(), rows(), PackedSequences([7], device="cpu"), causal=True, window=2.5)


@pytest.mark.parametrize("over, window, sinks, code", [
    (dict(causal=0), 4, 0, 1), (dict(causal=1), 0, 0, 1), (dict(causal=1), 4, -1, 1), (dict(causal=1, dtype=2), 4, 0, 1),
    (dict(causal=1, k_total=2 ** 30), 4, 0, 2), (dict(causal=1, q_total=2 ** 30), 4, 0, 2), (dict(causal=1, dim=20), 4, 0, 2),
])
def test_entry_refusals(over, window, sinks, code):
    for fn in (N.lib.vmb_packed_window_fwd, N.lib.vmb_packed_window_bwd):
        assert fn(ctypes.byref(packed(**over)), window, sinks, None) == code
        assert N.lib.vmb_last_error()
        assert fn(None, 4, 0, None) == 1
