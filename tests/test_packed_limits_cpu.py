"""Row numbers of the backward's statistics are 32-bit, with every sequence padded to 128 rows: many short sequences
pass that before their rows do, and are refused instead of wrapping around."""
import ctypes

import pytest
import torch

from test_ops_capi import packed
from vmonarch_b200 import PackedSequences
from vmonarch_b200 import _native as N


def test_too_many_padded_rows_are_refused():
    seqs = PackedSequences([1, 1], device="cpu")
    assert seqs.stat_rows == 256
    seqs.stat_rows = 2 ** 31  # as of 2^24 sequences of one row
    key = (True, torch.bfloat16, 2, 2, 64)
    with pytest.raises(AssertionError, match="padded"):
        seqs._template((True, True, 0.125, *key[1:]))
    seqs._template((False, True, 0.125, *key[1:]))  # the forward has no such rows
    assert N.lib.vmb_packed_bwd(ctypes.byref(packed(stat_rows=2 ** 31)), None) == 1
    assert b"row counts" in N.lib.vmb_last_error()
