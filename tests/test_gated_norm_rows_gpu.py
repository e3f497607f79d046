"""The gated residual norm over so many rows that every group of threads goes through several: the rings of loads wrap
around, the two buffers of the meetings alternate, and column sums run over many rows and across sequences. Tolerances
as in test_gated_norm_gpu.py (a column's sum passes some hundred roundings of 2^-24 in 32 bits here too: up to 50 rows
in a thread, then the blocks' partials in groups of 16)."""
import pytest
import torch

from test_gated_norm_gpu import check

pytestmark = pytest.mark.gpu


def rows_for(c):
    """At least six rows a group: two more than the most stages of a ring (148 blocks of up to 640 threads)."""
    return 15000 if c <= 512 else 9000 if c <= 2048 else 4600 if c <= 5120 else 2800


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("c", [80, 256, 264, 512, 520, 1040, 2048, 4096, 5120, 5128, 7000, 8192])
def test_rings_wrap_around(c, norm):
    n = rows_for(c)
    lens = [n * 2 // 5, 1, 0, n - n * 2 // 5 - 1]
    check(lens, c, torch.bfloat16, torch.float32, norm)
    check(lens, c, torch.float16, torch.float16, norm, ("post_weight",))


@pytest.mark.parametrize("c", [80, 2048, 5120, 8192])
def test_rings_of_the_first_norm(c):
    """Without a block output (three streams of loads instead of four, one instead of two forward)."""
    n = rows_for(c)
    check([n - 7, 7], c, torch.bfloat16, torch.float32, "layer", ("y", "gate", "post_weight"))
