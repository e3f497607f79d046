"""Values that are not finite in key tiles that one half of a 256-query unit sees whole and the other half in part:
the queries from their position on get them, always, and no earlier one."""
import pytest
import torch

from vmonarch_b200 import PackedSequences, packed_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("nq, nk", [(129, 256), (385, 512), (256, 256), (200, 330), (255, 128)])
def test_values_that_half_a_unit_sees(nq, nk, bad, d):
    heads = 16
    g = torch.Generator(device="cuda").manual_seed(nq)
    q, k, v = (torch.randn(n, heads, d, device="cuda", generator=g).to(torch.bfloat16) for n in (nq, nk, nk))
    seqs = PackedSequences([nq], [nk])
    clean = packed_attention(q, k, v, seqs, causal=True)
    lims = torch.arange(nq, device="cuda") + nk - nq + 1
    for at in sorted({nk - 128, nk - 127, nk - 65, nk - 30, nk - 1} | ({nk - 129, nk - 200} if nk > 200 else set())):
        w = v.clone()
        w[at, :, 5] = bad
        w[at, ::2, d - 1] = bad
        hit = torch.zeros_like(clean, dtype=torch.bool)
        hit[lims > at, :, 5] = True
        hit[lims > at, ::2, d - 1] = True
        for _ in range(20):  # whichever half comes first
            o = packed_attention(q, k, w, seqs, causal=True)
            assert torch.equal(o[~hit], clean[~hit])
            assert (o[hit] == bad).all() if bad == bad else torch.isnan(o[hit]).all()
