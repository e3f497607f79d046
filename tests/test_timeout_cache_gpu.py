"""The pipeline-timeout path of the windowed and the 8-bit attention kernels, exercised without a fault (see
test_timeout_packed_gpu.py): with the loads held and a short limit they report their codes, and the same calls compute the
same results afterwards."""
import pytest
import torch

from test_timeout_packed_gpu import held, rows
from vmonarch_b200 import _native as N
from vmonarch_b200 import PackedSequences, packed_attention, paged_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens, window, sinks", [([300, 1, 70], 100, 5), ([5000], 4000, 200)])
def test_windowed_packed_attention(lens, window, sinks, d):
    n = sum(lens)
    q, k, v, do = rows(n, 4, d).requires_grad_(), rows(n, 2, d).requires_grad_(), rows(n, 2, d).requires_grad_(), rows(n, 4, d)
    seqs = PackedSequences(lens)

    def forward():
        return packed_attention(q, k, v, seqs, causal=True, window=window, sinks=sinks)
    o = forward()

    def backward():
        return torch.autograd.grad(o, (q, k, v), do, retain_graph=True)
    want = [o, *backward()]
    assert held(forward) >> 24 != 0
    assert held(backward) >> 24 != 0
    for a, b in zip([forward(), *backward()], want):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    assert N.device_status(torch.device("cuda", 0)) == 0


@pytest.mark.parametrize("bits, window", [(8, None), (8, 300), (16, 300)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens, heads", [([40, 200, 1], 8), ([9000, 300, 0, 77], 8), ([9000, 300, 0, 77], 16), ([2000] * 400, 8)])
def test_cached_attention(lens, heads, d, bits, window):
    """Items of one block each, a cut item, 16 heads a pass, and several items a block; of four warps one gets no loads."""
    page, width = 16, -(-max(lens) // 16)
    table = torch.arange(width, dtype=torch.int32, device="cuda").repeat(len(lens), 1)
    kp, vp, q = rows(width, 1, page, d), rows(width + 1, 1, page, d)[1:], rows(len(lens), heads, d)
    kw = dict(window=window, sinks=7 if window else 0)
    if bits == 8:
        kp, vp = kp.to(torch.float8_e4m3fn), vp.to(torch.float8_e4m3fn)
        kw["k_scale"] = kw["v_scale"] = torch.full((width, 1), 0.5, device="cuda")
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def call():
        return paged_attention(q, kp, vp, table, lengths, **kw)
    want = call()
    assert held(call) >> 24 != 0
    assert torch.equal(call(), want)
    torch.cuda.synchronize()
    assert N.device_status(torch.device("cuda", 0)) == 0
