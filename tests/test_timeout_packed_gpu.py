"""The pipeline-timeout path of the packed and paged attention kernels, exercised without a fault (see
test_timeout_gpu.py): with the loads held and a short limit the kernels report their codes, and the same calls compute
the same results afterwards. In a block of the paged kernel one warp of four gives up while the others, whose loads
arrive, go on to the barriers that they share with it."""
import pytest
import torch

from vmonarch_b200 import _native as N
from vmonarch_b200 import PackedSequences, packed_attention, paged_attention

pytestmark = pytest.mark.gpu


def held(call):
    """The status after `call` with the loads held."""
    torch.cuda.synchronize()
    assert N.device_status(torch.device("cuda", 0)) == 0
    N.check(N.lib.vmb_test_pipeline_timeout(20000, 1), "vmb_test_pipeline_timeout")
    try:
        call()
        torch.cuda.synchronize()
        return N.device_status(torch.device("cuda", 0))
    finally:
        N.check(N.lib.vmb_test_pipeline_timeout(0, 0), "vmb_test_pipeline_timeout")


def rows(*shape):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(sum(shape))).to(torch.bfloat16)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[300, 1, 70], [5000]])  # uncut units; cut ones with their joins
def test_packed_attention(lens, d):
    n = sum(lens)
    q, k, v, do = rows(n, 4, d).requires_grad_(), rows(n, 2, d).requires_grad_(), rows(n, 2, d).requires_grad_(), rows(n, 4, d)
    seqs = PackedSequences(lens)

    def forward():
        return packed_attention(q, k, v, seqs, causal=True)
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


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens, heads", [([40, 200, 1], 8), ([9000, 300, 0, 77], 8), ([2000] * 200, 16)])
def test_paged_attention(lens, heads, d):
    """Items of one block each, a cut item, and several items a block."""
    page, width = 16, -(-max(lens) // 16)
    table = torch.arange(width, dtype=torch.int32, device="cuda").repeat(len(lens), 1)
    kp, vp, q = rows(width, 1, page, d), rows(width + 1, 1, page, d)[1:], rows(len(lens), heads, d)
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def call():
        return paged_attention(q, kp, vp, table, lengths)
    want = call()
    assert held(call) >> 24 != 0
    assert torch.equal(call(), want)
    torch.cuda.synchronize()
    assert N.device_status(torch.device("cuda", 0)) == 0
