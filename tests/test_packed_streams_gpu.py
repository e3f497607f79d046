"""A PackedSequences that is dropped while another stream still works with it: its lists' memory is not given to
others before that stream is done. (Nothing is written into what the allocator gives out here.)"""
import gc

import pytest
import torch

from vmonarch_b200 import PackedSequences, gated_residual_norm, packed_attention

pytestmark = pytest.mark.gpu
LENS = [700, 3, 90]


def attention(seqs):
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(sum(LENS), 4, 64, device="cuda", generator=g).to(torch.bfloat16).requires_grad_() for _ in range(3))

    def run():
        o = packed_attention(q, k, v, seqs[0], causal=True)
        return [o.detach(), *torch.autograd.grad(o, (q, k, v), torch.ones_like(o))]
    return run


def norm(seqs):
    x = torch.randn(sum(LENS), 64, device="cuda").to(torch.bfloat16)
    scale = torch.randn(len(LENS), 64, device="cuda").to(torch.bfloat16)
    return lambda: list(gated_residual_norm(x, x, scale=scale, seqs=seqs[0]))


@pytest.mark.parametrize("call", [attention, norm])
def test_dropped_while_another_stream_works(call):
    seqs = [PackedSequences(LENS)]
    run = call(seqs)
    want = run()  # the lists are made on this stream
    kept = [t for hit in seqs[0]._cache.values() for t in (hit if isinstance(hit, tuple) else (hit,)) if isinstance(t, torch.Tensor)]
    at, sizes = {t.data_ptr() for t in kept}, {t.nbytes for t in kept}
    assert at
    del kept
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)  # some 0.2 s
        got = run()
    seqs.clear()
    del run
    gc.collect()
    given = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(64)]
    assert not side.query(), "the other stream was done too soon for this test"
    assert not at & {t.data_ptr() for t in given}
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
