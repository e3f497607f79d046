"""The example model with a window: its gradients against the same model over a plain attention in 64 bits, and its tokens one
by one over the cache against its packed forward."""
import sys
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

from window_reference import window_reference

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))

pytestmark = pytest.mark.gpu
WINDOW, SINKS = 17, 3


def setup(seed):
    from packed_transformer import PackedTransformer, clips
    device = torch.device("cuda", 0)
    torch.manual_seed(seed)
    model = PackedTransformer(window=WINDOW, sinks=SINKS).to(device, torch.bfloat16)
    with torch.no_grad():  # its modulation starts at zero: let it take part
        model.modulation.weight.normal_(std=0.2)
    tokens, c, lens = clips(5, 60, 96, 16, torch.Generator().manual_seed(seed))
    return model, tokens.to(device), c.to(device, torch.bfloat16), lens


def test_gradients():
    """Four halves of a layer, each with a forward and a backward rounding of bf16 (2^-8) that the two attentions do not share,
    in both directions: 2 x 2 x 4 x 2^-8 in the Frobenius norm."""
    from vmonarch_b200 import PackedSequences
    model, tokens, c, lens = setup(0)
    seqs = PackedSequences(lens)
    target = tokens.roll(-1)

    def grads(logits):
        model.zero_grad()
        F.cross_entropy(logits.float(), target).backward()
        return {n: p.grad.double() for n, p in model.named_parameters()}

    def plain(_, q, k, v):
        return window_reference(q.double(), k.double(), v.double(), lens, lens, WINDOW, SINKS, q.size(2) ** -0.5)[0].to(q.dtype)
    got, want = grads(model(tokens, c, seqs)), grads(model.run(tokens, c, seqs, plain))
    for name in want:
        assert torch.isfinite(got[name]).all()
        assert (got[name] - want[name]).norm() <= 2 * 2 * 4 * 2.0 ** -8 * want[name].norm(), name


@pytest.mark.parametrize("bits", [16, 8])
def test_tokens_over_the_cache(bits):
    """Two roundings of bf16 activations a layer over the few layers of the model, as without a window; over an 8-bit cache, whose
    rounding test_cache8_gpu.py holds to its rule, for running."""
    from vmonarch_b200 import PackedSequences
    model, tokens, c, lens = setup(1)
    with torch.no_grad():
        want = model(tokens, c, PackedSequences(lens)).float()
    start = [0] + torch.tensor(lens).cumsum(0).tolist()
    half = [max(1, n // 2) for n in lens]
    cache = model.new_cache(64, page_size=8, dtype=torch.float8_e4m3fn if bits == 8 else None)
    ids = [cache.add() for _ in lens]
    rows = torch.cat([torch.arange(start[i], start[i] + half[i]) for i in range(5)]).cuda()
    got = dict(zip(rows.tolist(), model.prompt(tokens[rows], c, PackedSequences(half), cache, ids)))
    for t in range(max(lens)):
        live = [i for i in range(5) if half[i] + t < lens[i]]
        if live:
            at = [start[i] + half[i] + t for i in live]
            got.update(zip(at, model.step(tokens[at], c[live], cache, [ids[i] for i in live])))
    got = torch.stack([got[r] for r in range(len(tokens))]).float()
    assert torch.isfinite(got).all()
    if bits == 16:
        assert (got - want).norm() <= 2 * 4 * 2.0 ** -8 * want.norm()
