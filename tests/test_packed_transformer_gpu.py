"""The example that runs the packed attention, the paged cache and the gated norm together as a model."""
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))

pytestmark = pytest.mark.gpu


def test_trains_and_continues():
    from packed_transformer import PackedTransformer, clips, train
    from vmonarch_b200 import PackedSequences
    device = torch.device("cuda", 0)
    torch.manual_seed(0)
    model = PackedTransformer().to(device, torch.bfloat16)
    losses = train(model, 40, device)
    assert losses[-1] < 0.5 * losses[0]
    # token by token over the cache gives the packed forward's logits: two roundings of bf16 activations a layer
    # (2^-8 each) over the few layers of the model
    tokens, c, lens = clips(5, 60, 96, 16, torch.Generator().manual_seed(3))
    tokens, c = tokens.to(device), c.to(device, torch.bfloat16)
    seqs = PackedSequences(lens)
    with torch.no_grad():
        want = model(tokens, c, seqs).float()
    start = [0] + torch.tensor(lens).cumsum(0).tolist()
    half = [max(1, n // 2) for n in lens]
    cache = model.new_cache(64, page_size=8)
    ids = [cache.add() for _ in lens]
    rows = torch.cat([torch.arange(start[i], start[i] + half[i]) for i in range(5)]).to(device)
    got = {}
    logits = model.prompt(tokens[rows], c, PackedSequences(half), cache, ids)
    for r, x in zip(rows.tolist(), logits):
        got[r] = x
    live = list(range(5))
    for t in range(max(lens)):
        live = [i for i in live if half[i] + t < lens[i]]
        if not live:
            break
        at = [start[i] + half[i] + t for i in live]
        logits = model.step(tokens[at], c[live], cache, [ids[i] for i in live])
        for r, x in zip(at, logits):
            got[r] = x
    got = torch.stack([got[r] for r in range(len(tokens))]).float()
    assert ((got - want).norm() / want.norm()).item() <= 2 * 4 * 2.0 ** -8
