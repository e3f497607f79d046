"""A small conditioned, causal transformer over packed sequences: trained on clips of different lengths,
then continued token by token from a paged cache.

Every block's attention is ``packed_attention`` (training, prompts) or the cache's ``attend`` (one token at a
time), and everything between two blocks is one ``gated_residual_norm``: the norm after the block that ends, its
gate, the residual, and the modulated norm before the one that begins, with gates, scales and shifts that a
conditioning vector gives each sequence.

    python examples/packed_transformer.py [--steps 60]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from vmonarch_b200 import PackedSequences, PagedKVCache, gated_residual_norm, packed_attention  # noqa: E402


class Block(nn.Module):
    """Attention and MLP without their norms, which the model runs between them."""

    def __init__(self, dim, heads, kv_heads):
        super().__init__()
        self.shape = heads, kv_heads, dim // heads
        self.qkv = nn.Linear(dim, (heads + 2 * kv_heads) * (dim // heads), bias=False)
        self.out = nn.Linear(dim, dim, bias=False)
        self.mlp = nn.Sequential(nn.Linear(dim, 4 * dim), nn.GELU(approximate="tanh"), nn.Linear(4 * dim, dim))

    def heads(self, h):
        """q, k, v of every token: views of one projection, which the kernels read in place."""
        heads, kv_heads, d = self.shape
        qkv = self.qkv(h).unflatten(-1, (-1, d))
        return qkv.split((heads, kv_heads, kv_heads), 1)


class PackedTransformer(nn.Module):
    def __init__(self, vocab=96, cond=16, dim=256, heads=4, kv_heads=2, layers=2):
        super().__init__()
        self.embed = nn.Embedding(vocab, dim)
        self.blocks = nn.ModuleList(Block(dim, heads, kv_heads) for _ in range(layers))
        # one norm before the first block, one after each of the 2 * layers halves (the last one before the head)
        self.weight = nn.Parameter(torch.ones(2 * layers + 1, dim))
        self.post_weight = nn.Parameter(torch.ones(2 * layers, dim))
        self.modulation = nn.Linear(cond, (6 * layers + 2) * dim)
        nn.init.zeros_(self.modulation.weight)
        nn.init.zeros_(self.modulation.bias)
        self.head = nn.Linear(dim, vocab, bias=False)

    def run(self, tokens, cond, seqs, attend):
        """Logits of every token; attend(layer, q, k, v) is the attention."""
        halves = 2 * len(self.blocks)
        mod = self.modulation(cond).unflatten(-1, (3 * halves + 2, -1))   # (sequences, rows, dim)
        row = iter(mod.unbind(1))
        x = self.embed(tokens)
        x, h = gated_residual_norm(x, scale=next(row), shift=next(row), weight=self.weight[0], seqs=seqs)
        for i in range(halves):
            block = self.blocks[i // 2]
            if i % 2 == 0:
                y = block.out(attend(i // 2, *block.heads(h)).flatten(1))
            else:
                y = block.mlp(h)
            x, h = gated_residual_norm(x, y, gate=1 + next(row), scale=next(row), shift=next(row),
                                       weight=self.weight[i + 1], post_weight=self.post_weight[i], seqs=seqs)
        return self.head(h)

    def forward(self, tokens, cond, seqs):
        return self.run(tokens, cond, seqs, lambda _, q, k, v: packed_attention(q, k, v, seqs, causal=True))

    def new_cache(self, num_pages, page_size=16):
        _, kv_heads, d = self.blocks[0].shape
        return PagedKVCache(num_pages, page_size, kv_heads, d, layers=len(self.blocks), dtype=self.head.weight.dtype,
                            device=self.head.weight.device)

    @torch.no_grad()
    def prompt(self, tokens, cond, seqs, cache, ids):
        """Runs prompts, leaves their keys and values in the cache, and returns all logits."""
        slots = cache.reserve(ids, seqs.q_lens)

        def attend(layer, q, k, v):
            cache.write(layer, k, v, slots)
            return packed_attention(q, k, v, seqs, causal=True)

        return self.run(tokens, cond, seqs, attend)

    @torch.no_grad()
    def step(self, tokens, cond, cache, ids):
        """One more token of each sequence; returns their logits."""
        slots = cache.reserve(ids, [1] * len(ids))
        table, lengths = cache.tables(ids)

        def attend(layer, q, k, v):
            cache.write(layer, k, v, slots)
            return cache.attend(layer, q, table, lengths)

        return self.run(tokens, cond, PackedSequences([1] * len(ids), device=tokens.device), attend)


def clips(count, longest, vocab, cond, generator):
    """Packed counting sequences: each starts anywhere and goes on by a stride that its condition names."""
    lens = torch.randint(2, longest + 1, (count,), generator=generator).tolist()
    stride = torch.randint(0, cond, (count,), generator=generator)
    start = torch.randint(0, vocab, (count,), generator=generator)
    tokens = torch.cat([(s + (d + 1) * torch.arange(n)) % vocab for s, d, n in zip(start, stride, lens)])
    return tokens, F.one_hot(stride, cond).float(), lens


def train(model, steps, device, seed=0, vocab=96, cond=16):
    """Next-token training on packed clips; returns the losses."""
    g = torch.Generator().manual_seed(seed)
    opt = torch.optim.AdamW(model.parameters(), lr=2e-3)
    losses = []
    for _ in range(steps):
        tokens, c, lens = clips(24, 200, vocab, cond, g)
        seqs = PackedSequences(lens, device=device)
        logits = model(tokens.to(device), c.to(device, model.head.weight.dtype), seqs).float()
        last = torch.tensor(lens).cumsum(0) - 1  # the last token of a clip has no next one
        target = tokens.roll(-1)
        target[last] = -100
        loss = F.cross_entropy(logits, target.to(device))
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    return losses


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=60)
    args = ap.parse_args()
    device = torch.device("cuda", 0)
    torch.manual_seed(0)
    model = PackedTransformer().to(device, torch.bfloat16)
    losses = train(model, args.steps, device)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} over {args.steps} steps")
    tokens, c, lens = clips(3, 40, 96, 16, torch.Generator().manual_seed(1))
    tokens, c = tokens.to(device), c.to(device, torch.bfloat16)
    cache = model.new_cache(64)
    ids = [cache.add() for _ in lens]
    last = torch.tensor(lens, device=device).cumsum(0) - 1
    token = model.prompt(tokens, c, PackedSequences(lens, device=device), cache, ids)[last].argmax(-1)
    out = [token]
    for _ in range(11):
        token = model.step(token, c, cache, ids).argmax(-1)
        out.append(token)
    for i, row in enumerate(torch.stack(out, 1).tolist()):
        print(f"sequence {i}: ... {tokens[last[i]].item()} -> {row}")


if __name__ == "__main__":
    main()
