"""The example model over an 8-bit cache: every attention of its steps against the definition in 64 bits over what the cache holds,
and what it holds against what the model wrote."""
import pytest
import torch

from test_window_transformer_gpu import SINKS, WINDOW, setup
from window_reference import window_reference

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def test_every_attention_of_the_steps(monkeypatch):
    """P and the output rounded to 16 bits (2^-8 each): 2 x 2^-8 in the Frobenius norm, a sequence at a time. Rows that are held: four
    significant bits (2^-4), once more where a page grew and values became subnormal (2^-10 of a scale of at most |x| max / 224)."""
    from vmonarch_b200 import PackedSequences, PagedKVCache
    model, tokens, c, lens = setup(1)
    half = [max(1, n // 2) for n in lens]
    cache = model.new_cache(64, page_size=8, dtype=E4M3)
    ids = [cache.add() for _ in lens]
    written, calls, live = {}, [], list(ids)

    def held(layer, seq):
        at = torch.arange(cache.length(seq), device="cuda")
        pages = torch.tensor(cache.pages(seq), device="cuda")[at // 8]
        return [p[layer].view(torch.uint8)[pages, :, at % 8].view(E4M3).double() * s[layer][pages][..., None].double()
                for p, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]

    write, attend = PagedKVCache.write, PagedKVCache.attend

    def spied_write(self, layer, k, v, slots):
        write(self, layer, k, v, slots)
        first = 0
        rows = half if len(slots) == sum(half) and not calls else [1] * len(live)
        for seq, n in zip(live, rows):
            written.setdefault((layer, seq), []).append((k[first:first + n].double(), v[first:first + n].double()))
            first += n
        assert first == len(slots)

    def spied_attend(self, layer, q, table, lengths, **kw):
        assert kw == dict(window=WINDOW, sinks=SINKS)
        o = attend(self, layer, q, table, lengths, **kw)
        for i, seq in enumerate(live):
            k, v = held(layer, seq)
            ref = window_reference(q[i:i + 1].double(), k, v, [1], [len(k)], WINDOW, SINKS, q.size(2) ** -0.5)[0]
            assert (o[i].double() - ref[0]).norm() <= 2 * 2.0 ** -8 * ref.norm()
            for x, rows in zip((k, v), zip(*written[layer, seq])):
                rows = torch.cat(rows)
                assert ((x - rows).abs() <= rows.abs() * 2.0 ** -4 + 2 * 2.0 ** -10 * rows.abs().max() / 224).all()
        calls.append(len(live))
        return o
    monkeypatch.setattr(PagedKVCache, "write", spied_write)
    monkeypatch.setattr(PagedKVCache, "attend", spied_attend)
    start = [0] + torch.tensor(lens).cumsum(0).tolist()
    rows = torch.cat([torch.arange(start[i], start[i] + half[i]) for i in range(5)]).cuda()
    model.prompt(tokens[rows], c, PackedSequences(half), cache, ids)
    for t in range(max(lens)):
        who = [i for i in range(5) if half[i] + t < lens[i]]
        if who:
            live[:] = [ids[i] for i in who]
            model.step(tokens[[start[i] + half[i] + t for i in who]], c[who], cache, live)
    assert sum(calls) == len(model.blocks) * sum(n - h for n, h in zip(lens, half))
