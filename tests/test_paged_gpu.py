"""The paged cache's calls against plain indexing, and attention over it against its definition in 64 bits.

Attention: P rounded (u, the element type's rounding) and the output rounded (u): at most 2 u in the
Frobenius norm. The moves are copies: equal."""
import pytest
import torch

from packed_reference import packed_reference
from vmonarch_b200 import PagedKVCache, PackedSequences, append_pages, copy_pages, packed_attention, paged_attention

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11}


def pool(lens, hk, d, page, dtype, seed=0, spare=3, poison=True):
    """Pools whose unused slots hold NaN, a page table in random order and the dense keys and values."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    used = [-(-n // page) for n in lens]
    num = sum(used) + spare
    kp, vp = (torch.full((num, hk, page, d), float("nan") if poison else 0.0, device="cuda", dtype=dtype) for _ in range(2))
    k, v = (torch.randn(sum(lens), hk, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    order = torch.randperm(num, generator=g, device="cuda")
    table = torch.full((len(lens), max(used + [1])), -7, dtype=torch.int32, device="cuda")
    pos = row = 0
    for i, n in enumerate(lens):
        mine = order[pos:pos + used[i]]
        table[i, :used[i]] = mine
        at = torch.arange(n, device="cuda")
        kp[mine[at // page], :, at % page], vp[mine[at // page], :, at % page] = k[row:row + n], v[row:row + n]
        pos, row = pos + used[i], row + n
    return kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), k, v


def check(lens, h, hk, d, page, dtype, scale=None):
    kp, vp, table, lengths, k, v = pool(lens, hk, d, page, dtype)
    q = torch.randn(len(lens), h, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)).to(dtype)
    o, lse = paged_attention(q, kp, vp, table, lengths, sm_scale=scale, return_lse=True)
    ref, rlse = packed_reference(q.double(), k.double(), v.double(), [1] * len(lens), lens, False,
                                 d ** -0.5 if scale is None else scale)
    assert torch.isfinite(o).all()
    assert ((o.double() - ref).norm() / ref.norm().clamp_min(1e-30)).item() <= 2 * U[dtype]
    for i, n in enumerate(lens):  # every sequence for itself: a short one must not hide behind a long one
        assert (o[i].double() - ref[i]).norm() <= 2 * U[dtype] * ref[i].norm()
    live = rlse.T > float("-inf")
    assert torch.equal(lse > float("-inf"), live)
    # sums of exponentials (2e-5 of scores of some units), and the scores' own error: d / 16 truncating 32-bit
    # accumulations (2^-23 each) and three roundings (2^-24) of their size, which is about |lse|'s
    bound = 2e-5 + (2 * d / 16 + 3) * 2.0 ** -24 * rlse[rlse > float("-inf")].abs().max() if live.any() else 0
    assert not live.any() or (lse.double() - rlse.T)[live].abs().max() <= bound
    return q, kp, vp, table, lengths, o


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h, hk", [(4, 4), (8, 2), (8, 1), (5, 1), (16, 1), (24, 1), (18, 2), (1, 1)])
@pytest.mark.parametrize("d", [128, 64, 96, 40, 8])
def test_heads_and_types(h, hk, d, dtype):
    check([1, 16, 201, 777, 64], h, hk, d, 16, dtype)


@pytest.mark.parametrize("page", [1, 7, 8, 24, 64, 100, 256])
@pytest.mark.parametrize("lens", [[1], [0], [0, 3, 0], [63, 64, 65, 127, 128, 129], [5000, 0, 17, 256, 257], [20000, 20000],
                                  [1] * 300, list(range(1, 130))])
def test_lengths_and_pages(lens, page):
    check(lens, 4, 2, 64, page, torch.bfloat16)


def test_splits_and_widths():
    """Long sequences beside short ones (items cut over many blocks), and tables wider than they need be."""
    check([70000, 3, 0, 9000], 8, 2, 128, 32, torch.bfloat16)
    q, kp, vp, table, lengths, o = check([100, 30, 1], 8, 2, 128, 16, torch.bfloat16)
    wide = torch.full((3, 4096), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.size(1)] = table
    # another split, so another order of the same 32-bit sums
    assert (paged_attention(q, kp, vp, wide, lengths).float() - o.float()).norm() <= 2 * U[torch.bfloat16] * o.float().norm()
    view = torch.zeros(3, 2 * table.size(1), dtype=torch.int32, device="cuda")
    view[:, :table.size(1)] = table
    assert torch.equal(paged_attention(q, kp, vp, view[:, :table.size(1)], lengths), o)


@pytest.mark.parametrize("scale", [0.0, 3.0])
def test_scales(scale):
    check([300, 40], 4, 2, 64, 16, torch.float16, scale)


def test_pool_layouts():
    """Slot-major pools, both tensors interleaved in one buffer, and strided queries: read in place."""
    q, kp, vp, table, lengths, o = check([300, 2, 90], 8, 2, 64, 16, torch.bfloat16)
    slot_major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kp, vp)]
    both = torch.stack([kp, vp], 1)
    wide = torch.zeros(3, 8, 192, device="cuda", dtype=q.dtype)
    wide[..., :64] = q
    for k, v in (slot_major, both.unbind(1)):
        assert torch.equal(paged_attention(wide[..., :64], k, v, table, lengths), o)


def test_stream_graph_and_changing_lengths():
    """Captured once, replayed with other lengths: the schedule is made on the device."""
    kp, vp, table, lengths, k, v = pool([3000, 500], 2, 64, 16, torch.bfloat16, poison=False)
    q = torch.randn(2, 8, 64, device="cuda").to(torch.bfloat16)
    live = lengths.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged_attention(q, kp, vp, table, live)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(q, kp, vp, table, live)
    for a, b in ((3000, 500), (1, 1), (2999, 0), (64, 448)):
        live.copy_(torch.tensor([a, b], dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, paged_attention(q, kp, vp, table, live))


def test_other_pages_take_no_part():
    """Pages of the pool outside the table, and slots past a length, hold NaN (pool() puts it there): see
    check(). Page ids outside the pool read as zeros, lengths past the table are cut."""
    kp, vp, table, lengths, k, v = pool([40], 1, 64, 16, torch.bfloat16)
    q = torch.randn(1, 2, 64, device="cuda").to(torch.bfloat16)
    bad = table.clone()
    bad[0, 1] = kp.size(0) + 5
    o = paged_attention(q, kp, vp, bad, lengths)
    k[16:32], v[16:32] = 0, 0
    ref = packed_reference(q.double(), k.double(), v.double(), [1], [40], False, 0.125)[0]
    assert (o.double() - ref).norm() <= 2 * U[torch.bfloat16] * ref.norm()
    full = pool([48], 1, 64, 16, torch.bfloat16)
    assert torch.equal(paged_attention(q, *full[:3], full[3]), paged_attention(q, *full[:3], full[3] + 1000))


def test_offsets_past_32_bits():
    """A pool of more than 2^31 elements, read and written at its far end."""
    hk, page, d = 8, 128, 128
    num = 2 ** 31 // (hk * page * d) + 40
    kp = torch.zeros(num, hk, page, d, device="cuda", dtype=torch.bfloat16)
    vp = torch.zeros_like(kp)
    n = 300
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(n, hk, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    pages = torch.tensor([num - 1, num - 7, num - 3], device="cuda")
    at = torch.arange(n, device="cuda")
    append_pages(k, v, kp, vp, (pages[at // page] * page + at % page).to(torch.int32))
    src = pages.to(torch.int32)
    dst = src - 20
    copy_pages(kp, vp, src, dst)
    q = torch.randn(1, hk, d, generator=g, device="cuda").to(torch.bfloat16)
    ref = packed_reference(q.double(), k.double(), v.double(), [1], [n], False, d ** -0.5)[0]
    for p in (src, dst):
        o = paged_attention(q, kp, vp, p[None], torch.tensor([n], dtype=torch.int32, device="cuda"))
        assert (o.double() - ref).norm() <= 2 * U[torch.bfloat16] * ref.norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hk, page, d", [(2, 16, 128), (1, 1, 8), (3, 7, 40), (8, 24, 64)])
def test_moves(hk, page, d, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    num = 50
    kp, vp = (torch.randn(num, hk, page, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    perm = torch.randperm(num, generator=g, device="cuda").to(torch.int32)
    src, dst = perm[:20], perm[20:40].clone()
    wk, wv = kp.clone(), vp.clone()
    wk[dst.long()], wv[dst.long()] = wk[src.long()], wv[src.long()]
    dst[3], keep = num, dst[3].clone()  # a page outside the pool: that pair is skipped
    wk[keep.long()], wv[keep.long()] = kp[keep.long()], vp[keep.long()]
    views = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kp, vp)]
    for k, v in ((kp, vp), views):
        copy_pages(k, v, src, dst)
        assert torch.equal(k, wk) and torch.equal(v, wv)
    rows = min(33, num * page - 1)
    slots = torch.randperm(num * page, generator=g, device="cuda")[:rows].to(torch.int32)
    k, v = torch.randn(2, rows, hk, d, generator=g, device="cuda").to(dtype)
    wk[slots.long() // page, :, slots.long() % page] = k
    wv[slots.long() // page, :, slots.long() % page] = v
    for bad in (-1, num * page):  # padding, and a slot past the pool
        s = torch.cat([slots, torch.tensor([bad], dtype=torch.int32, device="cuda")])
        append_pages(torch.cat([k, k[:1]]).transpose(0, 1).contiguous().transpose(0, 1), torch.cat([v, v[:1]]), kp, vp, s)
        assert torch.equal(kp, wk) and torch.equal(vp, wv)
    before = kp.clone()
    append_pages(k[:0], v[:0], kp, vp, slots[:0])
    copy_pages(kp, vp, src[:0], dst[:0])
    assert torch.equal(kp, before)


def test_cache_prompt_then_tokens():
    """A prompt through packed_attention, its keys and values in the cache, then token by token, with a fork
    on the way: every token's output is the causal attention's over the whole sequence."""
    h, hk, d, total = 8, 2, 64, 90
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(total, n, d, generator=g, device="cuda").to(torch.bfloat16) for n in (h, hk, hk))
    ref = packed_reference(q.double(), k.double(), v.double(), [total], [total], True, d ** -0.5)[0]
    cache = PagedKVCache(40, 16, hk, d, layers=2)
    a = cache.add()
    slots = cache.reserve([a], [70])
    for layer in range(2):
        cache.write(layer, k[:70], v[:70], slots)
    o = packed_attention(q[:70], k[:70], v[:70], PackedSequences([70]), causal=True)
    assert (o.double() - ref[:70]).norm() <= 2 * U[torch.bfloat16] * ref[:70].norm()
    b = cache.fork(a)
    for t in range(70, total):
        slots = cache.reserve([a, b], [1, 1])
        table, lengths = cache.tables([a, b])
        for layer in range(2):
            cache.write(layer, torch.stack([k[t], -k[t]]), torch.stack([v[t], -v[t]]), slots)
            o = cache.attend(layer, q[[t, t]], table, lengths)
            assert (o[0].double() - ref[t]).norm() <= 2 * U[torch.bfloat16] * ref[t].norm()
    kb = torch.cat([k[:70], -k[70:]])
    vb = torch.cat([v[:70], -v[70:]])
    other = packed_reference(q[-1:].double(), kb.double(), vb.double(), [1], [total], False, d ** -0.5)[0]
    assert (o[1].double() - other[0]).norm() <= 2 * U[torch.bfloat16] * other.norm()
    cache.free(a)
    cache.compact()
    table, lengths = cache.tables([b])
    assert torch.equal(cache.attend(1, q[-1:], table, lengths)[0], o[1])


def test_refusals():
    kp, vp, table, lengths, k, v = pool([40], 2, 64, 16, torch.bfloat16)
    q = torch.zeros(1, 4, 64, device="cuda", dtype=torch.bfloat16)
    ok = dict(q=q, k_pages=kp, v_pages=vp, page_table=table, lengths=lengths)
    for bad in (dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(page_table=table.long()),
                dict(lengths=lengths.long()), dict(page_table=table[0]), dict(lengths=lengths.cpu()),
                dict(lengths=lengths[:0]), dict(v_pages=vp[:1]), dict(v_pages=vp.half()), dict(sm_scale=-1.0),
                dict(k_pages=kp.transpose(2, 3), v_pages=vp.transpose(2, 3))):
        with pytest.raises(AssertionError):
            paged_attention(**{**ok, **bad})
    slots = torch.zeros(40, dtype=torch.int32, device="cuda")
    for args in ((k, v, kp, vp, slots.long()), (k, v, kp, vp, slots[:3]), (k.half(), v.half(), kp, vp, slots),
                 (k[:, :1], v[:, :1], kp, vp, slots), (k, v.cpu(), kp, vp, slots)):
        with pytest.raises(AssertionError):
            append_pages(*args)
    with pytest.raises(AssertionError):
        copy_pages(kp, vp, slots, slots[:3])
