"""The paged cache in 8 bits, and with a window in 8 and 16: attention against its definition in 64 bits, rows that are appended
against their rule.

Attention: P rounded to 16 bits (u, half a step of the element type; fp16's 2^-11 over 8-bit pools, below u) and the output
rounded (u): at most 2 u in the Frobenius norm. Appended values and scales are exact: a scale is a power of two, so only the one
rounding of a quotient is left, which the reference makes too."""
import pytest
import torch

from vmonarch_b200 import PagedKVCache, PackedSequences, append_pages, copy_pages, packed_attention, paged_attention
from window_reference import visible, window_reference

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E4M3 = torch.float8_e4m3fn
ALL = 10 ** 9


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def pool8(lens, hk, d, page, seed=0, spare=3, scales=None):
    """8-bit pools whose unused slots hold NaN, their scales, a page table in random order, lengths, and what the tokens' keys
    and values stand for, in 64 bits."""
    g = gen(seed)
    used = [-(-n // page) for n in lens]
    num = sum(used) + spare
    order = torch.randperm(num, generator=g, device="cuda")
    table = torch.full((len(lens), max(used + [1])), -7, dtype=torch.int32, device="cuda")
    out = []
    for _ in range(2):
        codes = torch.full((num, hk, page, d), 0x7f, dtype=torch.uint8, device="cuda")
        x = torch.randn(sum(lens), hk, d, generator=g, device="cuda").to(E4M3)
        s = torch.exp2(torch.randn(num, hk, generator=g, device="cuda")) if scales is None else scales(num, hk, g)
        dense = torch.empty(sum(lens), hk, d, dtype=torch.float64, device="cuda")
        pos = row = 0
        for i, n in enumerate(lens):
            mine = order[pos:pos + used[i]]
            table[i, :used[i]] = mine
            at = torch.arange(n, device="cuda")
            codes[mine[at // page], :, at % page] = x[row:row + n].view(torch.uint8)
            dense[row:row + n] = x[row:row + n].double() * s[mine[at // page]][..., None].double()
            pos, row = pos + used[i], row + n
        out.append((codes.view(E4M3), s, dense))
    (kp, ks, k), (vp, vs, v) = out
    return kp, vp, ks, vs, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), k, v


def close(o, lse, ref, rlse, dtype, d):
    assert torch.isfinite(o).all()
    for i in range(o.size(0)):  # every sequence for itself: a short one must not hide behind a long one
        assert (o[i].double() - ref[i]).norm() <= 2 * U[dtype] * ref[i].norm()
    live = rlse.T > float("-inf")
    assert torch.equal(lse > float("-inf"), live)
    # sums of exponentials (2e-5 of scores of some units), and the scores' own error: d / 16 truncating 32-bit
    # accumulations (2^-23 each) and four roundings (2^-24) of their size, which is about |lse|'s
    bound = 2e-5 + (2 * d / 16 + 4) * 2.0 ** -24 * rlse[rlse > float("-inf")].abs().max() if live.any() else 0
    assert not live.any() or (lse.double() - rlse.T)[live].abs().max() <= bound


def check8(lens, h, hk, d, page, dtype, window=None, sinks=0, scales=None, q_by=1.0, sm_scale=None):
    kp, vp, ks, vs, table, lengths, k, v = pool8(lens, hk, d, page, scales=scales)
    q = (torch.randn(len(lens), h, d, device="cuda", generator=gen(9)) * q_by).to(dtype)
    o, lse = paged_attention(q, kp, vp, table, lengths, k_scale=ks, v_scale=vs, window=window, sinks=sinks, return_lse=True,
                             sm_scale=sm_scale)
    ref, rlse = window_reference(q.double(), k, v, [1] * len(lens), lens, window or ALL, sinks, sm_scale or d ** -0.5)
    close(o, lse, ref, rlse, dtype, d)
    return q, kp, vp, ks, vs, table, lengths, o


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h, hk", [(4, 4), (8, 2), (8, 1), (5, 1), (16, 1), (24, 1), (18, 2), (1, 1)])
@pytest.mark.parametrize("d", [128, 64, 96, 48, 16])
def test_heads_and_types(h, hk, d, dtype):
    check8([1, 16, 201, 777, 64], h, hk, d, 16, dtype)


@pytest.mark.parametrize("page", [1, 7, 8, 24, 64, 100, 256])
@pytest.mark.parametrize("lens", [[1], [0], [0, 3, 0], [63, 64, 65, 127, 128, 129], [5000, 0, 17, 256, 257], [20000, 20000],
                                  [1] * 300, list(range(1, 130))])
def test_lengths_and_pages(lens, page):
    check8(lens, 4, 2, 64, page, torch.bfloat16)


def test_splits():
    check8([70000, 3, 0, 9000], 8, 2, 128, 32, torch.bfloat16)
    check8([40000, 30], 16, 1, 128, 64, torch.float16, window=30000, sinks=100)


@pytest.mark.parametrize("h, hk, d", [(8, 2, 128), (4, 4, 64), (16, 1, 128), (6, 3, 48)])
@pytest.mark.parametrize("lens", [[512], [513, 1], [640, 0, 200], [768] * 5, [1024, 1023] + [1000] * 40, [1500] * 30])
def test_whole_and_cut(lens, h, hk, d):
    """Short caches, whose items may stay in one block, and the same ones under a table with room for long ones."""
    q, kp, vp, ks, vs, table, lengths, o = check8(lens, h, hk, d, 16, torch.bfloat16)
    wide = torch.full((len(lens), 3000), -7, dtype=torch.int32, device="cuda")
    wide[:, :table.size(1)] = table
    scales = dict(k_scale=ks, v_scale=vs)
    o2, lse2 = paged_attention(q, kp, vp, wide, lengths, return_lse=True, **scales)
    _, lse = paged_attention(q, kp, vp, table, lengths, return_lse=True, **scales)
    # each within 2 u of what both stand for
    for a, b in zip(o, o2):
        assert (a.double() - b.double()).norm() <= 4 * U[torch.bfloat16] * a.double().norm()
    live = lse > float("-inf")
    assert torch.equal(live, lse2 > float("-inf")) and (lse - lse2)[live].abs().max() <= 1e-4


@pytest.mark.parametrize("page", [16, 8, 64])
def test_pages_of_very_different_scales(page):
    """A page whose values are 2^40 times another's, whichever of them is attended to: every sequence to full precision."""
    def wide(num, hk, g):
        return torch.exp2(torch.randint(-20, 21, (num, hk), generator=g, device="cuda").float())
    kp, vp, ks, vs, table, lengths, k, v = pool8([300, 77, 1000], 2, 64, page, scales=wide)
    ks.fill_(0.25)
    ks[:, 1] = 4.0  # sharp: a few tokens take all
    k, at = k * 0, 0
    for i, n in enumerate((300, 77, 1000)):
        t = torch.arange(n, device="cuda")
        pages = table[i].long()[t // page]
        k[at:at + n] = kp.view(torch.uint8)[pages, :, t % page].view(E4M3).double() * ks[pages][..., None].double()
        at += n
    q = torch.randn(3, 4, 64, device="cuda", generator=gen(3)).to(torch.float16)
    o, lse = paged_attention(q, kp, vp, table, lengths, k_scale=ks, v_scale=vs, return_lse=True)
    ref, rlse = window_reference(q.double(), k, v, [1] * 3, [300, 77, 1000], ALL, 0, 0.125)
    fits = ref.abs().amax(2) < 60000  # of fp16
    assert fits.any()
    for i, j in fits.nonzero().tolist():
        assert (o[i, j].double() - ref[i, j]).norm() <= 2 * U[torch.float16] * ref[i, j].norm()
    bound = 2e-5 + (2 * 64 / 16 + 4) * 2.0 ** -24 * rlse.abs().max()
    assert (lse.double() - rlse.T).abs().max() <= bound


def test_values_that_a_small_page_holds():
    """All weight on tokens of a page whose scale is 2^-30 of the others': they are the output, to full precision."""
    page, d, n = 16, 64, 128
    kp, vp, ks, vs, table, lengths, k, v = pool8([n], 1, d, page)
    small = table[0, 3].long()
    ks.fill_(1.0)
    ks[small] = 64.0
    vs.fill_(1.0)
    vs[small] = 2.0 ** -30
    kp.view(torch.uint8)[small] = torch.full((1, page, d), 2.0, device="cuda").to(E4M3).view(torch.uint8)
    q = torch.ones(1, 1, d, device="cuda", dtype=torch.bfloat16)
    o = paged_attention(q, kp, vp, table, lengths, k_scale=ks, v_scale=vs)
    want = vp[small].double().mean(1) * 2.0 ** -30
    assert (o[0].double() - want).norm() <= 2 * U[torch.bfloat16] * want.norm()


@pytest.mark.parametrize("q_by", [2.0 ** -100, 2.0 ** -10, 1.0, 2.0 ** 30, 2.0 ** 100])
def test_queries_of_any_size(q_by):
    """bf16 queries outside fp16's range: scaled on their way into the products, with scores of some units."""
    check8([200, 33], 8, 2, 64, 16, torch.bfloat16, q_by=q_by, sm_scale=0.125 / q_by)


def test_scales_of_zero_and_page_ids_outside():
    """Zero scales stand for zeros, page ids outside the pool read as zeros, lengths past the table are cut."""
    kp, vp, ks, vs, table, lengths, k, v = pool8([48], 1, 64, 16)
    q = torch.randn(1, 2, 64, device="cuda", generator=gen(1)).to(torch.bfloat16)
    call = lambda t, n, ks, vs: paged_attention(q, kp, vp, t, n, k_scale=ks, v_scale=vs, return_lse=True)  # noqa: E731
    bad = table.clone()
    bad[0, 1] = kp.size(0) + 5
    zk, zv = ks.clone(), vs.clone()
    zk[table[0, 1].long()], zv[table[0, 1].long()] = 0, 0
    k[16:32], v[16:32] = 0, 0
    ref, rlse = window_reference(q.double(), k, v, [1], [48], ALL, 0, 0.125)
    for t, a, b in ((bad, ks, vs), (table, zk, zv)):
        close(*call(t, lengths, a, b), ref, rlse, torch.bfloat16, 64)
    assert torch.equal(call(table, lengths + 1000, ks, vs)[0], call(table, lengths, ks, vs)[0])
    o, lse = call(table, lengths, torch.zeros_like(ks), torch.zeros_like(vs))
    assert not o.any() and (lse - torch.tensor(48.0).log().item()).abs().max() <= 2e-5


# ------------------------------------------------------------------------------------------ windows
def pool16(lens, hk, d, page, dtype, window, sinks):
    """16-bit pools in which all that the new token must not see is NaN or infinite, and the table names no page of it."""
    kp, vp, _, _, table, lengths, k, v = pool8(lens, hk, d, page)
    kp, vp = (torch.full(t.shape, float("nan"), device="cuda", dtype=dtype) for t in (kp, vp))
    row = 0
    for i, n in enumerate(lens):
        at = torch.arange(n, device="cuda")
        seen = visible(1, n, window, sinks, "cuda")[0] if n else at.bool()
        pages = table[i].long()[at // page]
        for pool, x in ((kp, k), (vp, v)):
            rows = x[row:row + n].to(dtype)
            x[row:row + n] = rows.double()
            rows[~seen] = float("inf")
            pool[pages, :, at % page] = rows
        for j in range(-(-n // page)):
            if not seen[j * page:(j + 1) * page].any():
                table[i, j] = -99 if j % 2 else 2 ** 30
        row += n
    return kp, vp, table, lengths, k, v


@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 40)])
@pytest.mark.parametrize("page", [1, 7, 8, 16, 24, 100, 256])
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (15, 3), (16, 16), (17, 100), (64, 0), (100, 64), (300, 65), (1000, 4),
                                           (2 ** 31, 2 ** 31), (5, 4000)])
def test_windows_16(window, sinks, page, dtype, d):
    lens = [1, 16, 17, 201, 777, 64, 0, 3000, 301, 320, 2]
    kp, vp, table, lengths, k, v = pool16(lens, 2, d, page, dtype, window, sinks)
    q = torch.randn(len(lens), 6, d, device="cuda", generator=gen(9)).to(dtype)
    o, lse = paged_attention(q, kp, vp, table, lengths, window=window, sinks=sinks, return_lse=True)
    ref, rlse = window_reference(q.double(), k.nan_to_num(), v.nan_to_num(), [1] * len(lens), lens, window, sinks, d ** -0.5)
    close(o, lse, ref, rlse, dtype, d)


@pytest.mark.parametrize("page", [1, 7, 16, 24, 64])
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (15, 3), (17, 100), (100, 64), (1000, 4), (2 ** 31, 2 ** 31)])
def test_windows_8(window, sinks, page):
    lens = [1, 16, 17, 201, 777, 64, 0, 3000, 301, 320, 2]
    kp, vp, ks, vs, table, lengths, k, v = pool8(lens, 2, 64, page)
    row = 0
    for i, n in enumerate(lens):  # NaN where nothing must be seen
        at = torch.arange(n, device="cuda")
        out = at[~visible(1, n, window, sinks, "cuda")[0]] if n else at
        for pool in (kp, vp):
            pool.view(torch.uint8)[table[i].long()[out // page], :, out % page] = 0x7f
        gone = [j for j in range(-(-n // page)) if j * page >= min(sinks, n) and (j + 1) * page <= n - window]
        for s in (ks, vs):
            s[table[i, gone].long()] = float("nan")
        table[i, gone] = 2 ** 30
        row += n
    q = torch.randn(len(lens), 6, 64, device="cuda", generator=gen(9)).to(torch.bfloat16)
    o, lse = paged_attention(q, kp, vp, table, lengths, k_scale=ks, v_scale=vs, window=window, sinks=sinks, return_lse=True)
    ref, rlse = window_reference(q.double(), k, v, [1] * len(lens), lens, window, sinks, 0.125)
    close(o, lse, ref, rlse, torch.bfloat16, 64)


def test_long_windows_and_splits_16():
    lens, window, sinks = [70000, 3, 0, 9000, 30000], 20000, 1000
    kp, vp, table, lengths, k, v = pool16(lens, 2, 128, 32, torch.bfloat16, window, sinks)
    q = torch.randn(len(lens), 8, 128, device="cuda", generator=gen(9)).to(torch.bfloat16)
    o, lse = paged_attention(q, kp, vp, table, lengths, window=window, sinks=sinks, return_lse=True)
    ref, rlse = window_reference(q.double(), k, v, [1] * len(lens), lens, window, sinks, 128 ** -0.5)
    close(o, lse, ref, rlse, torch.bfloat16, 128)


# ------------------------------------------------------------------------------------------ appending
def pow2(top):
    """The least power of two s >= 2^-126 with top <= 448 s, in 64 bits."""
    s = torch.exp2(torch.ceil(torch.log2(top.double() / 448)))
    s = torch.where(s / 2 * 448 >= top, s / 2, s)
    return torch.where(top > 0, s, 0.0).clamp_min(2.0 ** -126)


def append_reference(x, pool, scale, slots):
    """The rule of append_pages, page by page; `pool` as values of 8 bits in float64, `scale` float64."""
    page_size = pool.size(2)
    order = {}
    for row, s in enumerate(slots.tolist()):
        if 0 <= s < pool.size(0) * page_size:
            order.setdefault(s // page_size, []).append((row, s % page_size))
    for page, rows in order.items():
        r, at = (torch.tensor(t, device="cuda") for t in zip(*rows))
        new = x[r].double()
        finite = torch.where(torch.isfinite(new), new, 0.0)
        need = pow2(finite.abs().amax((0, 2)))
        if not (at == 0).any():
            old = scale[page]
            need = torch.maximum(old, need)
            pool[page] = (pool[page] * (old / need)[:, None, None]).float().to(E4M3).double()
        scale[page] = need
        quotient = (new / need[None, :, None]).float()
        quotient = torch.where(torch.isfinite(quotient), quotient, float("nan"))
        pool[page][:, at] = quotient.to(E4M3).double().transpose(0, 1)


def same(a, b):
    a, b = a.double(), b.double()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def runs(num, page, count, g, longest=None):
    """Slots of `count` runs, each of neighbouring slots of a page of its own, with skipped rows between."""
    out = []
    for p in torch.randperm(num, generator=g, device="cuda")[:count].tolist():
        n = int(torch.randint(1, min(page, longest or page) + 1, (1,), generator=g, device="cuda"))
        first = int(torch.randint(0, page - n + 1, (1,), generator=g, device="cuda"))
        out += [p * page + first + i for i in range(n)] + [-1] * (p % 3)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hk, page, d", [(2, 16, 128), (1, 1, 16), (3, 7, 48), (8, 24, 64), (2, 33, 80), (1, 64, 128), (2, 200, 96)])
def test_append(hk, page, d, dtype):
    """Rounds of runs of any sizes: new pages, pages that go on, pages whose scale grows or does not."""
    g, num = gen(1), 40
    shape = (num, hk, page, d)
    pools = [torch.randn(shape, generator=g, device="cuda").to(E4M3) for _ in range(2)]
    scales = [torch.zeros(num, hk, device="cuda") for _ in range(2)]
    want = [(p.double() * 0, s.double()) for p, s in zip(pools, scales)]
    for p in pools:
        p.view(torch.uint8).zero_()
    for turn in range(6):
        slots = runs(num, page, (3, 20, 40, 1, 30, 25)[turn], g, (None, 1, None, None, 3, None)[turn])
        by = torch.exp2(torch.randint(-6, 7, (2, len(slots), hk, 1), generator=g, device="cuda").float())
        new = [(torch.randn(len(slots), hk, d, generator=g, device="cuda") * b).to(dtype) for b in by]
        if turn == 4:
            new[0][::2] = 0
        append_pages(*new, *pools, slots, k_scale=scales[0], v_scale=scales[1])
        for x, (ref, sref), p, s in zip(new, want, pools, scales):
            append_reference(x, ref, sref, slots)
            assert torch.equal(s.double(), sref)
            # what a page holds that was begun anew is void
            assert same(p, ref)
    k, v = new
    wide = torch.zeros(len(slots), hk, 3 * d, device="cuda", dtype=dtype)
    wide[..., :d], wide[..., d:2 * d] = k, v
    views = [p.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(E4M3) for p in pools]
    other = [torch.stack([s, s], 2)[..., 0] for s in scales]
    append_pages(wide[..., :d], wide[..., d:2 * d], *views, slots, k_scale=other[0], v_scale=other[1])
    for a, b in zip(views + other, pools + scales):
        assert same(a, b)


@pytest.mark.parametrize("page", [16, 64, 256])
def test_append_long_runs(page):
    """Prompts: every page of them whole, the last in part, many rows a team."""
    g, lens, hk, d = gen(2), [5000, 1, 300, page, page + 1], 4, 128
    used = [-(-n // page) for n in lens]
    num = sum(used) + 3
    order = torch.randperm(num, generator=g, device="cuda")
    slots, pos = [], 0
    for n, u in zip(lens, used):
        at = torch.arange(n, device="cuda")
        slots.append(order[pos:pos + u][at // page] * page + at % page)
        pos += u
    slots = torch.cat(slots).to(torch.int32)
    new = [torch.randn(len(slots), hk, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)]
    pools = [torch.zeros(num, hk, page, d, dtype=E4M3, device="cuda") for _ in range(2)]
    scales = [torch.zeros(num, hk, device="cuda") for _ in range(2)]
    append_pages(*new, *pools, slots, k_scale=scales[0], v_scale=scales[1])
    for x, p, s in zip(new, pools, scales):
        ref, sref = p.double() * 0, s.double() * 0
        append_reference(x, ref, sref, slots)
        assert torch.equal(s.double(), sref) and same(p, ref)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_extremes(dtype, page):
    """Infinities, NaN, zeros, the types' largest and smallest values, 448 times a power of two, and scales that are none."""
    info, hk, d = torch.finfo(dtype), 2, 32
    x = torch.randn(8, hk, d, generator=gen(3), device="cuda").to(dtype)
    x[0, 0, 3], x[1, 0, 4], x[2, 1, 5], x[3, 1] = float("inf"), float("-inf"), float("nan"), 0
    x[4, 0, 0], x[5, 0, 0], x[6, 1, 0] = info.max, info.tiny, 448 * 4.0
    x[7] = info.smallest_normal * 2.0 ** -7
    for rows in ([0], [1], [2], [3], [4], [5], [6], [7], [0, 1, 2], [3, 7], list(range(8))):
        for old in (0.0, 2.0 ** -126, 1.0, 0.3, 2.0 ** 100):
            for first in (0, 5):
                codes = torch.randn(3, hk, page, d, generator=gen(4), device="cuda").to(E4M3)
                scale = torch.full((3, hk), old, device="cuda")
                pools, scales = [codes.clone(), codes.clone()], [scale.clone(), scale.clone()]
                slots = torch.arange(page + first, page + first + len(rows), dtype=torch.int32, device="cuda")
                # pages of 64: skipped rows behind, as many as make the call one whose runs are a block's each
                skipped = 2 * page if page == 64 else 0
                padded = torch.cat([slots, torch.full((skipped,), -1, dtype=torch.int32, device="cuda")])
                new = torch.cat([x[rows], x[:1].expand(skipped, hk, d)])
                append_pages(new, new, *pools, padded, k_scale=scales[0], v_scale=scales[1])
                ref, sref = codes.double(), scale.double()
                append_reference(x[rows], ref, sref, slots)
                for p, s in zip(pools, scales):
                    assert torch.equal(s.double(), sref) and same(p, ref)


def test_copies_take_the_scales_along():
    g, num = gen(5), 30
    pools = [torch.randn(num, 3, 10, 48, generator=g, device="cuda").to(E4M3) for _ in range(2)]
    scales = [torch.rand(num, 3, generator=g, device="cuda") for _ in range(2)]
    perm = torch.randperm(num, generator=g, device="cuda").to(torch.int32)
    src, dst = perm[:10], perm[10:20].clone()
    want = [t.view(torch.uint8).clone() if t.dtype == E4M3 else t.clone() for t in pools + scales]
    for i in range(10):
        if i != 3:
            for t in want:
                t[dst[i]] = t[src[i]]
    dst[3] = num  # outside: skipped
    copy_pages(*pools, src, dst, k_scale=scales[0], v_scale=scales[1])
    for t, w in zip(pools + scales, want):
        assert torch.equal(t.view(torch.uint8) if t.dtype == E4M3 else t, w)


def test_offsets_past_32_bits():
    """Pools of more than 2^32 elements, written, copied and read at their far end."""
    hk, page, d = 8, 128, 128
    num = 2 ** 32 // (hk * page * d) + 40
    kp, vp = (torch.zeros(num, hk, page, d, device="cuda", dtype=E4M3) for _ in range(2))
    ks, vs = torch.zeros(2, num, hk, device="cuda")
    n, g = 300, gen(0)
    k, v = (torch.randn(n, hk, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    pages = torch.tensor([num - 1, num - 7, num - 3], device="cuda")
    at = torch.arange(n, device="cuda")
    append_pages(k, v, kp, vp, (pages[at // page] * page + at % page).to(torch.int32), k_scale=ks, v_scale=vs)
    src = pages.to(torch.int32)
    copy_pages(kp, vp, src, src - 20, k_scale=ks, v_scale=vs)
    q = torch.randn(1, hk, d, generator=g, device="cuda").to(torch.bfloat16)
    dense = [(p.view(torch.uint8)[pages].view(E4M3).double() * s[pages][..., None, None].double()).transpose(1, 2).reshape(-1, hk, d)[:n]
             for p, s in ((kp, ks), (vp, vs))]
    # an e4m3 value is off by at most 2^-4 of itself, or, below 2^-6 of the scale's step, by 2^-10 of the scale (at most |x| max / 224)
    for x, y in zip((k, v), dense):
        assert ((x.double() - y).abs() <= x.double().abs() * 2.0 ** -4 + 2.0 ** -10 * x.double().abs().max() / 224).all()
    ref = window_reference(q.double(), *dense, [1], [n], ALL, 0, d ** -0.5)[0]
    for p in (src, src - 20):
        o = paged_attention(q, kp, vp, p[None], torch.tensor([n], dtype=torch.int32, device="cuda"), k_scale=ks, v_scale=vs)
        assert (o.double() - ref).norm() <= 2 * U[torch.bfloat16] * ref.norm()


# ------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("window, sinks", [(None, 0), (24, 5)])
def test_cache_prompt_then_tokens(window, sinks):
    """A prompt, then token by token with a fork on the way, over 8-bit pools: each output is the attention over what the
    cache holds, which is what was written up to its rounding."""
    h, hk, d, total = 8, 2, 64, 90
    q, k, v = (torch.randn(total, n, d, generator=gen(2), device="cuda").to(torch.bfloat16) for n in (h, hk, hk))
    cache = PagedKVCache(40, 16, hk, d, layers=2, dtype=E4M3)
    a = cache.add()
    slots = cache.reserve([a], [70])
    for layer in range(2):
        cache.write(layer, k[:70], v[:70], slots)
    if window:
        packed_attention(q[:70], k[:70], v[:70], PackedSequences([70]), causal=True, window=window, sinks=sinks)

    def held(layer, seq):
        at = torch.arange(cache.length(seq), device="cuda")
        pages = torch.tensor(cache.pages(seq), device="cuda")[at // 16]
        return [p[layer].view(torch.uint8)[pages, :, at % 16].view(E4M3).double() * s[layer][pages][..., None].double()
                for p, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    b = cache.fork(a)
    for t in range(70, total):
        slots = cache.reserve([a, b], [1, 1])
        table, lengths = cache.tables([a, b])
        for layer in range(2):
            cache.write(layer, torch.stack([k[t], -k[t] * 3]), torch.stack([v[t], -v[t] * 3]), slots)
            o = cache.attend(layer, q[[t, t]], table, lengths, window=window, sinks=sinks)
            for i, seq in enumerate((a, b)):
                ref = window_reference(q[t:t + 1].double(), *held(layer, seq), [1], [t + 1], window or ALL, sinks, d ** -0.5)[0]
                assert (o[i].double() - ref[0]).norm() <= 2 * U[torch.bfloat16] * ref.norm()
    for i, (seq, by) in enumerate(((a, 1), (b, -3))):
        for x, y in zip((k, v), held(1, seq)):
            x = torch.cat([x[:70], x[70:] * by]).double()
            # two roundings to 4 significant bits at most: one more where a page grew and its values became subnormal
            assert ((x - y).abs() <= x.abs() * 2.0 ** -4 + 2 * 2.0 ** -10 * x.abs().max() / 224).all()
    cache.free(a)
    cache.compact()
    table, lengths = cache.tables([b])
    assert torch.equal(cache.attend(1, q[-1:], table, lengths, window=window, sinks=sinks)[0], o[1])


@pytest.mark.parametrize("window", [None, 100])
def test_stream_graph_and_changing_lengths(window):
    """A step that appends and attends, captured once and replayed with other rows, slots and lengths."""
    kp, vp, ks, vs, table, lengths, k, v = pool8([3000, 500], 2, 64, 16)
    for p in (kp, vp):
        u = p.view(torch.uint8)
        u[u == 0x7f] = 0
    q, x = torch.randn(2, 8, 64, device="cuda").to(torch.bfloat16), torch.randn(2, 2, 64, device="cuda").to(torch.bfloat16)
    live, slots = lengths.clone(), torch.zeros(2, dtype=torch.int32, device="cuda")
    first = [t.view(torch.uint8).clone() if t.dtype == E4M3 else t.clone() for t in (kp, vp, ks, vs)]

    def restore():
        for t, f in zip((kp, vp, ks, vs), first):
            (t.view(torch.uint8) if t.dtype == E4M3 else t).copy_(f)

    def step():
        append_pages(x, -x, kp, vp, slots, k_scale=ks, v_scale=vs)
        return paged_attention(q, kp, vp, table, live, k_scale=ks, v_scale=vs, window=window, sinks=3 if window else 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for a, b in ((3000, 500), (1, 1), (2999, 17), (64, 448)):
        live.copy_(torch.tensor([a, b], dtype=torch.int32))
        last = live.long() - 1
        slots.copy_(table.gather(1, (last // 16)[:, None])[:, 0] * 16 + (last % 16).int())
        x.normal_(generator=gen(a))
        restore()
        graph.replay()
        got, pages = out.clone(), [t.view(torch.uint8).clone() if t.dtype == E4M3 else t.clone() for t in (kp, vp, ks, vs)]
        restore()
        assert torch.equal(step(), got)
        for t, w in zip((kp, vp, ks, vs), pages):
            assert torch.equal(t.view(torch.uint8) if t.dtype == E4M3 else t, w)


def test_refusals():
    kp, vp, ks, vs, table, lengths, k, v = pool8([40], 2, 64, 16)
    q = torch.zeros(1, 4, 64, device="cuda", dtype=torch.bfloat16)
    ok = dict(q=q, k_pages=kp, v_pages=vp, page_table=table, lengths=lengths, k_scale=ks, v_scale=vs)
    for bad in (dict(k_scale=None), dict(v_scale=None), dict(k_scale=None, v_scale=None), dict(k_scale=ks[:-1]), dict(k_scale=ks.double()),
                dict(v_scale=vs.cpu()), dict(q=q.float()), dict(v_pages=vp.to(torch.bfloat16)),
                dict(k_pages=kp.to(torch.bfloat16), v_pages=vp.to(torch.bfloat16)), dict(window=0), dict(window=3, sinks=-1), dict(sinks=1),
                dict(k_pages=kp[..., :40], v_pages=vp[..., :40], q=q[..., :40]), dict(q=q[..., :32])):
        with pytest.raises(AssertionError):
            paged_attention(**{**ok, **bad})
    rows, slots = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32, device="cuda")
    for args, kw in (((rows, rows, kp, vp, slots), {}), ((rows, rows.half(), kp, vp, slots), dict(k_scale=ks, v_scale=vs)),
                     ((rows.float(), rows.float(), kp, vp, slots), dict(k_scale=ks, v_scale=vs)),
                     ((rows, rows, kp, vp, slots), dict(k_scale=ks, v_scale=vs[:1])), ((kp[0], vp[0], kp, vp, slots), dict(k_scale=ks, v_scale=vs))):
        with pytest.raises(AssertionError):
            append_pages(*args, **kw)
    with pytest.raises(AssertionError):
        copy_pages(kp, vp, slots, slots)
    wide = ks[:1].expand(ks.shape)  # may be read, but not written
    paged_attention(**{**ok, "k_scale": wide})
    with pytest.raises(AssertionError, match="expanded"):
        append_pages(rows, rows, kp, vp, slots, k_scale=wide, v_scale=vs)
    with pytest.raises(AssertionError, match="expanded"):
        copy_pages(kp, vp, slots, slots, k_scale=ks, v_scale=wide)
