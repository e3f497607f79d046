"""Paged attention over 8-bit pools where the weights of a call reach over many powers of two: a key that takes nearly all but has
small or no values, and pages whose value scales differ widely, column by column.

A weight P (that of a value, with its scale) is rounded to fp16's 11 bits, or to more, and the output to its type (u): every element is
off by at most (2^-11 + u) sum p |v|, whatever the other elements are, and by the error of the exponents: per score d / 16 truncating
32-bit accumulations (2^-23 each) and four roundings (2^-24) of its size, five roundings of the logarithm of the value scale, and
2e-5 for two exponentials and a logarithm; the sum below the line has as much again."""
import pytest
import torch

from vmonarch_b200 import paged_attention

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def codes(x):
    return x.to(E4M3).view(torch.uint8)


def pools(n, hk, d, page, seed=0):
    """One sequence of n tokens: 8-bit pools of its pages in order, as bytes, and scales of one."""
    g, num = gen(seed), -(-n // page)
    k, v = (codes(torch.randn(num, hk, page, d, generator=g, device="cuda")) for _ in range(2))
    ks, vs = torch.ones(2, num, hk, device="cuda")
    return k, v, ks, vs, torch.arange(num, dtype=torch.int32, device="cuda")[None]


def tokens(pool, scale, n):
    """What a pool's n tokens stand for, (n, hk, d) in 64 bits."""
    x = pool.view(E4M3).double() * scale[..., None, None].double()
    return x.transpose(1, 2).reshape(-1, x.size(1), x.size(3))[:n]


def check(q, k, v, ks, vs, table, n, sm_scale, window=None, sinks=0):
    """q (H, d) over the first n tokens, element by element. Returns the reference and what it is a part of, sum p |v|."""
    dtype, d = q.dtype, q.size(1)
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    o, lse = paged_attention(q[None], k.view(E4M3), v.view(E4M3), table, lengths, k_scale=ks, v_scale=vs, sm_scale=sm_scale,
                             window=window, sinks=sinks, return_lse=True)
    group = q.size(0) // k.size(1)
    kk, vv = (tokens(p, s, n).repeat_interleave(group, 1) for p, s in ((k, ks), (v, vs)))
    s = torch.einsum("hd,thd->ht", q.double(), kk) * sm_scale
    if window is not None:
        t = torch.arange(n, device="cuda")
        s[:, ~((t >= n - window) | (t < sinks))] = float("-inf")
    rlse = torch.logsumexp(s, 1)
    p = torch.exp(s - rlse[:, None])
    ref, size = torch.einsum("ht,thd->hd", p, vv), torch.einsum("ht,thd->hd", p, vv.abs())
    most = s[s > float("-inf")].abs().max()
    exponents = 2e-5 + (2 * d / 16 + 4) * 2.0 ** -24 * most
    scale = 5 * 2.0 ** -24 * vs[vs > 0].log2().abs().max()
    assert torch.isfinite(o).all()
    # (elements at the end of the output's range are off by half of its smallest step)
    step = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bound = (2.0 ** -11 + U[dtype] + 2 * exponents + scale) * size + step / 2
    off = (o[0].double() - ref).abs()
    assert (off <= bound).all(), (off / bound).max().item()
    assert (lse[0].double() - rlse).abs().max() <= exponents
    return ref, size


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h, hk, d", [(4, 1, 128), (8, 2, 64), (16, 1, 64), (18, 1, 128), (1, 1, 16)])
@pytest.mark.parametrize("nats", [3, 9, 17, 40, 80])
@pytest.mark.parametrize("window, sinks", [(None, 0), (3000, 4)])
def test_a_key_that_takes_all_but_has_no_value(window, sinks, nats, h, hk, d, dtype):
    """The first token is `nats` above thousands of others, and has a value of 0 in its even columns, of 2^-9 in the odd ones."""
    n, page = 4099, 16
    k, v, ks, vs, table = pools(n, hk, d, page)
    q = torch.zeros(h, d, device="cuda", dtype=dtype)
    q[:, 0] = 1.0
    k[..., 0] = codes(torch.randn(k.shape[:3], generator=gen(1), device="cuda").clamp(-2, 2))
    k[0, :, 0, 0] = codes(torch.tensor(256.0, device="cuda"))
    v[0, :, 0] = codes(torch.zeros(d, device="cuda"))
    v[0, :, 0, 1::2] = 1
    ref, size = check(q, k, v, ks, vs, table, n, nats / 256, window, sinks)
    assert (ref[:, 0::2] != 0).all()


@pytest.mark.parametrize("dtype, log, low", [(torch.bfloat16, 10, -20), (torch.bfloat16, 20, -20), (torch.bfloat16, 45, -20),
                                             (torch.bfloat16, 75, -100), (torch.bfloat16, 100, -100), (torch.float16, 10, -3),
                                             (torch.float16, 20, -13), (torch.float16, 27, -20)])  # (fp16 holds no wider ones)
@pytest.mark.parametrize("d, page", [(64, 16), (128, 64), (128, 8), (32, 1)])
def test_columns_of_pages_with_other_scales(d, page, dtype, log, low):
    """Scores alike; every other page has a scale 2^log times the others', and nothing but zeros in every fourth column."""
    n = 400
    k, v, ks, vs, table = pools(n, 1, d, page)
    vs[::2] = 2.0 ** low
    vs[1::2] = 2.0 ** (low + log)
    v[1::2, ..., 1::4] = 0
    q = torch.zeros(3, d, device="cuda", dtype=dtype)
    ref, size = check(q, k, v, ks, vs, table, n, 1.0)
    assert (ref[:, 1::4].abs() < 2.0 ** (low + 6)).all() and (ref[:, 1::4] != 0).all()


def test_one_and_a_half():
    """Two pages alike in score, one of 2^30 with a zero in column 1, one of 1 with a 3: the mean is 1.5."""
    k, v, ks, vs, table = pools(32, 1, 64, 16)
    v[0, ..., 1], v[1, ..., 1] = 0, codes(torch.tensor(3.0, device="cuda"))
    vs[0], vs[1] = 2.0 ** 30, 1.0
    for dtype in U:
        o = paged_attention(torch.zeros(1, 1, 64, device="cuda", dtype=dtype), k.view(E4M3), v.view(E4M3), table,
                            torch.tensor([32], dtype=torch.int32, device="cuda"), k_scale=ks, v_scale=vs)
        assert o[0, 0, 1] == 1.5


@pytest.mark.parametrize("h, hk, d", [(2, 1, 128), (12, 1, 64), (6, 3, 48)])
@pytest.mark.parametrize("spread", [4, 20, 60])
def test_weights_of_every_size(spread, h, hk, d):
    """Scores that grow or fall by `spread` nats over the sequence, or lie at random in that range, with scales of any kind (no powers
    of two) and values of zero in many places."""
    n, page = 9000, 24
    for order in ("up", "down", "any"):
        k, v, ks, vs, table = pools(n, hk, d, page, 3)
        num = ks.size(0)
        step = torch.linspace(-1, 1, num, device="cuda")
        step = step if order == "up" else -step if order == "down" else step[torch.randperm(num, generator=gen(5), device="cuda")]
        k[..., 0] = codes(torch.ones((), device="cuda"))
        k[..., 1:] = 0
        q = torch.zeros(h, d, device="cuda", dtype=torch.bfloat16)
        q[:, 0] = torch.where(torch.arange(h, device="cuda") % 2 == 0, 1.0, -1.0)
        ks[:] = (step[:, None] + 1.001) * 1.3
        vs[:] = torch.exp(torch.randn(vs.shape, generator=gen(6), device="cuda") * 8)
        v[torch.rand(v.shape, generator=gen(7), device="cuda") < 0.5] = 0
        check(q, k, v, ks, vs, table, n, spread / 2.6)


@pytest.mark.parametrize("log", [119, 118, -126, -120])
def test_scales_at_the_ends(log):
    """Value scales at the ends of what appending makes: outputs near bf16's largest and smallest normal values."""
    k, v, ks, vs, table = pools(3, 1, 64, 16)
    vs.fill_(2.0 ** log)
    v[0, 0, :, :4] = torch.tensor([0x7e, 0xfe, 0, 0x38], dtype=torch.uint8, device="cuda")  # 448, -448, 0, 1
    if log > 0:
        v[0, 0, :, 4:] = 0x48
        v[0, 0, 1:, :2] = 0  # (sums have 32 bits as well)
    check(torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16), k, v, ks, vs, table, 3, 1.0)


def test_unseen_and_not_a_number_beside_small_weights():
    """Slots past the length hold NaN, a page has scales of zero, a page lies outside: none of it reaches the small weights' columns."""
    n, page = 100, 16
    k, v, ks, vs, table = pools(n, 1, 64, page)
    q = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16)
    q[:, 0] = 1.0
    k[..., 0] = 0
    k[1, :, 3, 0] = codes(torch.tensor(256.0, device="cuda"))
    v[1, :, 3] = 0
    k[6, :, 4:], v[6, :, 4:] = 0x7f, 0x7f
    ks[2], vs[2] = 0, 0
    check(q, k, v, ks, vs, table, n, 30 / 256)
    k[4], v[4] = 0, 0
    far = table.clone()
    far[0, 4] = 10 ** 6
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    a, b = (paged_attention(q[None], k.view(E4M3), v.view(E4M3), t, lengths, k_scale=ks, v_scale=vs, sm_scale=30 / 256) for t in (table, far))
    assert torch.equal(a, b) and torch.isfinite(a).all()
