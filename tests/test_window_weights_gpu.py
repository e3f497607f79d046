"""Attention with a window and sinks in fp16 where a sink takes nearly all of the weight but has no value, so that the output is the
sum of small weights: packed and over a cache of 16 bits, element by element against the definition in 64 bits.

A weight P is rounded to fp16's 11 bits, but never in steps below 2^-31 of the largest weight, and the output to fp16: every element is
off by at most 2 x 2^-11 sum p |v| + 2^-32 max p sum |v|. To that come the exponents: d / 16 truncating 32-bit accumulations (2^-23
each) and four roundings (2^-24) of a score's size, and 2e-5, once above the line and once below. In bf16 P has the exponents of 32
bits: 2 x 2^-8 sum p |v|."""
import pytest
import torch

from vmonarch_b200 import PackedSequences, packed_attention, paged_attention
from window_reference import visible

pytestmark = pytest.mark.gpu
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def rows(n, h, d, seed, dtype):
    return torch.randn(n, h, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def bounds(q, k, v, seen, sm_scale, dtype):
    """(output, what it may be off by) of queries (n, H, D) that see keys (m, D) where `seen` (n, m) says."""
    s = torch.einsum("nhd,md->nhm", q.double(), k.double()) * sm_scale
    s = torch.where(seen[:, None], s, float("-inf"))
    p = torch.softmax(s, -1)
    size = torch.einsum("nhm,md->nhd", p, v.double().abs())
    exponents = 2e-5 + (2 * q.size(2) / 16 + 4) * 2.0 ** -24 * s[s > float("-inf")].abs().max()
    off = (2 * U[dtype] + 2 * exponents) * size
    if dtype == torch.float16:
        off = off + 2.0 ** -32 * p.amax(-1, keepdim=True) * torch.einsum("nm,md->nd", seen.double(), v.double().abs())[:, None] + 2.0 ** -25
    return torch.einsum("nhm,md->nhd", p, v.double()), off


def sink(n, d, dtype):
    """Keys and values of n tokens whose first is far above the others, for queries of (1, 0, 0 ...)."""
    k, v = rows(n, 1, d, 1, dtype)[:, 0], rows(n, 1, d, 2, dtype)[:, 0] * 512  # (small weights stay above fp16's smallest values)
    k[:, 0].clamp_(-2, 2)
    k[0, 0], v[0] = 256.0, 0.0
    return k, v


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nats", [3, 9, 12, 15, 17])
@pytest.mark.parametrize("nq, n, window, sinks", [(300, 300, 100, 4), (40, 3000, 1000, 1), (700, 1500, 260, 130), (1, 5000, 4000, 33)])
def test_packed(nq, n, window, sinks, nats, d, dtype):
    k, v = sink(n, d, dtype)
    q = rows(nq, 3, d, 3, dtype) * 0
    q[..., 0] = 1.0
    o = packed_attention(q, k[:, None], v[:, None], PackedSequences([nq], [n]), causal=True, window=window, sinks=sinks, sm_scale=nats / 256)
    ref, off = bounds(q, k, v, visible(nq, n, window, sinks, "cuda"), nats / 256, dtype)
    assert ((o.double() - ref).abs() <= off).all(), ((o.double() - ref).abs() / off).max().item()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h, d, page", [(4, 128, 16), (8, 64, 7), (16, 64, 64), (20, 40, 16)])
@pytest.mark.parametrize("nats", [3, 9, 15, 17, 20])
@pytest.mark.parametrize("n, window, sinks", [(77, 50, 1), (3000, 1000, 1), (9000, 8000, 40)])
def test_cached(n, window, sinks, nats, h, d, page, dtype):
    k, v = sink(n, d, dtype)
    num = -(-n // page)
    kp, vp = (torch.zeros(num, page, d, device="cuda", dtype=dtype) for _ in range(2))
    kp.view(-1, d)[:n], vp.view(-1, d)[:n] = k, v
    q = torch.zeros(1, h, d, device="cuda", dtype=dtype)
    q[..., 0] = 1.0
    table, lengths = torch.arange(num, dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda")
    o = paged_attention(q, kp[:, None], vp[:, None], table, lengths, window=window, sinks=sinks, sm_scale=nats / 256)
    ref, off = bounds(q, k, v, visible(1, n, window, sinks, "cuda"), nats / 256, dtype)
    assert ((o.double() - ref).abs() <= off).all(), ((o.double() - ref).abs() / off).max().item()
