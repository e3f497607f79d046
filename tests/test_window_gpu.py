"""Attention over packed sequences with a window and sinks against its definition in 64 bits.

Errors are relative in the Frobenius norm, in units u of half a rounding step (2^-8 for bf16, 2^-11 for fp16). Forward:
P rounded (u) and the output rounded (u): at most 2 u. Gradients: dS or P rounded (u), the rounding of P inside the o of
D = sum o dO (u, relative to |o| |dO|, which cancellation in dP - D can double), the output rounded (u): at most 4 u. Where a
reference is zero the result must be.
"""
import pytest
import torch

from vmonarch_b200 import PackedSequences, packed_attention
from window_reference import visible, window_reference

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
CASES = [  # lengths, keys, window, sinks, heads, key heads
    ([130], None, 20, 4, 4, 2), ([1, 0, 300, 7], None, 64, 0, 4, 1), ([700], None, 128, 128, 2, 1), ([700], None, 129, 127, 2, 2),
    ([5, 200, 300, 700], [9, 100, 1, 900], 100, 30, 2, 1),   # sequences whose first queries see no key
    ([31, 33, 65, 1], [32, 33, 64, 129], 1, 0, 2, 2), ([31, 33, 65, 1], [32, 33, 64, 129], 1, 1, 2, 2),
    ([2], [5000], 300, 200, 4, 1), ([64], [3000], 1000, 4, 8, 2), ([5000], [2], 1, 3, 4, 1), ([1], None, 1, 0, 1, 1),
    ([3, 4], [0, 0], 2, 2, 2, 1), ([900], None, 2, 600, 2, 1), ([900], None, 10 ** 12, 5, 2, 1), ([300, 1000], [600, 1000], 255, 10 ** 12, 2, 1),
]


def make(ql, kl, h, hk, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n, h: torch.randn(n, h, d, generator=g, device="cuda").to(dtype)  # noqa: E731
    return r(sum(ql), h), r(sum(kl), hk), r(sum(kl), hk), r(sum(ql), h)


def rel(x, ref):
    x, ref = x.double(), ref.double()
    assert torch.isfinite(x).all()
    return ((x - ref).norm() / ref.norm()).item() if ref.norm() > 0 else x.abs().max().item() if x.numel() else 0.0


def grads(fn, leaves, do):
    leaves = [t.detach().requires_grad_() for t in leaves]
    o = fn(*leaves)
    return [o.detach()] + list(torch.autograd.grad(o, leaves, do.to(o.dtype), allow_unused=True))


def own(seqs, window, sinks, **kw):
    return lambda *x: packed_attention(*x, seqs, causal=True, window=window, sinks=sinks, **kw)


def compare(ql, kl, window, sinks, h, hk, d, dtype, scale=None):
    kl = ql if kl is None else kl
    q, k, v, do = make(ql, kl, h, hk, d, dtype)
    seqs = PackedSequences(ql, kl)
    scale = d ** -0.5 if scale is None else scale
    got = grads(own(seqs, window, sinks, sm_scale=scale), (q, k, v), do)
    want = grads(lambda *x: window_reference(*x, ql, kl, window, sinks, scale)[0], [t.double() for t in (q, k, v)], do)
    want = [torch.zeros_like(g) if w is None else w for g, w in zip(got, want)]
    for x, ref, bound in zip(got, want, (2, 4, 4, 4)):
        assert rel(x, ref) <= bound * U[dtype]
    with torch.no_grad():
        o, lse = own(seqs, window, sinks, sm_scale=scale, return_lse=True)(q, k, v)
    assert torch.equal(o, got[0])
    ref = window_reference(q.double(), k.double(), v.double(), ql, kl, window, sinks, scale)[1]
    assert torch.equal(lse == float("-inf"), ref == float("-inf"))
    # scores of a few units, accumulated in 32 bits: 1e-5 is some twenty of their roundings
    assert (lse.double() - ref)[ref > float("-inf")].abs().max().item() <= 1e-5 if (ref > float("-inf")).any() else True


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [128, 64, 40])
@pytest.mark.parametrize("ql, kl, window, sinks, h, hk", CASES)
def test_forward_and_gradients(ql, kl, window, sinks, h, hk, d, dtype):
    compare(ql, kl, window, sinks, h, hk, d, dtype)


@pytest.mark.parametrize("window", [1, 63, 64, 65, 127, 128, 129, 200, 256, 257, 383, 384, 700])
@pytest.mark.parametrize("sinks", [0, 1, 64, 129, 300])
def test_edges_of_tiles(window, sinks):
    """Windows and sinks around the tiles' sizes, also where the two meet."""
    compare([777, 1, 256], [777, 200, 300], window, sinks, 2, 1, 64, torch.bfloat16)


def test_cut_units():
    """Few long sequences: units are cut inside the window, and inside the sinks, and joined."""
    for mask in ((6000, 300), (300, 6000), (9000, 4)):
        compare([20, 300], [9500, 300], *mask, 1, 1, 128, torch.bfloat16)
    compare([6200], None, 2500, 130, 1, 1, 128, torch.bfloat16)


def test_a_long_window_is_causal_attention():
    """Where the window takes in everything: the same but for the order of 64 numbers' sum (64 roundings of 2^-24, so 2^-18 of l,
    lse and what is made of them), which moves a result to its neighbour at most: one step, 2 u."""
    q, k, v, do = make([300, 40], [300, 700], 4, 2, 64, torch.bfloat16)
    seqs = PackedSequences([300, 40], [300, 700])
    want = grads(lambda *x: packed_attention(*x, seqs, causal=True), (q, k, v), do)
    for window, sinks in ((700, 0), (699, 1), (10 ** 12, 3)):
        for a, b in zip(grads(own(seqs, window, sinks), (q, k, v), do), want):
            assert rel(a, b) <= 2 * U[torch.bfloat16]


@pytest.mark.parametrize("scale", [0.0, 3.0])
def test_scales(scale):
    """Uniform weights, and scores spread over hundreds (the reference is raised many times, also from none)."""
    q, k, v, _ = make([900], [900], 2, 1, 64, torch.float16)
    o = own(PackedSequences([900]), 70, 5, sm_scale=scale)(q, k, v)
    assert rel(o, window_reference(q.double(), k.double(), v.double(), [900], [900], 70, 5, scale)[0]) <= 2 * U[torch.float16]


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq, nk, window, sinks", [(700, 700, 100, 20), (700, 700, 300, 0), (385, 640, 256, 129)])
def test_values_a_query_does_not_see(nq, nk, window, sinks, d, bad):
    """A value that is not finite reaches the queries that see it, and no other."""
    q, k, v, _ = make([nq], [nk], 4, 2, d, torch.bfloat16)
    fn = own(PackedSequences([nq], [nk]), window, sinks)
    clean = fn(q, k, v)
    seen = visible(nq, nk, window, sinks, "cuda")
    for at in (0, 3, 19, 20, 127, 128, 130, 255, 256, 300, nk - 200, nk - 129, nk - 1):
        w = v.clone()
        w[at, 1, 5] = bad
        w[at, 1, d - 1] = bad
        hit = torch.zeros_like(clean, dtype=torch.bool)
        hit[seen[:, at], 2:, 5] = True
        hit[seen[:, at], 2:, d - 1] = True
        for _ in range(3):
            o = fn(q, k, w)
            assert torch.equal(o[~hit], clean[~hit])
            assert torch.isnan(o[hit]).all() if bad != bad else (o[hit] == bad).all()
        # and a key: the queries that do not see it are as they were, up to rounding: 32 queries raise their softmax's reference
        # together, so one that sees the key changes the power of two against which its neighbours' P is rounded. Both results
        # are within 2 u of the exact one, so within 4 u of one another.
        x = k.clone()
        x[at, 1] = bad
        o = fn(q, x, v)
        assert rel(o[~seen[:, at]], clean[~seen[:, at]]) <= 4 * U[torch.bfloat16] and torch.equal(o[:, :2], clean[:, :2])


@pytest.mark.parametrize("d", [64, 128])
def test_other_sequences_take_no_part(d):
    """Infinities and NaN in the rows of another sequence, in all four tensors: nothing changes."""
    ql, kl = [70, 45, 300], [129, 45, 430]
    q, k, v, do = make(ql, kl, 4, 2, d, torch.bfloat16)
    fn = own(PackedSequences(ql, kl), 100, 7)
    clean = grads(fn, (q, k, v), do)
    bad = [t.clone() for t in (q, k, v, do)]
    for t, n0, n in ((bad[0], 70, 45), (bad[1], 129, 45), (bad[2], 129, 45), (bad[3], 70, 45)):
        t[n0:n0 + n:2] = float("nan")
        t[n0 + 1:n0 + n:2] = float("inf")
    dirty = grads(fn, bad[:3], bad[3])
    for c, x, (n0, n) in zip(clean, dirty, ((70, 45), (70, 45), (129, 45), (129, 45))):
        assert torch.equal(c[:n0], x[:n0]) and torch.equal(c[n0 + n:], x[n0 + n:])


def test_keys_out_of_sight_get_no_gradient():
    """Keys behind every query's window: zeros, not what was in the memory."""
    q, k, v, do = make([40], [2000], 2, 1, 64, torch.bfloat16)
    seqs = PackedSequences([40], [2000])
    junk = [torch.full((2000, 1, 64), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(8)]
    del junk
    _, _, dk, dv = grads(own(seqs, 100, 10), (q, k, v), do)
    for t in (dk, dv):
        assert not t[10:1861].any() and t[:10].any() and t[1861:].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_window_of_one_key_passes_no_score_gradient(dtype):
    q, k, v, do = make([300, 4], [300, 9], 4, 2, 64, dtype)
    o, dq, dk, dv = grads(own(PackedSequences([300, 4], [300, 9]), 1, 0), (q, k, v), do)
    assert not dq.any() and not dk.any() and dv.any()
    assert torch.equal(o[:300], v[:300].repeat_interleave(2, 1))


def test_gradient_against_differences():
    """sum(o w) along the gradient: its difference between the ends of a path is the sum over the path's pieces of
    (x+ - x-) . (g(x+) + g(x-)) / 2. The outputs' rounding (u |o| |w|, random) is below 2 % over the path taken; sixteen
    pieces leave the trapezoids' own error, which falls with their square, below that."""
    ql, kl = [170, 33], [170, 90]
    q, k, v, w = make(ql, kl, 4, 2, 64, torch.float16, seed=3)
    fn = own(PackedSequences(ql, kl), 40, 6)
    base = grads(fn, (q, k, v), w)[1:]
    for i in range(3):
        step = 0.1 * base[i].float() / base[i].float().pow(2).mean().sqrt()
        points = []
        for piece in range(17):
            x = [q, k, v]
            x[i] = (x[i].float() + (1 - piece / 8) * step).half()
            r = grads(fn, x, w)
            points.append((x[i].double(), (r[0].double() * w.double()).sum(), r[1 + i].double()))
        predicted = sum(((a[0] - b[0]) * (a[2] + b[2])).sum() / 2 for a, b in zip(points, points[1:]))
        assert abs((points[0][1] - points[-1][1] - predicted) / predicted) <= 0.02


def test_strides_streams_and_captured_steps():
    """Slices of one QKV projection, another stream, and a captured step on new values: the same bits."""
    n = [200, 3, 700]
    q, k, v, do = make(n, n, 4, 4, 64, torch.bfloat16)
    seqs = PackedSequences(n)
    fn = own(seqs, 150, 9)
    want = grads(fn, (q, k, v), do)
    for a, b in zip(grads(fn, torch.stack([q, k, v], 1).unbind(1), do), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = grads(fn, (q, k, v), do)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    leaves = [t.clone().requires_grad_() for t in make(n, n, 4, 4, 64, torch.bfloat16, seed=5)[:3]]

    def step():
        o = fn(*leaves)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        for t, x in zip(leaves, (q, k, v)):
            t.copy_(x)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, want):
        assert torch.equal(a, b)
