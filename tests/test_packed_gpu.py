"""Attention over packed sequences against its definition in 64 bits.

Errors are relative in the Frobenius norm, in units u of 2^-9 for bf16 (half of a rounding's
bound, above its root mean square) and 2^-11 for fp16. Forward: P rounded (u) and the output rounded (u): at most 2 u. Gradients: dS
or P rounded (u), the rounded o inside D = sum o dO (u, relative to |o| |dO|, which cancellation in
dP - D can double), the output rounded (u): at most 4 u. Where a reference is zero the result must be.
"""
import pytest
import torch

from packed_reference import packed_reference
from vmonarch_b200 import PackedSequences, packed_attention

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11}
CASES = [
    ([130], None, True, 4, 2), ([1, 0, 300, 7], None, True, 4, 1),
    ([1, 5, 257, 128, 513], [0, 200, 31, 128, 600], False, 3, 3),
    ([5, 200, 300, 700], [9, 100, 1, 900], True, 2, 1),   # sequences whose first queries see no key
    ([1000], None, False, 8, 2), ([31, 33, 65, 1], [32, 33, 64, 129], True, 2, 2),
    ([2], [5000], True, 4, 1), ([5000], [2], False, 4, 1), ([1], None, True, 1, 1), ([3, 4], [0, 0], False, 2, 1),
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [128, 64, 96, 40, 8])
@pytest.mark.parametrize("ql, kl, causal, h, hk", CASES)
def test_forward_and_gradients(ql, kl, causal, h, hk, d, dtype):
    kl = ql if kl is None else kl
    q, k, v, do = make(ql, kl, h, hk, d, dtype)
    seqs = PackedSequences(ql, kl)
    got = grads(lambda *x: packed_attention(*x, seqs, causal=causal), (q, k, v), do)
    want = grads(lambda *x: packed_reference(*x, ql, kl, causal, d ** -0.5)[0], [t.double() for t in (q, k, v)], do)
    want = [torch.zeros_like(g) if w is None else w for g, w in zip(got, want)]
    for x, ref, bound in zip(got, want, (2, 4, 4, 4)):
        assert rel(x, ref) <= bound * U[dtype]
    # without gradients, and the statistics
    with torch.no_grad():
        o, lse = packed_attention(q, k, v, seqs, causal=causal, return_lse=True)
    assert torch.equal(o, got[0])
    ref = packed_reference(q.double(), k.double(), v.double(), ql, kl, causal, d ** -0.5)[1]
    assert torch.equal(lse == float("-inf"), ref == float("-inf"))
    # scores of a few units, accumulated in 32 bits: 1e-5 is some twenty of their roundings
    assert (lse.double() - ref)[ref > float("-inf")].abs().max().item() <= 1e-5 if (ref > float("-inf")).any() else True


@pytest.mark.parametrize("scale", [0.0, 0.02, 3.0])
def test_scales(scale):
    """Uniform weights, and scores spread over hundreds (the reference is raised many times)."""
    ql = [400, 90]
    q, k, v, do = make(ql, ql, 2, 1, 64, torch.float16)
    seqs = PackedSequences(ql)
    o = packed_attention(q, k, v, seqs, sm_scale=scale)
    ref = packed_reference(q.double(), k.double(), v.double(), ql, ql, False, scale)[0]
    # the scores' own rounding in 32 bits: 2^-24 of their size times the products' sum, far below u
    assert rel(o, ref) <= 2 * U[torch.float16]


def test_rising_scores():
    """Every later key beats the earlier ones: each tile raises the softmax's reference."""
    n, d = 700, 64
    k = torch.zeros(n, 1, d, device="cuda")
    k[:, 0, 0] = torch.arange(n, device="cuda") * 0.25
    k = k.to(torch.bfloat16)
    q = torch.ones(n, 1, d, device="cuda", dtype=torch.bfloat16)
    v = torch.randn(n, 1, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
    for causal in (False, True):
        o = packed_attention(q, k, v, PackedSequences([n]), causal=causal, sm_scale=1.0)
        ref = packed_reference(q.double(), k.double(), v.double(), [n], [n], causal, 1.0)[0]
        assert rel(o, ref) <= 2 * U[torch.bfloat16]


def test_gradient_against_differences():
    """sum(o w) along the gradient: its difference between the ends of a path is the sum over the path's
    pieces of (x+ - x-) . (g(x+) + g(x-)) / 2. The two outputs are rounded to 16 bits (u |o| |w|,
    random), which over the path taken is below 2 %; sixteen pieces leave the trapezoids' own error, which
    falls with their square, below that."""
    ql, kl = [70, 33], [70, 90]
    q, k, v, w = make(ql, kl, 4, 2, 64, torch.float16, seed=3)
    seqs = PackedSequences(ql, kl)
    fn = lambda *x: packed_attention(*x, seqs, causal=True)  # noqa: E731
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


@pytest.mark.parametrize("d", [64, 128])
def test_other_sequences_take_no_part(d):
    """Infinities and NaN in the rows of another sequence, in all four tensors: nothing changes."""
    ql, kl = [70, 45, 200], [129, 45, 130]
    q, k, v, do = make(ql, kl, 4, 2, d, torch.bfloat16)
    seqs = PackedSequences(ql, kl)
    for causal in (False, True):
        fn = lambda *x: packed_attention(*x, seqs, causal=causal)  # noqa: E731
        clean = grads(fn, (q, k, v), do)
        bad = [t.clone() for t in (q, k, v, do)]
        for t, n0, n in ((bad[0], 70, 45), (bad[1], 129, 45), (bad[2], 129, 45), (bad[3], 70, 45)):
            t[n0:n0 + n:2] = float("nan")
            t[n0 + 1:n0 + n:2] = float("inf")
        dirty = grads(fn, bad[:3], bad[3])
        for c, x, (n0, n) in zip(clean, dirty, ((70, 45), (70, 45), (129, 45), (129, 45))):
            assert torch.equal(c[:n0], x[:n0]) and torch.equal(c[n0 + n:], x[n0 + n:])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_a_query_does_not_see(bad):
    """Causal: a value that is not finite reaches the queries from its position on, and no earlier one."""
    ql = [300, 40]
    q, k, v, _ = make(ql, ql, 4, 2, 128, torch.bfloat16)
    seqs = PackedSequences(ql)
    clean = packed_attention(q, k, v, seqs, causal=True)
    for at, col in ((7, 3), (130, 100), (260, 64), (299, 0), (305, 9)):
        w = v.clone()
        w[at, 1, col] = bad
        o = packed_attention(q, k, w, seqs, causal=True)
        hit = torch.zeros_like(o, dtype=torch.bool)
        end = 300 if at < 300 else 340
        hit[at:end, 2:, col] = True
        assert torch.equal(o[~hit], clean[~hit])
        if bad == float("inf"):
            assert (o[hit] == bad).all()
        else:
            assert torch.isnan(o[hit]).all()


def test_strides():
    """Slices of one QKV projection (rows 3 H D apart) and a head-major buffer are read in place; columns
    that are not contiguous and rows off the 16-byte grid through a copy. Same results."""
    n, h, d = [90, 161], 4, 64
    q, k, v, do = make(n, n, h, h, d, torch.bfloat16)
    seqs = PackedSequences(n)
    fn = lambda *x: packed_attention(*x, seqs, causal=True)  # noqa: E731
    want = grads(fn, (q, k, v), do)
    qkv = torch.stack([q, k, v], 1)
    major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    cols = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    odd = []
    for t in (q, k, v):
        buf = torch.empty(sum(n), h * d + 4, dtype=t.dtype, device="cuda")
        buf[:, 4:] = t.reshape(sum(n), h * d)
        odd.append(buf[:, 4:].view(sum(n), h, d))
    for views in (qkv.unbind(1), major, cols, odd):
        for a, b in zip(grads(fn, views, do.transpose(0, 1).contiguous().transpose(0, 1)), want):
            assert torch.equal(a, b)


def test_runs_are_alike_and_streams_are_the_callers():
    n = [700, 3, 90]
    q, k, v, do = make(n, n, 8, 2, 128, torch.bfloat16)
    seqs = PackedSequences(n)
    fn = lambda *x: packed_attention(*x, seqs, causal=True)  # noqa: E731
    want = grads(fn, (q, k, v), do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = grads(fn, (q, k, v), do)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_refusals():
    q, k, v, _ = make([8], [8], 2, 2, 64, torch.bfloat16)
    with pytest.raises(AssertionError, match="rows"):
        packed_attention(q, k, v, PackedSequences([7]))
    with pytest.raises(AssertionError, match="one CUDA device"):
        packed_attention(q, k, v, PackedSequences([8], device="cpu"))
    for scale in (-1.0, float("inf"), float("nan")):
        with pytest.raises(AssertionError, match="sm_scale"):
            packed_attention(q, k, v, PackedSequences([8]), sm_scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ql, kl, causal", [([1, 1, 1], None, True), ([70, 1, 3], [1, 1, 1], False), ([200, 90], [1, 1], True)])
def test_one_visible_key_passes_no_score_gradient(ql, kl, causal, dtype):
    """A softmax over one key is constant: the gradients of q and k are zeros, not roundings of zero."""
    kl = kl or ql
    q, k, v, do = make(ql, kl, 4, 2, 64, dtype)
    seqs = PackedSequences(ql, kl)
    _, dq, dk, dv = grads(lambda *x: packed_attention(*x, seqs, causal=causal), (q, k, v), do)
    assert not dq.any() and not dk.any() and dv.any()


@pytest.mark.parametrize("size", [2.0 ** -14, 1.0, 2.0 ** 10])
def test_fp16_gradients_of_many_keys(size):
    """P of 6000 keys and dS of small gradients lie below fp16's normal range: 4 u as in the module's docstring
    (outputs that are themselves below it excepted: their spacing is 2^-24)."""
    ql, kl = [64], [6000]
    q, k, v, do = make(ql, kl, 2, 1, 64, torch.float16)
    do = (do * size).to(torch.float16)
    do[:5] = 0
    seqs = PackedSequences(ql, kl)
    got = grads(lambda *x: packed_attention(*x, seqs), (q, k, v), do)
    want = grads(lambda *x: packed_reference(*x, ql, kl, False, 64 ** -0.5)[0], [t.double() for t in (q, k, v)], do)
    for x, ref in zip(got[1:], want[1:]):
        err = (x.double() - ref).norm().item()
        assert err <= 4 * U[torch.float16] * ref.norm().item() + 2.0 ** -25 * x.numel() ** 0.5


def test_captured_step():
    """A captured forward and backward follows the values in its inputs; its kernels start early as uncaptured ones do."""
    seqs = PackedSequences([200, 3, 700])
    q, k, v, do = make([200, 3, 700], [200, 3, 700], 4, 2, 64, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        o = packed_attention(*leaves, seqs, causal=True)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    new = make([200, 3, 700], [200, 3, 700], 4, 2, 64, torch.bfloat16, seed=1)
    with torch.no_grad():
        for t, x in zip((*leaves, do), new):
            t.copy_(x)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for x, ref in zip(out, step()):
        assert torch.equal(x, ref)


def test_gradients_carry_no_gradient():
    q, k, v, _ = make([20], [20], 2, 1, 64, torch.bfloat16)
    q.requires_grad_()
    o = packed_attention(q, k, v, PackedSequences([20]))
    dq, = torch.autograd.grad(o.float().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.float().sum().backward()


@pytest.mark.parametrize("ql, kl, causal", [([300, 2, 40], None, True), ([130], [3], False)])
def test_fp16_gradients_of_large_values(ql, kl, causal):
    """Value rows near the documented limit of the fp16 backward (a norm of 4094): 4 u as in the module's docstring."""
    kl = kl or ql
    q, k, v, do = make(ql, kl, 4, 2, 64, torch.float16)
    v = (v.float() * (4000 / v.float().norm(dim=-1, keepdim=True))).to(torch.float16)
    do = (do * 0.125).to(torch.float16)
    seqs = PackedSequences(ql, kl)
    got = grads(lambda *x: packed_attention(*x, seqs, causal=causal), (q, k, v), do)
    want = grads(lambda *x: packed_reference(*x, ql, kl, causal, 64 ** -0.5)[0], [t.double() for t in (q, k, v)], do)
    assert max(w.abs().max().item() for w in want) < 60000  # the results themselves are in range
    for x, ref in zip(got, want):
        assert rel(x, ref) <= 4 * U[torch.float16]
