"""The gated residual norm against its definition in 64 bits.

Everything is 32-bit and rounded once: errors in the Frobenius norm are at most the output type's rounding
u (2^-8 bf16, 2^-11 fp16), plus 1e-5 for the 32-bit arithmetic (some hundred roundings of 2^-24, the sums over
rows among them). fp32 gradients: 1e-5 alone."""
import pytest
import torch

from vmonarch_b200 import PackedSequences, gated_residual_norm

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}
NAMES = ("x", "y", "gate", "scale", "shift", "weight", "post_weight")


def make(lens, c, dtype, pdtype, skip=(), seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, dt=dtype, mean=0.0, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std + mean).to(dt)  # noqa: E731
    n, s = sum(lens), len(lens)
    t = dict(x=r(n, c, mean=0.5), y=r(n, c, std=2.0), gate=r(s, c, dt=pdtype, std=0.5), scale=r(s, c, dt=pdtype, std=0.3),
             shift=r(s, c, dt=pdtype), weight=r(c, dt=pdtype, mean=1.0, std=0.2),
             post_weight=r(c, dt=pdtype, mean=1.0, std=0.2))
    return {k: None if k in skip else v for k, v in t.items()}, r(n, c), r(n, c)


def reference(t, lens, norm, eps):
    rows = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), torch.tensor(lens, device="cuda"))
    per = lambda k, none: none if t[k] is None else t[k].reshape(-1, t["x"].size(1))[rows]  # noqa: E731
    x, y = t["x"], t["y"]
    if y is not None:
        if t["post_weight"] is not None:
            y = y * (y.pow(2).mean(1, keepdim=True) + eps).rsqrt() * t["post_weight"]
        x = x + per("gate", 1.0) * y
    z = x - x.mean(1, keepdim=True) if norm == "layer" else x
    n = z * (z.pow(2).mean(1, keepdim=True) + eps).rsqrt()
    h = n * (1.0 if t["weight"] is None else t["weight"]) * (1 + per("scale", 0.0)) + per("shift", 0.0)
    return x, h


def rel(a, b):
    assert torch.isfinite(a).all()
    return ((a.double() - b).norm() / b.norm().clamp_min(1e-30)).item()


def check(lens, c, dtype, pdtype, norm, skip=(), eps=1e-6, seqs=True, t=None, use=(True, True)):
    made, dx_new, dh = make(lens, c, dtype, pdtype, skip)
    t = made if t is None else t
    s = PackedSequences(lens) if seqs else None
    leaves = {k: None if v is None else v.detach().requires_grad_() for k, v in t.items()}
    x, h = gated_residual_norm(**leaves, norm=norm, eps=eps, seqs=s)
    exact = {k: None if v is None else v.detach().double().requires_grad_() for k, v in t.items()}
    rx, rh = reference(exact, lens, norm, eps)
    assert rel(h, rh) <= U[dtype] + 1e-5
    if t["y"] is None:
        assert x is leaves["x"]
    else:
        assert rel(x, rx) <= U[dtype] + 1e-5
    names = [k for k in NAMES if t[k] is not None]
    pick = lambda x, h: [o for o, on in zip((x, h), use) if on]  # noqa: E731
    got = torch.autograd.grad(pick(x, h), [leaves[k] for k in names], pick(dx_new, dh), allow_unused=True)
    want = torch.autograd.grad(pick(rx, rh), [exact[k] for k in names], pick(dx_new.double(), dh.double()),
                               allow_unused=True)
    for k, a, b in zip(names, got, want):
        if b is None or b.norm() == 0:
            assert a is None or a.abs().max() == 0, k
        else:
            assert a.shape == t[k].shape and a.dtype == t[k].dtype
            assert rel(a, b) <= U[a.dtype] + 1e-5, k
    with torch.no_grad():
        x2, h2 = gated_residual_norm(**t, norm=norm, eps=eps, seqs=s)
    assert torch.equal(h2, h) and torch.equal(x2, x)
    return x, h, got


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dtype, pdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                           (torch.float16, torch.float16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("c", [8, 80, 256, 264, 1040, 2048, 5120, 5128, 8192])
def test_widths_and_types(c, dtype, pdtype, norm):
    check([5, 0, 1, 130], c, dtype, pdtype, norm)


@pytest.mark.parametrize("skip", [("post_weight",), ("gate",), ("scale", "shift"), ("weight", "post_weight"),
                                  ("gate", "scale", "shift", "weight", "post_weight"), ("y", "gate", "post_weight"),
                                  ("y", "gate", "post_weight", "scale", "shift", "weight")])
def test_left_out_parts(skip):
    for norm in ("rms", "layer"):
        check([40, 3], 320, torch.bfloat16, torch.float32, norm, skip)


@pytest.mark.parametrize("lens", [[1], [1] * 24, [1] * 700, [3000], [2000, 1, 0, 0, 1999], [0, 7], [7, 0]])
def test_rows(lens):
    check(lens, 136, torch.bfloat16, torch.float32, "layer")
    if len(lens) == 1:
        check(lens, 5120, torch.float16, torch.float16, "rms", seqs=False)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("c", [80, 256, 264, 512, 520, 1040, 2048, 4096, 5120, 5128, 7000, 8192])
def test_many_rows(c, norm):
    """More rows than blocks, in runs that cross sequences: the other layout of the forward's threads."""
    check([301, 0, 1, 90], c, torch.bfloat16, torch.float32, norm)
    check([301, 0, 1, 90], c, torch.float16, torch.float16, norm, ("post_weight",))


@pytest.mark.parametrize("use", [(True, False), (False, True)])
def test_one_output_unused(use):
    check([30, 4], 320, torch.bfloat16, torch.float32, "layer", use=use)


def test_no_rows():
    t, _, _ = make([0, 0], 64, torch.bfloat16, torch.float32)
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    x, h = gated_residual_norm(**leaves, seqs=PackedSequences([0, 0]))
    assert x.shape == h.shape == (0, 64)
    for g in torch.autograd.grad((x, h), list(leaves.values()), (x.detach(), h.detach())):
        assert g.numel() == 0 or g.abs().max() == 0


def test_large_mean():
    """A mean a thousand times the spread: the variance is taken from the differences, not from squares."""
    t, _, _ = make([64], 1024, torch.float16, torch.float32)
    t["x"] = (torch.randn(64, 1024, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)) + 1000).half()
    t["y"] = torch.zeros_like(t["x"])
    x, h = gated_residual_norm(**t, norm="layer")
    rx, rh = reference({k: v.double() for k, v in t.items()}, [64], "layer", 1e-6)
    # the mean's own rounding in 32 bits is 1000 * 2^-24 of a spread of 1
    assert rel(h, rh) <= U[torch.float16] + 1e-4


def test_zero_rows():
    """A row of zeros: eps alone keeps the norm finite."""
    t, _, _ = make([6], 64, torch.bfloat16, torch.float32)
    t["x"][2], t["y"][2] = 0, 0
    check([6], 64, torch.bfloat16, torch.float32, "rms", t=t, eps=1e-3)


def test_gradient_against_differences():
    """The sum of both outputs' products with fixed weights, between the ends of a path along each gradient,
    against the trapezoids of the gradient over its sixteen pieces. fp32 gradients of fp16 outputs: the
    outputs' rounding (u |h| |w|, random) is below 2 % of the difference, the trapezoids' own error, which falls
    with their square, below that."""
    t, wx, wh = make([9, 20], 64, torch.float16, torch.float32, seed=4)
    seqs = PackedSequences([9, 20])

    def at(name, value):
        leaves = {k: v.detach().requires_grad_() for k, v in {**t, name: value}.items()}
        x, h = gated_residual_norm(**leaves, norm="layer", seqs=seqs)
        (g,) = torch.autograd.grad((x, h), [leaves[name]], (wx, wh))
        return value.double(), (x.double() * wx.double()).sum() + (h.double() * wh.double()).sum(), g.double()

    for name in NAMES:
        g = at(name, t[name])[2].float()
        step = 0.1 * g / g.pow(2).mean().sqrt()
        pts = [at(name, (t[name].float() + (1 - i / 8) * step).to(t[name].dtype)) for i in range(17)]
        predicted = sum(((a[0] - b[0]) * (a[2] + b[2])).sum() / 2 for a, b in zip(pts, pts[1:]))
        assert abs((pts[0][1] - pts[-1][1] - predicted) / predicted) <= 0.02, name


def test_strides_streams_and_repeats():
    """Rows inside a wider buffer are read in place, rows off the 16-byte grid and column-major parameters
    through a copy; another stream, and a second run, give the same bits."""
    lens, c = [33, 5], 320
    t, dx_new, dh = make(lens, c, torch.bfloat16, torch.float32)
    seqs = PackedSequences(lens)

    def run(t, dx_new, dh):
        leaves = {k: v.detach().requires_grad_() for k, v in t.items()}
        out = gated_residual_norm(**leaves, norm="layer", seqs=seqs)
        return [*out, *torch.autograd.grad(out, list(leaves.values()), (dx_new, dh))]

    want = run(t, dx_new, dh)
    wide = lambda v, off: torch.cat([v.new_zeros(v.size(0), off), v, v.new_zeros(v.size(0), 24)], 1)[:, off:off + c]  # noqa: E731
    for off in (8, 3):
        views = {k: wide(v, off) if k in ("x", "y") else v for k, v in t.items()}
        views["gate"] = t["gate"].T.contiguous().T
        for a, b in zip(run(views, wide(dx_new, off), wide(dh, off)), want):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(t, dx_new, dh)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_refusals():
    t, _, _ = make([6, 2], 64, torch.bfloat16, torch.float32)
    seqs = PackedSequences([6, 2])
    wide = torch.zeros(8, 8200, device="cuda", dtype=torch.bfloat16)
    for bad in (dict(x=t["x"].float()), dict(x=t["x"][None]), dict(x=t["x"][:, :60], y=t["y"][:, :60]), dict(x=wide, y=wide),
                dict(y=t["y"][:7]), dict(y=t["y"].half()), dict(y=None), dict(norm="batch"), dict(eps=-1.0),
                dict(eps=float("nan")), dict(gate=t["gate"][:1]), dict(gate=t["gate"].bfloat16()), dict(weight=t["gate"]),
                dict(scale=t["scale"].half()), dict(shift=t["shift"].cpu()), dict(seqs=PackedSequences([6, 3])),
                dict(seqs=PackedSequences([6, 2], device="cpu")), dict(seqs=None), dict(x=t["x"].cpu(), y=t["y"].cpu())):
        with pytest.raises(AssertionError):
            gated_residual_norm(**{**t, "seqs": seqs, **bad})
