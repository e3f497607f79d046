"""Measured cases of the packed-sequence and paged-cache operators.

Four operators, each with a plain form (elementary torch operations in 32 bits, rounded once at
the end) and the framework's own call:

  attention  softmax attention over packed sequences of different lengths, grouped heads, causal or
             not, alone (a prompt) or with its gradients (a training step)
  decode     attention of one new token per sequence over a paged key / value cache
  pages      rows written into a paged cache ("append") and whole pages copied ("copy")
  norm       gated residual with a norm after the block and a modulated norm before the next one,
             alone or with its gradients

``own`` selects the framework's kernels; the plain forms import nothing but torch.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# score elements that one chunk of the plain forms holds (1 GiB in 32 bits)
_CHUNK = 1 << 28


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one short prompt on a small model: latency of a single call
        dict(name="prompt_short", op="attention", backward=False, causal=True, seqs=1, longest=130, kv_longest=0, mix=1,
             heads=8, kv_heads=2, dim=64, dtype="bf16"),
        # a serving batch of prompts of mixed lengths, one of them a single token
        dict(name="prompt_packed", op="attention", backward=False, causal=True, seqs=16, longest=4093, kv_longest=0,
             mix=2, heads=40, kv_heads=8, dim=128, dtype="bf16"),
        # one long prompt: 21 video frames of 1560 tokens
        dict(name="prompt_long", op="attention", backward=False, causal=True, seqs=1, longest=32760, kv_longest=0,
             mix=3, heads=16, kv_heads=4, dim=128, dtype="bf16"),
        # training step of a cross attention: clips of mixed lengths over captions, one caption empty
        dict(name="train_cross", op="attention", backward=True, causal=False, seqs=5, longest=4680, kv_longest=301,
             mix=4, heads=8, kv_heads=8, dim=64, dtype="fp16"),
        # training step over packed clips of up to ten frames, grouped heads
        dict(name="train_packed", op="attention", backward=True, causal=True, seqs=4, longest=15600, kv_longest=0,
             mix=5, heads=16, kv_heads=4, dim=128, dtype="bf16"),
        # the next token of one short conversation
        dict(name="decode_one", op="decode", seqs=1, longest=201, mix=6, heads=8, kv_heads=2, dim=64, page=16,
             pool=64, dtype="fp16"),
        # a serving step over a batch whose sequences are at different lengths
        dict(name="decode_batch", op="decode", seqs=64, longest=8190, mix=7, heads=40, kv_heads=8, dim=128, page=16,
             pool=20000, dtype="bf16"),
        # few, very long sequences in a pool whose offsets pass 2^31 elements
        dict(name="decode_long", op="decode", seqs=3, longest=262143, mix=8, heads=16, kv_heads=4, dim=128, page=64,
             pool=66000, dtype="bf16"),
        # the keys and values of a prompt written into their pages
        dict(name="append_prompt", op="append", tokens=32760, kv_heads=8, dim=128, page=16, pool=6000, dtype="bf16"),
        # pages of forked sequences copied before they are written
        dict(name="copy_pages", op="copy", moves=2047, kv_heads=8, dim=128, page=16, pool=6000, dtype="bf16"),
        # a serving step's 24 new tokens between two blocks, rms norms on both sides
        dict(name="norm_step", op="norm", backward=False, seqs=24, longest=1, mix=9, width=5120, dtype="bf16",
             mod="bf16", norm="rms", post=True),
        # a training step of a 40 x 128 wide block over packed clips, modulated layer norm
        dict(name="norm_train", op="norm", backward=True, seqs=3, longest=16380, mix=10, width=5120, dtype="bf16",
             mod="fp32", norm="layer", post=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "decode", "decode", "append", "copy", "norm", "norm"])
    mix, dtype = rng.randrange(1 << 20), rng.choice(["bf16", "bf16", "fp16"])
    dim = rng.choice([128, 128, 64, 64, 96, 80, 40])
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8])
        case = dict(op=op, backward=rng.random() < 0.5, causal=rng.random() < 0.7, seqs=_log(rng, 1, 24),
                    longest=_log(rng, 1, 32760), kv_longest=_log(rng, 1, 16380) if rng.random() < 0.3 else 0, mix=mix,
                    heads=kv_heads * rng.choice([1, 2, 3, 4, 5, 8]), kv_heads=kv_heads, dim=dim, dtype=dtype)
        while work(case)["flops"] > 2e12 or _scores(case) > 4e9:
            case["longest"] = 1 + case["longest"] * 2 // 3
            case["kv_longest"] = case["kv_longest"] and 1 + case["kv_longest"] * 2 // 3
        return case
    if op == "decode":
        kv_heads, page = rng.choice([1, 2, 4, 8]), rng.choice([8, 16, 24, 32, 64, 128, 256])
        case = dict(op=op, seqs=_log(rng, 1, 256), longest=_log(rng, 1, 262143), mix=mix,
                    heads=kv_heads * rng.choice([1, 2, 4, 5, 8, 16]), kv_heads=kv_heads, dim=dim, page=page, pool=0,
                    dtype=dtype)
        while sum(_lengths(case["seqs"], case["longest"], mix)) * kv_heads > 3e6:
            case["longest"] = 1 + case["longest"] * 2 // 3
        case["pool"] = sum(-(-n // page) for n in _lengths(case["seqs"], case["longest"], mix)) + rng.randrange(1, 99)
        return case
    if op == "append":
        tokens, page = _log(rng, 1, 65520), rng.choice([8, 16, 24, 32, 64, 128, 256])
        return dict(op=op, tokens=tokens, kv_heads=rng.choice([1, 2, 4, 8]), dim=dim, page=page,
                    pool=-(-tokens // page) + rng.randrange(1, 99), dtype=dtype)
    if op == "copy":
        moves = _log(rng, 1, 2047)
        return dict(op=op, moves=moves, kv_heads=rng.choice([1, 2, 4, 8]), dim=dim,
                    page=rng.choice([8, 16, 24, 32, 64]), pool=2 * moves + rng.randrange(1, 99), dtype=dtype)
    case = dict(op=op, backward=rng.random() < 0.6, seqs=_log(rng, 1, 24), longest=_log(rng, 1, 16380), mix=mix,
                width=40 * _log(rng, 2, 200), dtype=dtype, mod=rng.choice([dtype, "fp32"]),
                norm=rng.choice(["rms", "layer"]), post=rng.random() < 0.6)
    while sum(_lengths(case["seqs"], case["longest"], mix)) * case["width"] > 1.2e8:
        case["longest"] = 1 + case["longest"] * 2 // 3
    return case


def _lengths(count, longest, mix, empty=False):
    """`count` lengths up to `longest`, spread over their logarithm; the longest itself, and from three
    sequences on one of a single token (of none with `empty`), are among them."""
    rng = random.Random(mix)
    out = [longest] + ([0 if empty else 1] if count >= 3 else [])
    while len(out) < count:
        out.append(_log(rng, 1, longest))
    out = out[:count]
    rng.shuffle(out)
    return out


def _lens(case):
    q = _lengths(case["seqs"], case["longest"], case["mix"])
    return q, (_lengths(case["seqs"], case["kv_longest"], case["mix"] + 1, True) if case["kv_longest"] else q)


def _visible(nq, nk, causal):
    """Query-key pairs of one sequence; causal: query i sees keys up to nk - nq + i."""
    if not causal:
        return nq * nk
    full = min(nq, nk)  # the last `full` queries see nk - full + 1 ... nk keys
    return full * (2 * nk - full + 1) // 2


def _scores(case):
    return sum(a * b for a, b in zip(*_lens(case))) * case["heads"]


def work(case):
    op = case["op"]
    if op == "attention":
        ql, kl = _lens(case)
        pairs = sum(_visible(a, b, case["causal"]) for a, b in zip(ql, kl)) * case["heads"]
        q = sum(ql) * case["heads"] * case["dim"] * 2
        kv = sum(kl) * case["kv_heads"] * case["dim"] * 2
        if case["backward"]:  # reads q, k, v, dO; writes o, dQ, dK, dV; two products forward, five backward
            return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * case["dim"]}
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * case["dim"]}
    if op == "decode":
        n = sum(_lengths(case["seqs"], case["longest"], case["mix"]))
        return {"bytes": 4 * n * case["kv_heads"] * case["dim"] + 4 * case["seqs"] * case["heads"] * case["dim"],
                "flops": 4 * n * case["heads"] * case["dim"]}
    if op == "append":
        return {"bytes": 8 * case["tokens"] * case["kv_heads"] * case["dim"] + 4 * case["tokens"], "flops": 0}
    if op == "copy":
        return {"bytes": 8 * case["moves"] * case["page"] * case["kv_heads"] * case["dim"] + 8 * case["moves"],
                "flops": 0}
    rows, c = sum(_lengths(case["seqs"], case["longest"], case["mix"])), case["width"]
    mod = 4 if case["mod"] == "fp32" else 2
    params = (3 * case["seqs"] + 1 + int(case["post"])) * c * mod
    if case["backward"]:  # x, y, both gradients in; x', h, dx, dy and the parameters' gradients out
        return {"bytes": 8 * rows * c * 2 + 2 * params, "flops": 40 * rows * c}
    return {"bytes": 4 * rows * c * 2 + params, "flops": 14 * rows * c}


# ------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype) * std


def _rows_of(lens):
    """Sequence index of every packed row."""
    return torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).cuda()


def _inputs(case, seed):
    g, dt, op = _gen(seed), _DTYPES[case["dtype"]], case["op"]
    if op == "attention":
        ql, kl = _lens(case)
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]

        def tokens(lens, heads):  # N(0, 1) around a mean that the sequence shares
            mean = _randn(g, len(lens), heads, d, std=0.3)
            return (_randn(g, sum(lens), heads, d) + mean[_rows_of(lens)]).to(dt)

        s = dict(q=tokens(ql, h), k=tokens(kl, hk), v=tokens(kl, hk), ql=ql, kl=kl)
        if case["backward"]:
            s["do"] = _randn(g, sum(ql), h, d).to(dt)
        return s
    if op == "norm":
        lens, c = _lengths(case["seqs"], case["longest"], case["mix"]), case["width"]
        rows, md = sum(lens), _DTYPES[case["mod"]]
        s = dict(lens=lens, rows=_rows_of(lens))
        # a residual stream with a mean and a spread of its own per column beside a block's output
        s["x"] = (_randn(g, rows, c) * (0.5 + _randn(g, c, std=0.5).abs()) + _randn(g, c, std=0.5)).to(dt)
        s["y"] = _randn(g, rows, c, std=2.0).to(dt)
        for name, std, mean in (("gate", 0.3, 0.0), ("scale", 0.3, 0.0), ("shift", 0.3, 0.0)):
            s[name] = (_randn(g, len(lens), c, std=std) + mean).to(md)
        s["weight"] = (_randn(g, c, std=0.2) + 1.0).to(md)
        s["post_weight"] = (_randn(g, c, std=0.2) + 1.0).to(md) if case["post"] else None
        if case["backward"]:
            s["dx_new"], s["dh"] = _randn(g, rows, c).to(dt), _randn(g, rows, c).to(dt)
        return s
    pool, page, hk, d = case["pool"], case["page"], case["kv_heads"], case["dim"]
    s = dict(k_pages=_randn(g, pool, hk, page, d, dtype=dt), v_pages=_randn(g, pool, hk, page, d, dtype=dt))
    order = torch.randperm(pool, generator=g, device="cuda")
    if op == "decode":
        lens = _lengths(case["seqs"], case["longest"], case["mix"])
        used = [-(-n // page) for n in lens]
        table = torch.zeros(len(lens), max(used), dtype=torch.int32, device="cuda")
        pos = 0
        for i, n in enumerate(used):
            table[i, :n] = order[pos:pos + n]
            pos += n
        s.update(q=_randn(g, len(lens), case["heads"], d, dtype=dt), table=table, lens=lens,
                 lengths=torch.tensor(lens, dtype=torch.int32).cuda())
    elif op == "append":
        n = case["tokens"]
        at = torch.arange(n, device="cuda")
        s.update(k=_randn(g, n, hk, d, dtype=dt), v=_randn(g, n, hk, d, dtype=dt),
                 slots=(order[at // page] * page + at % page).to(torch.int32))
    else:
        n = case["moves"]
        s.update(src=order[:n].to(torch.int32), dst=order[n:2 * n].to(torch.int32))
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if own:
        from vmonarch_b200 import PackedSequences
        if case["op"] == "attention":
            s["seqs"] = PackedSequences(s["ql"], s["kl"], device="cuda")
        elif case["op"] == "norm":
            s["seqs"] = PackedSequences(s["lens"], device="cuda")
        if case.get("backward"):
            for name in _LEAVES[case["op"]]:
                if s.get(name) is not None:
                    s[name].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------- passes
_LEAVES = {"attention": ("q", "k", "v"),
           "norm": ("x", "y", "gate", "scale", "shift", "weight", "post_weight")}


def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](case, state)


def _own_attention(case, s):
    from vmonarch_b200 import packed_attention
    o = packed_attention(s["q"], s["k"], s["v"], s["seqs"], causal=case["causal"])
    if not case["backward"]:
        return o
    return (o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"]))


def _own_decode(case, s):
    from vmonarch_b200 import paged_attention
    return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"])


def _own_append(case, s):
    from vmonarch_b200 import append_pages
    append_pages(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"])
    return s["k_pages"], s["v_pages"]


def _own_copy(case, s):
    from vmonarch_b200 import copy_pages
    copy_pages(s["k_pages"], s["v_pages"], s["src"], s["dst"])
    return s["k_pages"], s["v_pages"]


def _own_norm(case, s):
    from vmonarch_b200 import gated_residual_norm
    x, h = gated_residual_norm(s["x"], s["y"], gate=s["gate"], scale=s["scale"], shift=s["shift"],
                               weight=s["weight"], post_weight=s["post_weight"], norm=case["norm"], eps=1e-6,
                               seqs=s["seqs"])
    if not case["backward"]:
        return x, h
    leaves = [s[n] for n in _LEAVES["norm"] if s[n] is not None]
    return (x.detach(), h.detach(), *torch.autograd.grad((x, h), leaves, (s["dx_new"], s["dh"])))


def _plain_attention(case, s):
    h, hk, d, causal = case["heads"], case["kv_heads"], case["dim"], case["causal"]
    group, scale, back = h // hk, d ** -0.5, case["backward"]
    dt = s["q"].dtype
    o = torch.zeros(s["q"].shape, device="cuda")
    dq, dk, dv = (torch.zeros(s[n].shape, device="cuda") for n in "qkv") if back else (None,) * 3
    q0 = k0 = 0
    for nq, nk in zip(s["ql"], s["kl"]):
        if nq and nk:
            k = s["k"][k0:k0 + nk].float().transpose(0, 1)      # (hk, nk, d)
            v = s["v"][k0:k0 + nk].float().transpose(0, 1)
            step = max(1, min(nq, _CHUNK // (h * nk)))
            for i in range(0, nq, step):
                n = min(step, nq - i)
                last = min(nk, max(1, nk - nq + i + n)) if causal else nk  # keys that some row sees
                rows = slice(q0 + i, q0 + i + n)

                def heads(t):  # (n, h, d) -> (hk, group * n, d)
                    return t[rows].float().view(n, hk, group, d).permute(1, 2, 0, 3).reshape(hk, group * n, d)

                def back_to(t):
                    return t.view(hk, group, n, d).permute(2, 0, 1, 3).reshape(n, h, d)

                q = heads(s["q"])
                p = q @ k[:, :last].transpose(1, 2)
                p *= scale
                if causal:
                    at = torch.arange(i, i + n, device="cuda")[:, None] + (nk - nq)
                    hide = torch.arange(last, device="cuda")[None] > at
                    p.view(hk, group, n, last).masked_fill_(hide, -math.inf)
                top = p.amax(2, keepdim=True)
                top = torch.where(top == -math.inf, torch.zeros_like(top), top)
                p = torch.exp(p - top)
                total = p.sum(2, keepdim=True)
                p /= torch.where(total == 0, torch.ones_like(total), total)
                o[rows] = back_to(p @ v[:, :last])
                if back:
                    do = heads(s["do"])
                    dv[k0:k0 + last] += (p.transpose(1, 2) @ do).transpose(0, 1)
                    ds = do @ v[:, :last].transpose(1, 2)
                    ds = p * (ds - (p * ds).sum(2, keepdim=True)) * scale
                    dq[rows] = back_to(ds @ k[:, :last])
                    dk[k0:k0 + last] += (ds.transpose(1, 2) @ q).transpose(0, 1)
        q0, k0 = q0 + nq, k0 + nk
    return tuple(t.to(dt) for t in (o, dq, dk, dv)) if back else o.to(dt)


def _plain_decode(case, s):
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    q = s["q"].float().view(len(s["lens"]), hk, case["heads"] // hk, d)
    o = torch.empty_like(q)
    for i, n in enumerate(s["lens"]):
        used = s["table"][i, :-(-n // page)].long()
        k = s["k_pages"][used].float().transpose(0, 1).reshape(hk, -1, d)[:, :n]
        v = s["v_pages"][used].float().transpose(0, 1).reshape(hk, -1, d)[:, :n]
        p = q[i] @ k.transpose(1, 2) * d ** -0.5
        p = torch.exp(p - p.amax(2, keepdim=True))
        o[i] = (p / p.sum(2, keepdim=True)) @ v
    return o.view(s["q"].shape).to(s["q"].dtype)


def _plain_append(case, s):
    page, at = torch.div(s["slots"], case["page"], rounding_mode="floor").long(), (s["slots"] % case["page"]).long()
    s["k_pages"][page, :, at] = s["k"]
    s["v_pages"][page, :, at] = s["v"]
    return s["k_pages"], s["v_pages"]


def _plain_copy(case, s):
    src, dst = s["src"].long(), s["dst"].long()
    s["k_pages"][dst] = s["k_pages"][src]
    s["v_pages"][dst] = s["v_pages"][src]
    return s["k_pages"], s["v_pages"]


def _plain_norm(case, s):
    eps, rows, layer = 1e-6, s["rows"], case["norm"] == "layer"
    dt, md = s["x"].dtype, s["gate"].dtype
    y, weight, post = s["y"].float(), s["weight"].float(), s["post_weight"]
    gate, scale = s["gate"].float()[rows], 1.0 + s["scale"].float()[rows]
    ry = torch.rsqrt((y * y).mean(1, keepdim=True) + eps) if post is not None else 1.0
    yn = y * ry
    yw = yn * post.float() if post is not None else yn
    x = s["x"].float() + gate * yw
    mean = x.mean(1, keepdim=True) if layer else 0.0
    xc = x - mean
    r = torch.rsqrt((xc * xc).mean(1, keepdim=True) + eps)
    xn = xc * r
    h = xn * weight * scale + s["shift"].float()[rows]
    if not case["backward"]:
        return x.to(dt), h.to(dt)

    def per_seq(t):
        return torch.zeros(s["gate"].shape, device="cuda").index_add_(0, rows, t)

    dh = s["dh"].float()
    g = dh * weight * scale
    dx = r * (g - xn * (g * xn).mean(1, keepdim=True) - (g.mean(1, keepdim=True) if layer else 0.0))
    dx += s["dx_new"].float()
    dyw = dx * gate
    grads = [per_seq(dx * yw), per_seq(dh * xn * weight), per_seq(dh), (dh * xn * scale).sum(0)]
    if post is not None:
        t = dyw * post.float()
        dy = ry * (t - yn * (t * yn).mean(1, keepdim=True))
        grads.append((dyw * yn).sum(0))
    else:
        dy = dyw
    return (x.to(dt), h.to(dt), dx.to(dt), dy.to(dt), *(t.to(md) for t in grads))


_own = {"attention": _own_attention, "decode": _own_decode, "append": _own_append, "copy": _own_copy,
        "norm": _own_norm}
_plain = {"attention": _plain_attention, "decode": _plain_decode, "append": _plain_append, "copy": _plain_copy,
          "norm": _plain_norm}


# -------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The outputs of :func:`run` in 64 bits, from each operator's definition; gradients by automatic
    differentiation of it. None for the page moves, whose outputs are copies."""
    if case["op"] in ("append", "copy"):
        return None
    s = _inputs(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "decode":
        d, group, outs = case["dim"], case["heads"] // case["kv_heads"], []
        for i, n in enumerate(s["lens"]):
            at = torch.arange(n, device="cuda")
            page, slot = s["table"][i].long()[at // case["page"]], at % case["page"]
            heads = []
            for j in range(case["kv_heads"]):
                k, v = s["k_pages"][page, j, slot].double(), s["v_pages"][page, j, slot].double()
                x = s["q"][i, j * group:(j + 1) * group].double() @ k.T / math.sqrt(d)
                heads.append(torch.softmax(x, -1) @ v)
            outs.append(torch.cat(heads))
        return torch.stack(outs)
    names = [n for n in _LEAVES["norm"] if s[n] is not None]
    t = {n: s[n].double().requires_grad_(case["backward"]) for n in names}
    eps, rows, c = 1e-6, s["rows"], case["width"]
    y = t["y"]
    if case["post"]:
        y = torch.nn.functional.rms_norm(y, (c,), t["post_weight"], eps)
    x = t["x"] + t["gate"][rows] * y
    fn = torch.nn.functional.layer_norm if case["norm"] == "layer" else torch.nn.functional.rms_norm
    h = fn(x, (c,), eps=eps) * t["weight"] * (1 + t["scale"][rows]) + t["shift"][rows]
    if not case["backward"]:
        return x, h
    grads = torch.autograd.grad((x, h), [t[n] for n in names], (s["dx_new"].double(), s["dh"].double()))
    return (x.detach(), h.detach(), *grads)


def _exact_attention(case, s):
    d, group, back = case["dim"], case["heads"] // case["kv_heads"], case["backward"]
    outs = [torch.zeros(s[n].shape, device="cuda", dtype=torch.float64) for n in (("q", "q", "k", "v") if back else "q")]
    q0 = k0 = 0
    for nq, nk in zip(s["ql"], s["kl"]):
        at = torch.arange(nq, device="cuda")
        seen = at - nq + nk + 1 if case["causal"] else torch.full_like(at, nk)  # leading keys each query sees
        for j in range(case["heads"] if nk else 0):
            for i in range(0, nq, 8192):
                m = min(8192, nq - i)
                w = max(1, min(nk, int(seen[i + m - 1])))
                q = s["q"][q0 + i:q0 + i + m, j].double().requires_grad_(back)
                k = s["k"][k0:k0 + w, j // group].double().requires_grad_(back)
                v = s["v"][k0:k0 + w, j // group].double().requires_grad_(back)
                mask = torch.arange(w, device="cuda")[None] < seen[i:i + m, None]
                x = torch.where(mask, q @ k.T / math.sqrt(d), -1e300)
                p = torch.where(mask, torch.softmax(x, -1), 0.0)
                o = p @ v
                outs[0][q0 + i:q0 + i + m, j] = o.detach()
                if back:
                    gq, gk, gv = torch.autograd.grad(o, (q, k, v), s["do"][q0 + i:q0 + i + m, j].double())
                    outs[1][q0 + i:q0 + i + m, j] = gq
                    outs[2][k0:k0 + w, j // group] += gk
                    outs[3][k0:k0 + w, j // group] += gv
        q0, k0 = q0 + nq, k0 + nk
    return tuple(outs) if back else outs[0]
