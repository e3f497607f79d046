"""Measured cases of windowed attention, the 8-bit paged cache and the page tables on the GPU.

Four operators, each with a plain form (elementary torch operations, in 32 bits where they compute) and the framework's own call:

  window   causal softmax attention over packed sequences, each query over the last `window` keys and the first `sinks`
           ones, grouped heads, alone (a prompt, behind a cached prefix or not) or with its gradients (a training step)
  decode   attention of one new token per sequence over a paged cache, in 16 bits with a window and sinks, or in 8 bits
           (e4m3 values with a power-of-two scale for each page and head) with or without them
  append   rows quantised into an 8-bit paged cache: a page's scale grows where its new rows need it, and what the page held is
           brought to the new scale
  tables   page tables and slot maps from lengths: sequences cut back to the tokens they keep, pages returned to the stack of
           free ones, pages taken from it for the tokens to come

``own`` selects the framework's kernels; the plain forms import nothing but torch.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_E4M3 = torch.float8_e4m3fn
# score elements that one chunk of the plain forms holds (1 GiB in 32 bits)
_CHUNK = 1 << 28


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one short prompt on a small model: latency of a single call
        dict(name="window_short", op="window", backward=False, seqs=1, longest=701, prefix=0, mix=1, window=256, sinks=4,
             heads=8, kv_heads=2, dim=64, dtype="bf16"),
        # a serving batch of prompts of mixed lengths, one of them a single token, in a model with a window of 1024
        dict(name="window_packed", op="window", backward=False, seqs=16, longest=8190, prefix=0, mix=2, window=1024, sinks=4,
             heads=40, kv_heads=8, dim=128, dtype="bf16"),
        # a small fp16 training step: clips of up to nine frames of 520 tokens, over the last frame's length of tokens and 77 first ones
        dict(name="window_train_small", op="window", backward=True, seqs=5, longest=4680, prefix=0, mix=3, window=520, sinks=77,
             heads=8, kv_heads=8, dim=64, dtype="fp16"),
        # a training step on clips of up to ten frames of 1560 tokens, over the last two frames' length and the first frame
        dict(name="window_train", op="window", backward=True, seqs=4, longest=15600, prefix=0, mix=5, window=3120, sinks=1560,
             heads=16, kv_heads=4, dim=128, dtype="bf16"),
        # a serving step of 64 sequences of mixed lengths over a 16-bit cache, window of 4095 and sinks
        dict(name="decode_window", op="decode", bits=16, seqs=64, longest=32760, mix=6, window=4095, sinks=4, heads=40,
             kv_heads=8, dim=128, page=16, dtype="bf16"),
        # one new token of one short sequence, 8-bit cache: latency
        dict(name="decode8_one", op="decode", bits=8, seqs=1, longest=201, mix=7, window=0, sinks=0, heads=8, kv_heads=2,
             dim=64, page=16, dtype="fp16"),
        # a serving step of 64 sequences of mixed lengths over an 8-bit cache
        dict(name="decode8_batch", op="decode", bits=8, seqs=64, longest=8190, mix=8, window=0, sinks=0, heads=40,
             kv_heads=8, dim=128, page=16, dtype="bf16"),
        # a few very long sequences over an 8-bit cache
        dict(name="decode8_long", op="decode", bits=8, seqs=3, longest=262143, mix=9, window=0, sinks=0, heads=16, kv_heads=4,
             dim=128, page=64, dtype="bf16"),
        # a serving step's new keys and values, one token of each of 64 sequences
        dict(name="append_step", op="append", seqs=64, longest=1, mix=10, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # long prompts' keys and values
        dict(name="append_prompts", op="append", seqs=3, longest=16380, mix=11, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # a serving step of 64 sequences that drop up to 4 drafted tokens and take up to 5 new ones
        dict(name="tables_step", op="tables", seqs=64, longest=8190, mix=12, drafts=4, page=16),
        # a batch of 1024 requests evicted and another one admitted
        dict(name="tables_prompts", op="tables", seqs=1024, longest=4093, mix=13, drafts=0, page=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "window", "window", "decode", "decode", "decode", "append", "append", "tables"])
    mix, dtype = rng.randrange(1 << 20), rng.choice(["bf16", "bf16", "fp16"])
    if op == "window":
        kv_heads = rng.choice([1, 2, 4, 8])
        longest = _log(rng, 1, 32760)
        case = dict(op=op, backward=rng.random() < 0.5, seqs=_log(rng, 1, 24), longest=longest,
                    prefix=_log(rng, 1, 8190) if rng.random() < 0.3 else 0, mix=mix, window=_log(rng, 1, 8190),
                    sinks=_log(rng, 1, 1560) if rng.random() < 0.7 else 0, heads=kv_heads * rng.choice([1, 2, 3, 4, 5, 8]),
                    kv_heads=kv_heads, dim=rng.choice([128, 128, 64, 64, 96, 80, 40]), dtype=dtype)
        while work(case)["flops"] > 6e11 or _scores(case) > 3e9:
            case["longest"] = 1 + case["longest"] * 2 // 3
            case["prefix"] = case["prefix"] and 1 + case["prefix"] * 2 // 3
        return case
    page = rng.choice([8, 16, 16, 24, 32, 64, 128, 256])
    if op == "decode":
        kv_heads, bits = rng.choice([1, 2, 4, 8]), rng.choice([8, 8, 16])
        windowed = bits == 16 or rng.random() < 0.5
        case = dict(op=op, bits=bits, seqs=_log(rng, 1, 256), longest=_log(rng, 1, 262143), mix=mix,
                    window=_log(rng, 1, 16380) if windowed else 0, sinks=_log(rng, 1, 520) if windowed and rng.random() < 0.6 else 0,
                    heads=kv_heads * rng.choice([1, 2, 4, 5, 8, 16]), kv_heads=kv_heads,
                    dim=rng.choice([128, 128, 64, 64, 96, 80, 48]), page=page, dtype=dtype)
        while case["seqs"] * case["longest"] * kv_heads > 3e6:
            case["longest"] = 1 + case["longest"] * 2 // 3
        return case
    if op == "append":
        case = dict(op=op, seqs=_log(rng, 1, 256), longest=_log(rng, 1, 16380) if rng.random() < 0.6 else 1, mix=mix,
                    kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([128, 128, 64, 96, 80, 48]), page=page, dtype=dtype)
        while sum(_lengths(case["seqs"], case["longest"], mix)) > 20000:
            case["longest"] = 1 + case["longest"] * 2 // 3
        return case
    case = dict(op=op, seqs=_log(rng, 1, 2048), longest=_log(rng, 1, 32760), mix=mix,
                drafts=rng.choice([0, 1, 3, 8, 17]), page=page)
    while case["seqs"] * case["longest"] > 4e6:
        case["longest"] = 1 + case["longest"] * 2 // 3
    return case


def _lengths(count, longest, mix):
    """`count` lengths up to `longest`, spread over their logarithm; the longest itself, and from three sequences on one
    of a single token, are among them."""
    rng = random.Random(mix)
    out = [longest] + ([1] if count >= 3 else [])
    out = (out + [_log(rng, 1, longest) for _ in range(count - len(out))])[:count]
    rng.shuffle(out)
    return out


def _lens(case):
    """Queries and keys of every sequence."""
    q = _lengths(case["seqs"], case["longest"], case["mix"])
    before = _lengths(case["seqs"], case["prefix"], case["mix"] + 1) if case["prefix"] else [0] * len(q)
    return q, [a + b for a, b in zip(q, before)]


def _pairs(nq, nk, span):
    """Query-key pairs of one sequence where the query behind n keys sees the last of them and the first, `span` at most."""
    first, last = nk - nq + 1, nk
    ramp = max(0, min(last, span) - first + 1)  # queries that see every key so far
    return ramp * (2 * first + ramp - 1) // 2 + (nq - ramp) * span


def _scores(case):
    """Score elements that a form without the window would hold."""
    return sum(a * b for a, b in zip(*_lens(case))) * case["heads"]


def _grow(case):
    """Lengths before, tokens that are kept and tokens to come of every sequence of a `tables` case."""
    rng = random.Random(case["mix"] + 2)
    before = _lengths(case["seqs"], case["longest"], case["mix"])
    if not case["drafts"]:
        return before, [0] * len(before), _lengths(case["seqs"], case["longest"], case["mix"] + 1)
    keep = [max(0, n - rng.randint(0, case["drafts"])) for n in before]
    return before, keep, [rng.randint(0, case["drafts"] + 1) for _ in before]


def work(case):
    op = case["op"]
    if op == "window":
        ql, kl = _lens(case)
        span = case["window"] + case["sinks"]
        pairs = sum(_pairs(a, b, span) for a, b in zip(ql, kl)) * case["heads"]
        q = sum(ql) * case["heads"] * case["dim"] * 2
        kv = sum(kl) * case["kv_heads"] * case["dim"] * 2
        if case["backward"]:  # reads q, k, v, dO; writes o, dQ, dK, dV; two products forward, five backward
            return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * case["dim"]}
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * case["dim"]}
    if op == "decode":
        lens = _lengths(case["seqs"], case["longest"], case["mix"])
        span = case["window"] + case["sinks"] if case["window"] else case["longest"]
        n, size = sum(min(a, span) for a in lens), case["bits"] // 8
        scales = 8 * n * case["kv_heads"] / case["page"] if case["bits"] == 8 else 0
        return {"bytes": 2 * size * n * case["kv_heads"] * case["dim"] + scales + 4 * case["seqs"] * case["heads"] * case["dim"],
                "flops": 4 * n * case["heads"] * case["dim"]}
    if op == "append":
        n = sum(_lengths(case["seqs"], case["longest"], case["mix"]))
        return {"bytes": 6 * n * case["kv_heads"] * case["dim"] + 4 * n, "flops": 4 * n * case["kv_heads"] * case["dim"]}
    before, keep, counts = _grow(case)
    pages = sum(_ceil(a, case["page"]) - _ceil(k, case["page"]) + 2 * (_ceil(k + c, case["page"]) - _ceil(k, case["page"]))
                for a, k, c in zip(before, keep, counts))
    return {"bytes": 4 * (sum(counts) + 4 * len(counts) + 2 * pages), "flops": 0}


def _ceil(a, b):
    return -(-a // b)


# ------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _starts(lens):
    return [sum(lens[:i]) for i in range(len(lens))]


def _rows_of(lens):
    """Sequence index of every packed row."""
    return torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).cuda()


def _places(lens):
    """Position of every packed row in its sequence."""
    rows = _rows_of(lens)
    return torch.arange(len(rows), device="cuda") - torch.tensor(_starts(lens)).cuda()[rows]


def _pow2_scale(top):
    """The least power of two s with top <= 448 s (448: the largest e4m3 value), 2^-126 at least."""
    m, e = torch.frexp(top)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.ldexp(torch.ones_like(top), torch.where(top > 0, e, torch.full_like(e, -126)).clamp_min(-126))


def _pool(g, pages, hk, page, dim, dtype, bits):
    """Keys or values of a pool: N(0, 1) with a spread of its own per channel; 8 bits: e4m3 values and their scales."""
    x = _randn(g, pages, hk, page, dim) * (0.4 + _randn(g, hk, 1, dim, std=0.6).abs())
    if bits == 16:
        return x.to(dtype), None
    scale = _pow2_scale(x.abs().amax((2, 3)))
    return (x / scale[..., None, None]).to(_E4M3), scale


def _inputs(case, seed):
    g, op = _gen(seed), case["op"]
    if op == "window":
        ql, kl = _lens(case)
        h, hk, d, dt = case["heads"], case["kv_heads"], case["dim"], _DTYPES[case["dtype"]]

        def tokens(lens, heads):  # N(0, 1) around a mean that the sequence shares
            return (_randn(g, sum(lens), heads, d) + _randn(g, len(lens), heads, d, std=0.3)[_rows_of(lens)]).to(dt)

        s = dict(q=tokens(ql, h), k=tokens(kl, hk), v=tokens(kl, hk), ql=ql, kl=kl)
        if case["backward"]:
            s["do"] = _randn(g, sum(ql), h, d).to(dt)
        return s
    page = case["page"]
    if op == "tables":
        before, keep, counts = _grow(case)
        used = [_ceil(n, page) for n in before]
        width = max(used + [_ceil(k + c, page) for k, c in zip(keep, counts)]) + 1
        pool = max(sum(used), sum(_ceil(k + c, page) for k, c in zip(keep, counts))) + 77
        order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
        table = torch.full((len(before), width), -1, dtype=torch.int32, device="cuda")
        table[_rows_of(used), _places(used)] = order[:sum(used)]
        left = pool - sum(used)
        free = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
        free[:left] = order[sum(used):]
        ints = [torch.tensor(x, dtype=torch.int32).cuda() for x in (before, keep, counts, [left])]
        return dict(table=table, lengths=ints[0], keep=ints[1], counts=ints[2], free=free, num_free=ints[3], total=sum(counts))
    hk, d, dt = case["kv_heads"], case["dim"], _DTYPES[case["dtype"]]
    lens = _lengths(case["seqs"], case["longest"], case["mix"])
    if op == "decode":
        used = [_ceil(n, page) for n in lens]
        pool = sum(used) + 13
        order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
        table = torch.zeros((len(lens), max(used)), dtype=torch.int32, device="cuda")
        table[_rows_of(used), _places(used)] = order[:sum(used)]
        k, ks = _pool(g, pool, hk, page, d, dt, case["bits"])
        v, vs = _pool(g, pool, hk, page, d, dt, case["bits"])
        return dict(q=_randn(g, len(lens), case["heads"], d).to(dt), k_pages=k, v_pages=v, k_scale=ks, v_scale=vs, table=table,
                    lengths=torch.tensor(lens, dtype=torch.int32).cuda())
    # append: every sequence holds some tokens, whose last page its new rows may continue
    rng = random.Random(case["mix"] + 3)
    held = [rng.randint(0, 3 * page) for _ in lens]
    used = [_ceil(a + b, page) for a, b in zip(held, lens)]
    pool = sum(used) + 13
    order = torch.randperm(pool, generator=g, device="cuda")
    k, ks = _pool(g, pool, hk, page, d, dt, 8)
    v, vs = _pool(g, pool, hk, page, d, dt, 8)
    rows = _rows_of(lens)
    at = _places(lens) + torch.tensor(held).cuda()[rows]
    slots = order[torch.tensor(_starts(used)).cuda()[rows] + at // page] * page + at % page
    spread = 0.4 + _randn(g, 2, 1, hk, d, std=0.6).abs()
    new = _randn(g, 2, len(rows), hk, d) * spread
    return dict(k=new[0].to(dt), v=new[1].to(dt), k_pages=k, v_pages=v, k_scale=ks, v_scale=vs, slots=slots.to(torch.int32))


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if own and case["op"] == "window":
        from vmonarch_b200 import PackedSequences
        s["seqs"] = PackedSequences(s["ql"], s["kl"], device="cuda")
        if case["backward"]:
            for name in ("q", "k", "v"):
                s[name].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------- passes
def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](case, state)


def _own_window(case, s):
    from vmonarch_b200 import packed_attention
    o = packed_attention(s["q"], s["k"], s["v"], s["seqs"], causal=True, window=case["window"], sinks=case["sinks"])
    if not case["backward"]:
        return o
    return (o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"]))


def _own_decode(case, s):
    from vmonarch_b200 import paged_attention
    return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], k_scale=s["k_scale"],
                           v_scale=s["v_scale"], window=case["window"] or None, sinks=case["sinks"])


def _own_append(case, s):
    from vmonarch_b200 import append_pages
    append_pages(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _own_tables(case, s):
    from vmonarch_b200 import reserve_pages, truncate_pages
    truncate_pages(s["table"], s["lengths"], s["keep"], s["free"], s["num_free"], page_size=case["page"])
    slots = reserve_pages(s["table"], s["lengths"], s["counts"], s["free"], s["num_free"], page_size=case["page"],
                          total=s["total"])
    return slots, s["table"], s["lengths"], s["num_free"]


def _plain_window(case, s):
    h, hk, d, window, sinks = case["heads"], case["kv_heads"], case["dim"], case["window"], case["sinks"]
    group, scale, back = h // hk, d ** -0.5, case["backward"]
    dt = s["q"].dtype
    o = torch.zeros(s["q"].shape, device="cuda")
    dq, dk, dv = (torch.zeros(s[n].shape, device="cuda") for n in "qkv") if back else (None,) * 3
    for nq, nk, q0, k0 in zip(s["ql"], s["kl"], _starts(s["ql"]), _starts(s["kl"])):
        # as many queries at a time as fit with the keys that one of them sees, which are about window + sinks + queries
        step = max(1, min(nq, _CHUNK // (h * min(nk, 2 * (window + sinks) + 128)), window + sinks + 128))
        for i in range(0, nq, step):
            n, first = min(step, nq - i), nk - nq + i  # position of the first query
            low = max(0, first - window + 1)
            at = torch.arange(first + n, device="cuda")
            if low > sinks:
                at = torch.cat([at[:sinks], at[low:]])
            pos = torch.arange(first, first + n, device="cuda")[:, None]
            hide = (at > pos) | ((at <= pos - window) & (at >= sinks))
            rows = slice(q0 + i, q0 + i + n)
            k, v = (s[x][k0 + at].float().transpose(0, 1) for x in "kv")           # (hk, keys, d)
            q = s["q"][rows].float().view(n, hk, group, d).permute(1, 2, 0, 3).reshape(hk, group * n, d)
            p = q @ k.transpose(1, 2) * scale
            p.view(hk, group, n, -1).masked_fill_(hide, -math.inf)
            p = torch.exp(p - p.amax(2, keepdim=True))
            p /= p.sum(2, keepdim=True)
            o[rows] = (p @ v).view(hk, group, n, d).permute(2, 0, 1, 3).reshape(n, h, d)
            if back:
                do = s["do"][rows].float().view(n, hk, group, d).permute(1, 2, 0, 3).reshape(hk, group * n, d)
                dv.index_add_(0, k0 + at, (p.transpose(1, 2) @ do).transpose(0, 1))
                ds = do @ v.transpose(1, 2)
                ds = p * (ds - (p * ds).sum(2, keepdim=True)) * scale
                dq[rows] = (ds @ k).view(hk, group, n, d).permute(2, 0, 1, 3).reshape(n, h, d)
                dk.index_add_(0, k0 + at, (ds.transpose(1, 2) @ q).transpose(0, 1))
    return tuple(t.to(dt) for t in (o, dq, dk, dv)) if back else o.to(dt)


def _plain_decode(case, s):
    hk, d, page, window = case["kv_heads"], case["dim"], case["page"], case["window"]
    b, h, lengths = s["q"].size(0), case["heads"], s["lengths"].long()[:, None]
    if window and s["table"].size(1) > _ceil(window, page) + _ceil(case["sinks"], page) + 2:
        # only the pages that hold a visible token
        first = torch.arange(_ceil(case["sinks"], page), device="cuda").expand(b, -1)
        recent = torch.clamp(lengths - window, min=0) // page + torch.arange(_ceil(window, page) + 1, device="cuda")
        recent = torch.where(recent < first.size(1), s["table"].size(1), recent)  # those of the sinks are there already
        col = torch.cat([first, recent], 1)
    else:
        col = torch.arange(s["table"].size(1), device="cuda").expand(b, -1)
    pages = torch.gather(s["table"], 1, col.clamp(max=s["table"].size(1) - 1)).long()
    at = (col[..., None] * page + torch.arange(page, device="cuda")).reshape(b, -1)
    seen = at < lengths
    if window:
        seen &= (at >= lengths - window) | (at < case["sinks"])

    def read(pool, scale):
        x = pool[pages].float() if scale is None else pool.view(torch.uint8)[pages].view(_E4M3).float()
        if scale is not None:
            x *= scale[pages][..., None, None]
        return x.transpose(1, 2).reshape(b, hk, -1, d)

    q = s["q"].float().view(b, hk, h // hk, d)
    p = q @ read(s["k_pages"], s["k_scale"]).transpose(2, 3) * d ** -0.5
    p = p.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(p - p.amax(3, keepdim=True))
    o = (p / p.sum(3, keepdim=True)) @ read(s["v_pages"], s["v_scale"])
    return o.view(b, h, d).to(s["q"].dtype)


def _plain_append(case, s):
    page, at = (s["slots"] // case["page"]).long(), (s["slots"] % case["page"]).long()
    for x, pool, scale in ((s["k"], s["k_pages"], s["k_scale"]), (s["v"], s["v_pages"], s["v_scale"])):
        codes, x = pool.view(torch.uint8), x.float()
        top = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(2), "amax")
        fresh = torch.zeros_like(scale[:, 0], dtype=torch.bool)
        fresh[page[at == 0]] = True
        touched = torch.zeros_like(fresh)
        touched[page] = True
        need = _pow2_scale(top)
        new = torch.where(fresh[:, None], need, torch.maximum(scale, need))
        new = torch.where(touched[:, None], new, scale)
        grown = ((new > scale) & ~fresh[:, None]).nonzero(as_tuple=True)
        old = codes[grown].view(_E4M3).float() * (scale[grown] / new[grown])[:, None, None]
        codes[grown] = old.to(_E4M3).view(torch.uint8)
        codes[page, :, at] = (x / new[page][..., None]).to(_E4M3).view(torch.uint8)
        scale.copy_(new)
    return s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _plain_tables(case, s):
    page, table, lengths, free, num_free = case["page"], s["table"], s["lengths"], s["free"], s["num_free"]
    col = torch.arange(table.size(1), device="cuda")

    def between(low, high):  # the entries of a table that hold the tokens [low, high) beyond the page of low - 1
        return (col >= ((low + page - 1) // page)[:, None]) & (col < ((high + page - 1) // page)[:, None])

    kept = torch.minimum(lengths, s["keep"])
    back = table[between(kept, lengths)]
    free.index_copy_(0, num_free + torch.arange(back.numel(), device="cuda"), back.flip(0))
    num_free += back.numel()
    grown = kept + s["counts"]
    take = between(kept, grown)
    number = take.sum(dtype=torch.int32)
    order = take.flatten().cumsum(0).view(take.shape) - 1
    table.copy_(torch.where(take, free[(num_free - 1 - order).clamp(0, free.numel() - 1)], table))
    num_free -= number
    lengths.copy_(grown)
    ends = s["counts"].cumsum(0)
    row = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(ends, row, right=True)
    at = row - (ends - s["counts"])[seq] + kept[seq]
    slots = table[seq, at // page] * page + (at % page).to(torch.int32)
    return slots, table, lengths, num_free


_own = {"window": _own_window, "decode": _own_decode, "append": _own_append, "tables": _own_tables}
_plain = {"window": _plain_window, "decode": _plain_decode, "append": _plain_append, "tables": _plain_tables}


# -------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The outputs of :func:`run` in 64 bits, from each operator's definition; gradients by automatic differentiation of it,
    8-bit values as they are before their rounding. None for the tables, which are whole numbers."""
    if case["op"] == "tables":
        return None
    s = _inputs(case, seed)
    if case["op"] == "window":
        return _exact_window(case, s)
    if case["op"] == "append":
        return _exact_append(case, s)
    d, group, page, outs = case["dim"], case["heads"] // case["kv_heads"], case["page"], []
    for i, n in enumerate(s["lengths"].tolist()):
        at = torch.arange(n, device="cuda")
        if case["window"]:
            at = at[(at < case["sinks"]) | (n - 1 - at < case["window"])]
        where, slot = s["table"][i].long()[at // page], at % page
        for j in range(case["kv_heads"]):
            if case["bits"] == 8:
                k, v = (s[x + "_pages"].view(torch.uint8)[where, j, slot].view(_E4M3).double() * s[x + "_scale"][where, j, None].double()
                        for x in "kv")
            else:
                k, v = s["k_pages"][where, j, slot].double(), s["v_pages"][where, j, slot].double()
            x = s["q"][i, j * group:(j + 1) * group].double() @ k.T / math.sqrt(d)
            outs.append(torch.softmax(x, -1) @ v)
    return torch.cat(outs).view(s["q"].shape)


def _exact_append(case, s):
    page, slot = s["slots"].long() // case["page"], s["slots"].long() % case["page"]
    begun = torch.zeros(s["k_scale"].size(0), dtype=torch.bool, device="cuda")
    begun[page[slot == 0]] = True
    pools, scales = [], []
    for name in "kv":
        rows = s[name].double()
        values, was = s[name + "_pages"].double(), s[name + "_scale"].double()
        largest = torch.zeros_like(was).index_reduce_(0, page, rows.abs().amax(-1), "amax")
        needed = torch.exp2(torch.ceil(torch.log2(largest / 448)).clamp_min(-126))
        half = needed / 2  # a logarithm just above a whole number was a rounding
        needed = torch.where((half * 448 >= largest) & (half >= 2.0 ** -126), half, needed)
        hit = torch.zeros_like(begun)
        hit[page] = True
        now = torch.where(hit[:, None], torch.where(begun[:, None], needed, torch.maximum(was, needed)), was)
        values = torch.where(begun[:, None, None, None], values, values * (was / now)[..., None, None])
        values[page, :, slot] = rows / now[page][..., None]
        pools.append(values)
        scales.append(now)
    return (*pools, *scales)


def _exact_window(case, s):
    d, group, back = case["dim"], case["heads"] // case["kv_heads"], case["backward"]
    outs = [torch.zeros(s[n].shape, device="cuda", dtype=torch.float64) for n in (("q", "q", "k", "v") if back else "q")]
    q0 = k0 = 0
    for nq, nk in zip(s["ql"], s["kl"]):
        for i in range(0, nq, 8192):
            m = min(8192, nq - i)
            w = nk - nq + i + m                                   # keys up to the last of these queries
            ahead = torch.arange(w, device="cuda")[None] - torch.arange(w - m, w, device="cuda")[:, None]  # key - query
            mask = (ahead <= 0) & ((ahead > -case["window"]) | (torch.arange(w, device="cuda") < case["sinks"]))
            for j in range(case["heads"]):
                q = s["q"][q0 + i:q0 + i + m, j].double().requires_grad_(back)
                k = s["k"][k0:k0 + w, j // group].double().requires_grad_(back)
                v = s["v"][k0:k0 + w, j // group].double().requires_grad_(back)
                o = torch.softmax((q @ k.T / math.sqrt(d)).masked_fill(~mask, -math.inf), -1) @ v
                outs[0][q0 + i:q0 + i + m, j] = o.detach()
                if back:
                    gq, gk, gv = torch.autograd.grad(o, (q, k, v), s["do"][q0 + i:q0 + i + m, j].double())
                    outs[1][q0 + i:q0 + i + m, j] = gq
                    outs[2][k0:k0 + w, j // group] += gk
                    outs[3][k0:k0 + w, j // group] += gv
        q0, k0 = q0 + nq, k0 + nk
    return tuple(outs) if back else outs[0]
