"""Attention over packed sequences of different lengths (no reference counterpart).

A batch of sequences is held as rows, one sequence after another: q is (total_q, H, D), k and v are
(total_k, Hk, D) with H a multiple of Hk (query head h reads key / value head h // (H // Hk)). The
lengths are known on the host, as a data loader or a scheduler knows them, and are turned once into
a :class:`PackedSequences`, which every layer of a step then shares.
"""
from __future__ import annotations

import ctypes
import heapq
import struct
import threading

import numpy as np
import torch

from . import _native as N
from .kernel import SUPPORTED_DTYPES

#: head dims: multiples of 8 up to this
MAX_DIM = 128
_FWD_ROWS, _DQ_ROWS, _KV_ROWS, _STEP = 256, 128, 128, 64
_FIELDS = 12  # int32 per vmb_packed_unit
_NEVER_MASKED = -(1 << 30)
_SMS = 148
# least steps of a piece when a unit is cut: below it, set-up and join cost more than the cut gains
_LEAST = {"fwd": 8, "dq": 8, "kv": 16}
# measured, in steps (of 1.1 to 2 us): what a unit costs beside its own and what a piece of one costs more, and the
# kernel that joins the pieces: its launch, and how many pieces it joins in a step
_SETUP, _PIECE, _JOIN, _JOINED = {"fwd": 3, "dq": 5, "kv": 8}, 3, 3, 40
# lists of more blocks than this (eight for each SM) are even enough without looking
_MANY = 8 * _SMS
# held while something is added to what a PackedSequences keeps: two threads that made the same list would each hold one
_making = threading.RLock()


def _lengths(x, what):
    if isinstance(x, torch.Tensor):
        x = x.tolist()
    a = np.asarray(list(x), dtype=np.int64)
    assert a.ndim == 1 and len(a) >= 1, f"{what} must be a list of at least one length"
    assert (a >= 0).all(), f"{what} must not be negative"
    assert a.sum() < 2 ** 31, f"{what} add up to more than 2^31 - 1 rows"
    return a


def _tiles(lens, rows):
    """(sequence, first local row) of every `rows`-row tile of sequences of the given lengths."""
    count = -(-lens // rows)
    seq = np.repeat(np.arange(len(lens)), count)
    first = (np.arange(len(seq)) - np.repeat(np.cumsum(count) - count, count)) * rows
    return seq, first


def _span(steps, heads, setup):
    """Steps until the last SM is done, when units of -`steps` steps start in list order wherever an SM is free."""
    load = [0] * _SMS
    for n in steps.tolist():
        n = setup - n
        for _ in range(heads):
            heapq.heapreplace(load, load[0] + n)
    return max(load)


def _pieces(steps, limit):
    """How many equal pieces of about `limit` steps each unit makes."""
    return np.maximum(-(-steps // limit), 1)


def _piece_steps(steps, pieces):
    which = np.repeat(np.arange(len(steps)), pieces)
    k = np.arange(len(which)) - np.repeat(np.cumsum(pieces) - pieces, pieces)  # piece of its unit
    n, total = pieces[which], steps[which]
    return which, k, total * k // n, total * (k + 1) // n


def _cut(u, heads, kind):
    """Cuts the units of a list into equal pieces, so far as the SMs finish sooner by it: the pieces' set-up
    and their join included. Returns the list and its number of pieces (parts)."""
    steps = u[:, 6].astype(np.int64)
    if not len(u):
        return u, 0
    least, setup = _LEAST[kind], _SETUP[kind]
    total = int(steps.sum()) * heads
    share = max(-(-total // _SMS), 1)
    limits = [max(least, -(-share * n // 8)) for n in (11, 10, 9, 8, 4, 2)]
    best = _pieces(steps, limits[1])  # a unit far above everybody's fair share is cut in any case
    if len(u) * heads <= _MANY:
        best, best_cost = None, 0
        for limit in dict.fromkeys([int(steps.max()) + 1, *limits]):
            pieces = _pieces(steps, limit)
            if best is not None and (best_cost <= 1.03 * (share + setup) or pieces.max() == 1):
                continue
            cuts = int(pieces[pieces > 1].sum()) * heads
            join = _JOIN + cuts // _JOINED if cuts else 0
            evenly = (total + setup * int(pieces.sum()) * heads + _PIECE * cuts) // _SMS + join
            if best is not None and evenly >= 0.98 * best_cost:
                continue  # even if it ended evenly
            which, _, begin, end = _piece_steps(steps, pieces)
            cost = _span(np.sort(begin - end - _PIECE * (pieces[which] > 1)), heads, setup) + join
            if best is None or cost < 0.98 * best_cost:
                best, best_cost = pieces, cost
    if best.max() == 1:
        return u, 0
    which, k, begin, end = _piece_steps(steps, best)
    out = u[which]
    out[:, 5], out[:, 6] = begin, end
    is_part = best[which] > 1
    out[is_part, 7] = np.arange(int(is_part.sum()))
    out[:, 9] = np.where(k == 0, best[which], 0)  # for _joins; the kernels do not read it
    return out, int(is_part.sum())


def _joins(u):
    """(first unit, pieces) of every cut unit of a list."""
    first = np.nonzero((u[:, 7] >= 0) & (u[:, 9] > 0))[0]
    return np.stack([first, u[first, 9]], 1).astype(np.int32)


class PackedSequences:
    """The lengths of a batch of packed sequences, and the work lists made from them.

    Args:
        lengths: rows of each sequence (ints, or a tensor, which is read back to the host); zero is
            allowed.
        kv_lengths: keys of each sequence, where they differ from its queries (cross attention, a
            prompt behind a cached prefix); default: `lengths`.
        device: where the tensors of the sequences live.

    The object holds device copies of its work lists, made at the first call of each kind (direction, causal, head
    counts), which waits for the copy; keep it for as long as the lengths stand, e.g. for all layers of a step. It may
    be used on any stream and by several threads. A captured graph reads the lists where they are: make one call of
    each kind before the capture, and keep the object for as long as the graph.
    """

    def __init__(self, lengths, kv_lengths=None, device="cuda"):
        self.q_lens = _lengths(lengths, "lengths")
        self.k_lens = self.q_lens if kv_lengths is None else _lengths(kv_lengths, "kv_lengths")
        assert len(self.q_lens) == len(self.k_lens), "lengths and kv_lengths must name the same sequences"
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._index = self.device.index if self.device.type == "cuda" else None
        self.total_q, self.total_k = int(self.q_lens.sum()), int(self.k_lens.sum())
        self.q_start = np.cumsum(self.q_lens) - self.q_lens
        self.k_start = np.cumsum(self.k_lens) - self.k_lens
        stat = -(-self.q_lens // _DQ_ROWS) * _DQ_ROWS
        self.stat_start, self.stat_rows = np.cumsum(stat) - stat, int(stat.sum())
        self._cache = {}
        self._home = None  # the stream on which all that is kept was allocated; None: there is none, or several

    @property
    def num_sequences(self) -> int:
        return len(self.q_lens)

    def __repr__(self):
        return f"PackedSequences({self.num_sequences} sequences, {self.total_q} queries, {self.total_k} keys)"

    def _kept(self, key, make, *args):
        """What is kept under `key`, made by make(*args) at the first call."""
        hit = self._cache.get(key)
        if hit is None:
            with _making:
                hit = self._cache.get(key)
                if hit is None:
                    hit = self._cache[key] = make(*args)
        return hit

    def _stream(self):
        """Handle of the device's current stream."""
        return 0 if self._index is None else N.raw_stream(self._index)

    def _on_device(self, array):
        assert self.device.type != "cuda" or not torch.cuda.is_current_stream_capturing(), \
            "the first call of a kind with these sequences copies their lists: make one before the capture"
        stream = self._stream()
        self._home = stream if not self._cache or stream == self._home else None
        return torch.from_numpy(array).to(self.device)

    def _use(self, tensors):
        """Kept tensors that the current stream is about to read: where they belong to another, the allocator learns that
        their memory stays in use here, whenever the object goes."""
        if self._stream() != self._home:
            stream = torch.cuda.current_stream(self.device)
            for t in tensors:
                t.record_stream(stream)

    def _starts(self):
        """First query row of every sequence, int32 on the device."""
        starts = self._cache.get("starts")
        if starts is None:
            starts = self._kept("starts", lambda: self._on_device(self.q_start.astype(np.int32)))
        self._use((starts,))
        return starts

    # ------------------------------------------------------------------------------ work lists
    def _query_units(self, rows, causal):
        """Units of `rows` queries for the forward and dQ kernels, and their key tiles."""
        seq, first = _tiles(self.q_lens, rows)
        nq, nk = self.q_lens[seq], self.k_lens[seq]
        u = np.zeros((len(seq), _FIELDS), dtype=np.int32)
        valid = np.minimum(nq - first, rows)
        vis0 = nk - nq + first + 1 if causal else nk
        u[:, 0], u[:, 1], u[:, 2], u[:, 3] = self.q_start[seq] + first, valid, self.k_start[seq], nk
        u[:, 4] = vis0
        seen = np.clip(vis0 + (valid - 1 if causal else 0), 0, nk)
        u[:, 6] = -(-seen // 128)
        u[:, 7] = -1
        u[:, 8] = self.stat_start[seq] + first
        return u

    def _key_units(self, causal, group):
        """Units of 128 keys for the dK / dV kernel and their (head, query tile) steps."""
        seq, first = _tiles(self.k_lens, _KV_ROWS)
        nq, nk = self.q_lens[seq], self.k_lens[seq]
        u = np.zeros((len(seq), _FIELDS), dtype=np.int32)
        vis0 = first - (nk - nq) if causal else np.full_like(first, _NEVER_MASKED)
        u[:, 0], u[:, 1] = self.q_start[seq], nq
        u[:, 2], u[:, 3] = self.k_start[seq] + first, np.minimum(nk - first, _KV_ROWS)
        u[:, 4] = vis0
        u[:, 6] = group * np.maximum(-(-nq // _STEP) - np.maximum(vis0, 0) // _STEP, 0)
        u[:, 7] = -1
        u[:, 8] = self.stat_start[seq]
        # queries below this one see one key at most, and a softmax over one key has no gradient
        u[:, 10] = np.maximum(nq - nk + 1, 0) if causal else np.where(nk == 1, nq, 0)
        return u

    def _list(self, *key):
        """The device list of a kernel's units, most work first (blocks start in list order), then the joins
        of those that are cut. key: kind, causal, heads, group."""
        return self._kept(key, self._make_list, *key)[0]

    def _make_list(self, kind, causal, heads, group):
        if kind == "kv":
            u = self._key_units(causal, group)
            u, parts = _cut(u, heads // group, kind)
        else:
            u = self._query_units(_FWD_ROWS if kind == "fwd" else _DQ_ROWS, causal)
            u, parts = _cut(u, heads, kind)
        u = u[np.argsort(u[:, 5] - u[:, 6], kind="stable")]
        joins = _joins(u)
        dev = self._on_device(np.concatenate([u.reshape(-1), joins.reshape(-1)]))
        at = dev.data_ptr()
        return N.PackedList(at, at + u.nbytes if len(joins) else None, len(u), len(joins), parts, 0), dev

    def _template(self, key):
        """vmb_packed_args of a kind of call, everything but the tensors, its workspace size, and the device lists
        that it names."""
        hit = self._cache.get(key)
        return self._kept(key, self._make_template, *key) if hit is None else hit

    def _make_template(self, backward, causal, sm_scale, dtype, heads, kv_heads, dim):
        assert not backward or self.stat_rows < 2 ** 31, \
            f"the backward's statistics have 32-bit rows: {self.num_sequences} sequences padded to 128 rows each are too many"
        a = N.PackedArgs()
        a.q_total, a.k_total, a.stat_rows = self.total_q, self.total_k, self.stat_rows
        a.heads, a.kv_heads, a.dim = heads, kv_heads, dim
        a.dtype, a.causal, a.sm_scale = N.dtype_code(dtype), causal, sm_scale
        lists = [(kind, causal, heads, heads // kv_heads) for kind in (("dq", "kv") if backward else ("fwd",))]
        if backward:
            a.q_units, a.kv_units = (self._list(*x) for x in lists)
            size = N.lib.vmb_packed_bwd_workspace_bytes(ctypes.byref(a))
        else:
            a.units = self._list(*lists[0])
            size = N.lib.vmb_packed_fwd_workspace_bytes(ctypes.byref(a))
        return bytes(a), size, tuple(self._cache[x][1] for x in lists)


# vmb_packed_args begins with the vmb_rows of q, k, v, o, dout, dq, dk, dv, o_low and lse
_FWD_TENSORS = struct.Struct("12q")
_REST = struct.Struct("16q")
_REST_AT = _FWD_TENSORS.size
_WORKSPACE = struct.Struct("2q")
_WORKSPACE_AT = N.PackedArgs.workspace.offset


def _place(t):
    """`t` (rows, heads, dim), or a dense copy where the kernels cannot address it in place (contiguous
    columns, 16-byte aligned rows and heads), and its vmb_rows."""
    ptr, (row, head, col) = t.data_ptr(), t.stride()
    if col == 1 and row > 0 and head > 0 and not (row | head) & 7 and not ptr & 15:
        return t, ptr, row, head
    n, h, d = t.shape
    row, head = row if n > 1 else h * d, head if h > 1 else d  # strides of single rows and heads do not count
    if not (col == 1 or d == 1) or row <= 0 or head <= 0 or (row | head) & 7 or ptr & 15:
        t = t.contiguous()
        if t.data_ptr() & 15:
            t = t.clone(memory_format=torch.contiguous_format)
        ptr, row, head = t.data_ptr(), h * d, d
    return t, ptr, row, head


def _forward(q, k, v, seqs, key, device, lse=None, aux=None):
    """Runs the forward into a new o. `aux`: the bytes kept for a backward, o_low and then (unless `lse` is
    given) the statistics."""
    q, *qr = _place(q)
    k, *kr = _place(k)
    v, *vr = _place(v)
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    template, size, lists = seqs._template(key)
    seqs._use(lists)
    a = N.PackedArgs.from_buffer_copy(template)
    heads, dim = key[4], key[6]
    row = heads * dim
    _FWD_TENSORS.pack_into(a, 0, *qr, *kr, *vr, o.data_ptr(), row, dim)
    if aux is not None or lse is not None:
        low = aux.data_ptr() if aux is not None else 0
        stat = lse.data_ptr() if lse is not None else low + 2 * seqs.total_q * row
        _REST.pack_into(a, _REST_AT, *_NO_ROWS, low, row, dim, stat)
    if size:
        ws = torch.empty(size, dtype=torch.uint8, device=device)
        _WORKSPACE.pack_into(a, _WORKSPACE_AT, ws.data_ptr(), size)
    N.launch("vmb_packed_fwd", N.lib.vmb_packed_fwd, device, ctypes.byref(a))
    return q, k, v, o


_NO_ROWS = (0,) * 12  # dout, dq, dk, dv of a forward


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, seqs, key, return_lse):
        device, rows, heads, dim = q.device, seqs.total_q, key[4], key[6]
        lse = torch.empty((heads, rows), dtype=torch.float32, device=device) if return_lse else None
        # o_low (16-bit) and the statistics behind it, in one buffer
        aux = torch.empty(rows * heads * (2 * dim + (0 if return_lse else 4)), dtype=torch.uint8, device=device)
        q, k, v, o = _forward(q, k, v, seqs, key, device, lse, aux)
        ctx.save_for_backward(q, k, v, o, aux, *([lse] if return_lse else []))
        ctx.meta = seqs, key
        if not return_lse:
            return o
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    @N.once_differentiable
    def backward(ctx, do, _=None):
        q, k, v, o, aux, *lse = ctx.saved_tensors
        seqs, key = ctx.meta
        heads, kv_heads, dim = key[4:]
        row, kv_row, device = heads * dim, kv_heads * dim, q.device
        do, *dor = _place(do)
        dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
        template, size, lists = seqs._template((True, *key[1:]))
        seqs._use(lists)
        a = N.PackedArgs.from_buffer_copy(template)
        _FWD_TENSORS.pack_into(a, 0, *_place(q)[1:], *_place(k)[1:], *_place(v)[1:], o.data_ptr(), row, dim)
        low = aux.data_ptr()
        stat = lse[0].data_ptr() if lse else low + 2 * seqs.total_q * row
        _REST.pack_into(a, _REST_AT, *dor, dq.data_ptr(), row, dim, dk.data_ptr(), kv_row, dim, dv.data_ptr(), kv_row, dim,
                        low, row, dim, stat)
        if size:
            ws = torch.empty(size, dtype=torch.uint8, device=device)
            _WORKSPACE.pack_into(a, _WORKSPACE_AT, ws.data_ptr(), size)
        N.launch("vmb_packed_bwd", N.lib.vmb_packed_bwd, device, ctypes.byref(a))
        return dq, dk, dv, None, None, None


def packed_attention(q, k, v, seqs, *, causal=False, sm_scale=None, return_lse=False):
    """
    Softmax attention over packed sequences, differentiable in q, k and v (backward only).

    Args:
        q: (total_q, H, D), bf16 or fp16, D a multiple of 8 up to 128
        k, v: (total_k, Hk, D), the same dtype, H a multiple of Hk
        seqs: the sequences' lengths, a :class:`PackedSequences` on the same device
        causal: query i of a sequence of nq queries and nk keys sees its first nk - nq + i + 1 keys
        sm_scale: softmax scale, not negative; defaults to 1 / sqrt(D)
        return_lse: also return the log of each softmax's sum
    Returns:
        o: (total_q, H, D); a query that sees no key has o = 0
        lse (with return_lse): (H, total_q) float32, natural logarithm, -inf where no key is seen;
            carries no gradient
    Views with contiguous columns and 16-byte aligned rows and heads (slices of a packed QKV
    projection) are read in place, others through a dense copy. Rows of other sequences and keys that
    a query does not see take no part, whatever they hold; in the backward pass that covers other
    sequences' rows, while within a sequence a value that is not finite reaches the gradients of its
    whole 64- or 128-row tile. The fp16 backward needs value rows with a norm below 4094.
    """
    dtype = q.dtype
    assert dtype in SUPPORTED_DTYPES, f"unsupported dtype {dtype}"
    assert k.dtype == dtype and v.dtype == dtype, "q, k and v must share a dtype"
    assert q.dim() == 3 and k.dim() == 3 and v.shape == k.shape and q.size(2) == k.size(2), \
        "q must be (total_q, H, D), k and v (total_k, Hk, D)"
    rows, heads, d = q.shape
    kv_rows, kv_heads, _ = k.shape
    assert 8 <= d <= MAX_DIM and d % 8 == 0, f"head dim {d} is not a multiple of 8 up to {MAX_DIM}"
    assert kv_heads >= 1 and heads >= 1 and heads % kv_heads == 0, "H must be a multiple of Hk"
    device = q.device
    assert q.is_cuda and k.device == device and v.device == device and seqs.device == device, \
        "q, k, v and seqs must be on one CUDA device"
    assert rows == seqs.total_q and kv_rows == seqs.total_k, \
        f"q and k have {rows} and {kv_rows} rows, the sequences {seqs.total_q} and {seqs.total_k}"
    sm_scale = d ** -0.5 if sm_scale is None else float(sm_scale)
    assert 0 <= sm_scale < float("inf"), "sm_scale must be finite and not negative"
    key = (False, bool(causal), sm_scale, dtype, heads, kv_heads, d)
    if N.derived(q.requires_grad or k.requires_grad or v.requires_grad):
        return _PackedAttention.apply(q, k, v, seqs, key, return_lse)
    lse = torch.empty((heads, rows), dtype=torch.float32, device=device) if return_lse else None
    o = _forward(q, k, v, seqs, key, device, lse)[3]
    return (o, lse) if return_lse else o
