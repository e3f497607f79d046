"""Attention over packed sequences of different lengths (no reference counterpart).

A batch of sequences is held as rows, one sequence after another: q is (total_q, H, D), k and v are
(total_k, Hk, D) with H a multiple of Hk (query head h reads key / value head h // (H // Hk)). The
lengths are known on the host, as a data loader or a scheduler knows them, and are turned once into
a :class:`PackedSequences`, which every layer of a step then shares.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import _native as N
from .kernel import SUPPORTED_DTYPES

#: head dims: multiples of 8 up to this
MAX_DIM = 128
_FWD_ROWS, _DQ_ROWS, _KV_ROWS, _STEP = 256, 128, 128, 64
_FIELDS = 12  # int32 per vmb_packed_unit
_NEVER_MASKED = -(1 << 30)


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


class PackedSequences:
    """The lengths of a batch of packed sequences, and the work lists made from them.

    Args:
        lengths: rows of each sequence (ints, or a tensor, which is read back to the host); zero is
            allowed.
        kv_lengths: keys of each sequence, where they differ from its queries (cross attention, a
            prompt behind a cached prefix); default: `lengths`.
        device: where the tensors of the sequences live.

    The object holds device copies of its work lists, made at the first call that needs them; keep it
    for as long as the lengths stand, e.g. for all layers of a step. It may be used on any stream.
    """

    def __init__(self, lengths, kv_lengths=None, device="cuda"):
        self.q_lens = _lengths(lengths, "lengths")
        self.k_lens = self.q_lens if kv_lengths is None else _lengths(kv_lengths, "kv_lengths")
        assert len(self.q_lens) == len(self.k_lens), "lengths and kv_lengths must name the same sequences"
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.total_q, self.total_k = int(self.q_lens.sum()), int(self.k_lens.sum())
        self.q_start = np.cumsum(self.q_lens) - self.q_lens
        self.k_start = np.cumsum(self.k_lens) - self.k_lens
        stat = -(-self.q_lens // _DQ_ROWS) * _DQ_ROWS
        self.stat_start, self.stat_rows = np.cumsum(stat) - stat, int(stat.sum())
        self._cache = {}

    @property
    def num_sequences(self) -> int:
        return len(self.q_lens)

    def __repr__(self):
        return f"PackedSequences({self.num_sequences} sequences, {self.total_q} queries, {self.total_k} keys)"

    def _starts(self):
        """First query row of every sequence, int32 on the device."""
        hit = self._cache.get("starts")
        if hit is None:
            hit = self._cache["starts"] = torch.from_numpy(self.q_start.astype(np.int32)).to(self.device)
        return hit

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
        return u

    def _list(self, kind, causal, heads, group):
        """The device list of a kernel's units, most work first (blocks start in list order)."""
        key = (kind, causal, group if kind == "kv" else 0)
        hit = self._cache.get(key)
        if hit is None:
            u = self._key_units(causal, group) if kind == "kv" else \
                self._query_units(_FWD_ROWS if kind == "fwd" else _DQ_ROWS, causal)
            u = u[np.argsort(u[:, 5] - u[:, 6], kind="stable")]
            dev = torch.from_numpy(np.ascontiguousarray(u)).to(self.device)
            hit = self._cache[key] = (N.PackedList(dev.data_ptr(), None, len(u), 0, 0, 0), dev)
        return hit[0]


def _in_place(t):
    """`t` when the kernels can address it: contiguous columns, 16-byte aligned rows and heads."""
    if t.stride(2) == 1 or t.size(2) == 1:
        if t.data_ptr() % 16 == 0 and all(
                n <= 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:2], t.stride()[:2])):
            return t
    return t.contiguous()


def _rows(t):
    return N.Rows(t.data_ptr(), t.stride(0) if t.size(0) > 1 else t.size(1) * t.size(2),
                  t.stride(1) if t.size(1) > 1 else t.size(2))


def _args(q, k, v, o, o_low, lse, seqs, causal, sm_scale):
    a = N.PackedArgs()
    a.q, a.k, a.v, a.o = _rows(q), _rows(k), _rows(v), _rows(o)
    a.lse = lse.data_ptr() if lse is not None else None
    if o_low is not None:
        a.o_low = _rows(o_low)
    a.q_total, a.k_total, a.stat_rows = seqs.total_q, seqs.total_k, seqs.stat_rows
    a.heads, a.kv_heads, a.dim = q.size(1), k.size(1), q.size(2)
    a.dtype, a.causal, a.sm_scale = N.dtype_code(q.dtype), causal, sm_scale
    return a


def _forward(q, k, v, seqs, causal, sm_scale, want_lse, want_low=False):
    q, k, v = _in_place(q), _in_place(k), _in_place(v)
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    o_low = torch.empty_like(o) if want_low else None
    lse = torch.empty((q.size(1), q.size(0)), dtype=torch.float32, device=q.device) if want_lse else None
    if o.numel():
        a = _args(q, k, v, o, o_low, lse, seqs, causal, sm_scale)
        a.units = seqs._list("fwd", causal, q.size(1), q.size(1) // k.size(1))
        N.check(N.lib.vmb_packed_fwd(ctypes.byref(a), N.stream_ptr(q.device)), "vmb_packed_fwd")
    return q, k, v, o, o_low, lse


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, seqs, causal, sm_scale):
        q, k, v, o, o_low, lse = _forward(q, k, v, seqs, causal, sm_scale, True, True)
        ctx.save_for_backward(q, k, v, o, o_low, lse)
        ctx.meta = seqs, causal, sm_scale
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, _):
        q, k, v, o, o_low, lse = ctx.saved_tensors
        seqs, causal, sm_scale = ctx.meta
        do = _in_place(do)
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        a = _args(q, k, v, o, o_low, lse, seqs, causal, sm_scale)
        a.dout, a.dq, a.dk, a.dv = _rows(do), _rows(dq), _rows(dk), _rows(dv)
        heads, group = q.size(1), q.size(1) // k.size(1)
        a.q_units = seqs._list("dq", causal, heads, group)
        a.kv_units = seqs._list("kv", causal, heads, group)
        nbytes = N.lib.vmb_packed_bwd_workspace_bytes(ctypes.byref(a))
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
        N.check(N.lib.vmb_packed_bwd(ctypes.byref(a), N.stream_ptr(q.device)), "vmb_packed_bwd")
        return dq, dk, dv, None, None, None


def packed_attention(q, k, v, seqs, *, causal=False, sm_scale=None, return_lse=False):
    """
    Softmax attention over packed sequences, differentiable in q, k and v.

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
    whole 64- or 128-row tile.
    """
    assert q.dtype in SUPPORTED_DTYPES, f"unsupported dtype {q.dtype}"
    assert k.dtype == q.dtype and v.dtype == q.dtype, "q, k and v must share a dtype"
    assert q.dim() == 3 and k.dim() == 3 and v.shape == k.shape and q.size(2) == k.size(2), \
        "q must be (total_q, H, D), k and v (total_k, Hk, D)"
    d = q.size(2)
    assert 8 <= d <= MAX_DIM and d % 8 == 0, f"head dim {d} is not a multiple of 8 up to {MAX_DIM}"
    assert k.size(1) >= 1 and q.size(1) >= 1 and q.size(1) % k.size(1) == 0, "H must be a multiple of Hk"
    assert q.is_cuda and k.device == q.device and v.device == q.device and seqs.device == q.device, \
        "q, k, v and seqs must be on one CUDA device"
    assert q.size(0) == seqs.total_q and k.size(0) == seqs.total_k, \
        f"q and k have {q.size(0)} and {k.size(0)} rows, the sequences {seqs.total_q} and {seqs.total_k}"
    sm_scale = d ** -0.5 if sm_scale is None else float(sm_scale)
    assert 0 <= sm_scale < float("inf"), "sm_scale must be finite and not negative"
    causal = bool(causal)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        o, lse = _PackedAttention.apply(q, k, v, seqs, causal, sm_scale)
    else:
        *_, o, _, lse = _forward(q, k, v, seqs, causal, sm_scale, return_lse)
    return (o, lse) if return_lse else o
