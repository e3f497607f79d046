"""The elementwise and normalising work between two blocks of a transformer, fused (no reference
counterpart): a norm after the block, its gate, the residual, and the modulated norm before the next block.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _native as N
from .kernel import SUPPORTED_DTYPES

#: widths: multiples of 8 up to this
MAX_WIDTH = 8192


def _place(t, rows, cols):
    """`t` (rows, cols), or a dense copy where the kernels cannot address it in place (contiguous columns, 16-byte
    aligned rows), and its vmb_matrix."""
    ptr, (row, col) = t.data_ptr(), t.stride()
    if rows <= 1:
        row = cols
    if col != 1 or row < 0 or row & 7 or ptr & 15:
        t = _dense(t.contiguous())
        ptr, row = t.data_ptr(), cols
    return t, ptr, row


def _dense(t):
    return t if t.is_contiguous() and not t.data_ptr() & 15 else t.clone(memory_format=torch.contiguous_format)


_PARAMS = ("gate", "scale", "shift", "weight", "post_weight")
_WEIGHTS = ("weight", "post_weight")
# vmb_gated_norm_args up to its workspace: x, y, x_new, h, five parameters, stats, seq_start | dx_new, dh, dx, dy,
# five gradients | sizes
_ARGS = struct.Struct("25q5if")
assert _ARGS.size == N.GatedNormArgs.workspace.offset
_NO_GRADS = (0,) * 11
_NO_ROWS = None, 0, 0


def _forward(x, y, params, seqs, sizes, stats):
    rows, cols = sizes[:2]
    x, x_ptr, x_row = _place(x, rows, cols)
    y, y_ptr, y_row = _NO_ROWS if y is None else _place(y, rows, cols)
    x_new = None if y is None else torch.empty_like(x, memory_format=torch.contiguous_format)
    h = torch.empty_like(x, memory_format=torch.contiguous_format)
    a = N.GatedNormArgs()
    _ARGS.pack_into(a, 0, x_ptr, x_row, y_ptr, y_row, 0 if x_new is None else x_new.data_ptr(), h.data_ptr(),
                    *[0 if t is None else t.data_ptr() for t in params], 0 if stats is None else stats.data_ptr(),
                    seqs._starts().data_ptr() if sizes[2] > 1 else 0, *_NO_GRADS, *sizes)
    N.launch("vmb_gated_norm_fwd", N.lib.vmb_gated_norm_fwd, x.device, ctypes.byref(a))
    return x, y, x_new, h


class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, seqs, sizes, *params):
        stats = torch.empty(3 * sizes[0], dtype=torch.float32, device=x.device)
        x, y, x_new, h = _forward(x, y, params, seqs, sizes, stats)
        ctx.save_for_backward(x, y, stats, *params)
        ctx.meta = seqs, sizes
        ctx.set_materialize_grads(False)
        return (h,) if y is None else (x_new, h)

    @staticmethod
    @N.once_differentiable
    def backward(ctx, *grads):
        x, y, stats, *params = ctx.saved_tensors
        seqs, sizes = ctx.meta
        rows, cols = sizes[:2]
        dx_new, dh = (None, *grads) if y is None else grads
        dx_new, dxn_ptr, dxn_row = _NO_ROWS if dx_new is None else _place(dx_new, rows, cols)
        dh, dh_ptr, dh_row = _NO_ROWS if dh is None else _place(dh, rows, cols)
        _, x_ptr, x_row = _place(x, rows, cols)
        _, y_ptr, y_row = _NO_ROWS if y is None else _place(y, rows, cols)
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
        dy = None if y is None else torch.empty_like(x, memory_format=torch.contiguous_format)
        out = [torch.empty_like(t) if need and t is not None else None for t, need in zip(params, ctx.needs_input_grad[4:])]
        a = N.GatedNormArgs()
        _ARGS.pack_into(a, 0, x_ptr, x_row, y_ptr, y_row, 0, 0, *[0 if t is None else t.data_ptr() for t in params],
                        stats.data_ptr(), seqs._starts().data_ptr() if sizes[2] > 1 else 0, dxn_ptr, dxn_row, dh_ptr, dh_row,
                        dx.data_ptr(), 0 if dy is None else dy.data_ptr(),
                        *[0 if t is None else t.data_ptr() for t in out], *sizes)
        size = N.lib.vmb_gated_norm_bwd_workspace_bytes(ctypes.byref(a))
        if size > 0:
            ws = torch.empty(size, dtype=torch.uint8, device=x.device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), size
        N.launch("vmb_gated_norm_bwd", N.lib.vmb_gated_norm_bwd, x.device, ctypes.byref(a))
        return (dx, dy, None, None, *out)


def gated_residual_norm(x, y=None, *, gate=None, scale=None, shift=None, weight=None, post_weight=None, norm="rms",
                        eps=1e-6, seqs=None):
    """
    x_new = x + gate * y', h = norm(x_new) * weight * (1 + scale) + shift; differentiable in every tensor (backward only).

    Args:
        x: (T, C) residual stream, bf16 or fp16, C a multiple of 8 up to 8192
        y: (T, C) output of the block that ends, or None (the first norm of a model)
        gate, scale, shift: one row per sequence, (S, C), or without `seqs` (C,) or (1, C); a missing gate is
            1, a missing scale or shift 0
        weight: (C,) of the norm before the next block
        post_weight: (C,) of an rms norm of y before the gate; without it y' = y
        norm: "rms", or "layer" (mean taken off); both over C, without a bias of their own
        eps: added to the mean square (both norms of a call)
        seqs: the :class:`PackedSequences` whose queries are the rows, where gate, scale or shift differ
            from sequence to sequence. A (B, N, C) batch is x.flatten(0, 1) with PackedSequences([N] * B).
        The parameters share one dtype: x's, or fp32.
    Returns:
        (x_new, h), both (T, C) in x's dtype; with y None (x, h)
    All arithmetic is 32-bit; h is formed from x_new before its rounding.
    """
    kind, device, shape = x.dtype, x.device, x.shape
    assert kind in SUPPORTED_DTYPES, f"unsupported dtype {kind}"
    assert len(shape) == 2, "x must be (T, C)"
    rows, c = shape
    assert 8 <= c <= MAX_WIDTH and c % 8 == 0, f"width {c} is not a multiple of 8 up to {MAX_WIDTH}"
    assert y is None or (y.shape == shape and y.dtype == kind and y.device == device), "y must be like x"
    assert y is not None or (gate is None and post_weight is None), "gate and post_weight need y"
    assert norm in ("rms", "layer"), f"norm must be 'rms' or 'layer', not {norm!r}"
    eps = float(eps)
    assert 0 <= eps < float("inf"), "eps must be finite and not negative"
    assert x.is_cuda, "vmonarch_b200 needs CUDA tensors"
    count = 1
    if seqs is not None:
        count = seqs.num_sequences
        assert seqs.device == device, "x and seqs must be on one CUDA device"
        assert seqs.total_q == rows, f"x has {rows} rows, the sequences {seqs.total_q}"
        assert count <= 65535, "at most 65535 sequences"
    needed = x.requires_grad or (y is not None and y.requires_grad)
    params, dtype, wide, tall = [], None, (c,), (count, c)
    for name, t in zip(_PARAMS, (gate, scale, shift, weight, post_weight)):
        if t is not None:
            assert t.device == device, f"{name} must be on x's device"
            if t.dtype != dtype:
                assert dtype is None and t.dtype in (kind, torch.float32), "the parameters must share one dtype, x's or fp32"
                dtype = t.dtype
            if seqs is None:
                assert t.shape == wide or t.shape == tall, f"{name} must be ({c},)"
            elif name in _WEIGHTS:
                assert t.shape == wide, f"{name} must be ({c},)"
            else:
                assert t.shape == tall, f"{name} must be ({count}, {c})"
            needed = needed or t.requires_grad
            if t.data_ptr() & 15 or not t.is_contiguous():
                t = _dense(t)
        params.append(t)
    code = N.dtype_code(kind)
    sizes = (rows, c, count, code, N.VMB_DTYPE_F32 if dtype == torch.float32 else code, norm == "layer", eps)
    if N.derived(needed):
        out = _GatedNorm.apply(x, y, seqs, sizes, *params)
        return (x, out[0]) if y is None else out
    x_new, h = _forward(x, y, params, seqs, sizes, None)[2:]
    return (x if y is None else x_new), h
