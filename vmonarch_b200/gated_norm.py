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


def _place(t):
    """`t` (T, C), or a dense copy where the kernels cannot address it in place (contiguous columns, 16-byte
    aligned rows), and its vmb_matrix."""
    ptr, (row, col) = t.data_ptr(), t.stride()
    n, c = t.shape
    if n <= 1:
        row = c
    if col != 1 or row < 0 or row & 7 or ptr & 15:
        t = _dense(t.contiguous())
        ptr, row = t.data_ptr(), c
    return t, ptr, row


def _dense(t):
    return t if t.is_contiguous() and not t.data_ptr() & 15 else t.clone(memory_format=torch.contiguous_format)


_PARAMS = ("gate", "scale", "shift", "weight", "post_weight")
# vmb_gated_norm_args up to its workspace: x, y, x_new, h, five parameters, stats, seq_start | dx_new, dh, dx, dy,
# five gradients | sizes
_ARGS = struct.Struct("25q5if")
assert _ARGS.size == N.GatedNormArgs.workspace.offset
_NO_GRADS = (0,) * 11


def _sizes(x, params, seqs, norm, eps):
    dtype = N.dtype_code(x.dtype)
    fp32 = any(t is not None and t.dtype == torch.float32 for t in params)
    rows, cols = x.shape
    return rows, cols, 1 if seqs is None else seqs.num_sequences, dtype, N.VMB_DTYPE_F32 if fp32 else dtype, norm == "layer", eps


def _starts(seqs):
    return seqs._starts().data_ptr() if seqs is not None and seqs.num_sequences > 1 else 0


def _forward(x, y, params, seqs, norm, eps, stats):
    x, *xr = _place(x)
    yr = (0, 0)
    if y is not None:
        y, *yr = _place(y)
    params = [t if t is None else _dense(t) for t in params]
    x_new = torch.empty_like(x, memory_format=torch.contiguous_format) if y is not None else None
    h = torch.empty_like(x, memory_format=torch.contiguous_format)
    a = N.GatedNormArgs()
    _ARGS.pack_into(a, 0, *xr, *yr, 0 if x_new is None else x_new.data_ptr(), h.data_ptr(),
                    *[0 if t is None else t.data_ptr() for t in params], 0 if stats is None else stats.data_ptr(),
                    _starts(seqs), *_NO_GRADS, *_sizes(x, params, seqs, norm, eps))
    rc = N.lib.vmb_gated_norm_fwd(ctypes.byref(a), N.raw_stream(x.device.index))
    if rc:
        N.check(rc, "vmb_gated_norm_fwd")
    return x, y, params, x_new, h


class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, seqs, norm, eps, *params):
        shapes = [None if t is None else t.shape for t in params]
        stats = torch.empty((3, x.size(0)), dtype=torch.float32, device=x.device)
        x, y_in, dense, x_new, h = _forward(x, y, params, seqs, norm, eps, stats)
        ctx.save_for_backward(x, y_in, stats, *dense)
        ctx.meta = seqs, norm, eps, shapes
        ctx.set_materialize_grads(False)
        return (h,) if y is None else (x_new, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        x, y, stats, *params = ctx.saved_tensors
        seqs, norm, eps, shapes = ctx.meta
        dx_new, dh = grads if y is not None else (None, *grads)
        dxr = dhr = yr = (0, 0)
        if dx_new is not None:
            dx_new, *dxr = _place(dx_new)
        if dh is not None:
            dh, *dhr = _place(dh)
        if y is not None:
            yr = _place(y)[1:]
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
        dy = torch.empty_like(x, memory_format=torch.contiguous_format) if y is not None else None
        out = [torch.empty(shape, dtype=t.dtype, device=x.device) if t is not None and need else None
               for t, need, shape in zip(params, ctx.needs_input_grad[5:], shapes)]
        a = N.GatedNormArgs()
        _ARGS.pack_into(a, 0, *_place(x)[1:], *yr, 0, 0, *[0 if t is None else t.data_ptr() for t in params],
                        stats.data_ptr(), _starts(seqs), *dxr, *dhr, dx.data_ptr(), 0 if dy is None else dy.data_ptr(),
                        *[0 if t is None else t.data_ptr() for t in out], *_sizes(x, params, seqs, norm, eps))
        size = N.lib.vmb_gated_norm_bwd_workspace_bytes(ctypes.byref(a))
        if size > 0:
            ws = torch.empty(size, dtype=torch.uint8, device=x.device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), size
        rc = N.lib.vmb_gated_norm_bwd(ctypes.byref(a), N.raw_stream(x.device.index))
        if rc:
            N.check(rc, "vmb_gated_norm_bwd")
        return (dx, dy, None, None, None, *out)


def gated_residual_norm(x, y=None, *, gate=None, scale=None, shift=None, weight=None, post_weight=None, norm="rms",
                        eps=1e-6, seqs=None):
    """
    x_new = x + gate * y', h = norm(x_new) * weight * (1 + scale) + shift; differentiable in every tensor.

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
    assert x.dtype in SUPPORTED_DTYPES, f"unsupported dtype {x.dtype}"
    assert x.dim() == 2, "x must be (T, C)"
    c = x.size(1)
    assert 8 <= c <= MAX_WIDTH and c % 8 == 0, f"width {c} is not a multiple of 8 up to {MAX_WIDTH}"
    assert y is None or (y.shape == x.shape and y.dtype == x.dtype and y.device == x.device), "y must be like x"
    assert y is not None or (gate is None and post_weight is None), "gate and post_weight need y"
    assert norm in ("rms", "layer"), f"norm must be 'rms' or 'layer', not {norm!r}"
    eps = float(eps)
    assert 0 <= eps < float("inf"), "eps must be finite and not negative"
    assert x.is_cuda, "vmonarch_b200 needs CUDA tensors"
    if seqs is not None:
        assert seqs.device == x.device, "x and seqs must be on one CUDA device"
        assert seqs.total_q == x.size(0), f"x has {x.size(0)} rows, the sequences {seqs.total_q}"
        assert seqs.num_sequences <= 65535, "at most 65535 sequences"
    params = (gate, scale, shift, weight, post_weight)
    dtype = None
    for name, t in zip(_PARAMS, params):
        if t is None:
            continue
        assert t.device == x.device, f"{name} must be on x's device"
        assert t.dtype in (x.dtype, torch.float32) and t.dtype == (dtype or t.dtype), \
            "the parameters must share one dtype, x's or fp32"
        dtype = t.dtype
        if name in ("weight", "post_weight") or seqs is None:
            assert t.shape == (c,) or (seqs is None and t.shape == (1, c)), f"{name} must be ({c},)"
        else:
            assert t.shape == (seqs.num_sequences, c), f"{name} must be ({seqs.num_sequences}, {c})"
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, y, *params)):
        out = _GatedNorm.apply(x, y, seqs, norm, eps, *params)
        return (x, out[0]) if y is None else out
    x_new, h = _forward(x, y, params, seqs, norm, eps, None)[3:]
    return (x if y is None else x_new), h
