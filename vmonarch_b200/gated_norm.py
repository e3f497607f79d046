"""The elementwise and normalising work between two blocks of a transformer, fused (no reference
counterpart): a norm after the block, its gate, the residual, and the modulated norm before the next block.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as N
from .kernel import SUPPORTED_DTYPES

#: widths: multiples of 8 up to this
MAX_WIDTH = 8192


def _rows_in_place(t):
    """`t` (T, C) when the kernels can address it: contiguous columns, 16-byte aligned rows."""
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (t.size(0) <= 1 or t.stride(0) >= 0 and t.stride(0) % 8 == 0):
        return t
    return t.contiguous()


def _dense(t):
    return t if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0) else t.clone(memory_format=torch.contiguous_format)


def _matrix(t):
    return N.Matrix(t.data_ptr(), t.stride(0) if t.size(0) > 1 else t.size(1))


def _args(x, y, params, seqs, norm, eps):
    a = N.GatedNormArgs()
    a.x = _matrix(x)
    if y is not None:
        a.y = _matrix(y)
    a.param_dtype = a.dtype = N.dtype_code(x.dtype)
    for name, t in zip(_PARAMS, params):
        if t is not None:
            setattr(a, name, t.data_ptr())
            a.param_dtype = N.VMB_DTYPE_F32 if t.dtype == torch.float32 else a.dtype
    a.rows, a.cols, a.seqs = x.size(0), x.size(1), seqs.num_sequences if seqs is not None else 1
    if a.seqs > 1:
        a.seq_start = seqs._starts().data_ptr()
    a.layer, a.eps = norm == "layer", eps
    return a


_PARAMS = ("gate", "scale", "shift", "weight", "post_weight")


def _forward(x, y, params, seqs, norm, eps, want_stats):
    x, y = _rows_in_place(x), y if y is None else _rows_in_place(y)
    params = [_dense(t) for t in params]
    x_new = torch.empty(x.shape, dtype=x.dtype, device=x.device) if y is not None else None
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((3, x.size(0)), dtype=torch.float32, device=x.device) if want_stats else None
    a = _args(x, y, params, seqs, norm, eps)
    a.x_new, a.h = N.ptr(x_new), h.data_ptr()
    a.stats = N.ptr(stats)
    N.check(N.lib.vmb_gated_norm_fwd(ctypes.byref(a), N.stream_ptr(x.device)), "vmb_gated_norm_fwd")
    return x, y, params, x_new, h, stats


class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, seqs, norm, eps, *params):
        shapes = [None if t is None else t.shape for t in params]
        xs, ys, dense, x_new, h, stats = _forward(x, y, params, seqs, norm, eps, True)
        ctx.save_for_backward(xs, ys, stats, *dense)
        ctx.meta = seqs, norm, eps, shapes
        ctx.set_materialize_grads(False)
        return (h,) if y is None else (x_new, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        x, y, stats, *params = ctx.saved_tensors
        seqs, norm, eps, shapes = ctx.meta
        dx_new, dh = grads if y is not None else (None, *grads)
        a = _args(x, y, params, seqs, norm, eps)
        dx_new, dh = (None if t is None else _rows_in_place(t) for t in (dx_new, dh))
        if dx_new is not None:
            a.dx_new = _matrix(dx_new)
        if dh is not None:
            a.dh = _matrix(dh)
        a.stats = stats.data_ptr()
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dy = torch.empty(x.shape, dtype=x.dtype, device=x.device) if y is not None else None
        a.dx, a.dy = dx.data_ptr(), N.ptr(dy)
        out = []
        for name, t, need, shape in zip(_PARAMS, params, ctx.needs_input_grad[5:], shapes):
            g = torch.empty(shape, dtype=t.dtype, device=x.device) if t is not None and need else None
            setattr(a, "d" + name, N.ptr(g))
            out.append(g)
        nbytes = N.lib.vmb_gated_norm_bwd_workspace_bytes(ctypes.byref(a))
        if nbytes > 0:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
        N.check(N.lib.vmb_gated_norm_bwd(ctypes.byref(a), N.stream_ptr(x.device)), "vmb_gated_norm_bwd")
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
    _, _, _, x_new, h, _ = _forward(x, y, params, seqs, norm, eps, False)
    return (x if y is None else x_new), h
