"""Operators inside a hyper-connection's branch.

``HyperConnection`` hands its caller a branch input and takes a branch output back.  What a
mixture-of-experts feed-forward branch does in between runs on these HIP kernels:

    bi, add_residual = hc(H)
    y = rms_norm(bi.flatten(0, 1), weight)                  # (tokens, dim)
    x = y[token]                                            # rows sorted by expert (the caller's router)
    x = grouped_matmul(x, w_up, offsets)                    # each row times its expert's weight
    x = grouped_matmul(act(x), w_down, offsets)
    out = combine(x)                                        # back to tokens
    H = add_residual(dropout(out, 0.1, rng).view_as(bi))

``examples/expert_branch.py`` is the whole of it, training and decoding.  For serving, ``rms_norm_mx``,
``quantize_mx`` and ``grouped_matmul_mx`` work in 8 bits: e4m3 values with a power-of-two scale for every
32 of a row (microscaling), which the matrix instructions of gfx950 multiply in.

Tensors are fp32, bf16 or fp16 on a ROCm GPU and are computed in fp32; each op runs on the current stream,
waits for nothing on the host and may be captured in a HIP graph.  Gradients are of the first order in reverse
mode; second derivatives and, in eager calls, forward mode raise.  Not part of ``mhc.__all__``, which stays the reference's.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _branch as _k
from . import _branch_library as _l
from . import _lib
from ._branch import Rng

__all__ = ["rms_norm", "rms_norm_mx", "quantize_mx", "grouped_matmul", "grouped_matmul_mx", "dropout"]


def _first_order(grad: Optional[torch.Tensor], name: str, *differentiable: bool) -> Optional[torch.Tensor]:
    """A gradient that a launcher computed.  Under create_graph, where something that went into it is differentiable,
    it carries a node that raises: it would count as a constant otherwise."""
    if grad is None or not torch.is_grad_enabled() or not any(differentiable):
        return grad
    return torch._C._functions.DelayedError(f"mhc: {name} has no second derivative".encode(), 1)(
        grad.detach().requires_grad_())


class _RmsNorm(torch.autograd.Function):
    """(x, weight, residual) -> y, or (y, h) with a residual.  Keeps h (x without a residual) and rstd."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps: float):
        x = x.contiguous()
        y, h, rstd = _k.rms_norm_forward(x, weight, residual, eps, want_rstd=any(ctx.needs_input_grad))
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        need_x = ctx.needs_input_grad[0] or ctx.needs_input_grad[2]
        dx, dw = dh, None
        if dy is not None:
            dx, dw = _k.rms_norm_backward(dy, h, dh, weight, rstd, need_x, ctx.needs_input_grad[1])
            dw = None if dw is None else dw.to(weight.dtype)
            dx = _first_order(dx, "rms_norm", need_x)
            dw = _first_order(dw, "rms_norm", need_x, dy.requires_grad)
        return (dx if ctx.needs_input_grad[0] else None,
                dw,
                dx if ctx.needs_input_grad[2] else None,
                None)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p: float, rng):
        # a device state may move on before the backward: what the forward drew from is kept
        y, used = _k.dropout(x, p, rng, residual, want_used=isinstance(rng, torch.Tensor))
        ctx.p, ctx.rng = p, rng if used is None else None
        if used is not None:
            ctx.save_for_backward(used)
        return y

    @staticmethod
    def backward(ctx, dy):
        dx = None
        if ctx.needs_input_grad[0]:
            dx, _ = _k.dropout(dy, ctx.p, ctx.rng if ctx.rng is not None else ctx.saved_tensors[0])
            dx = _first_order(dx, "dropout", dy.requires_grad)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None


class _GroupedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets):
        ctx.save_for_backward(x, weight, offsets)
        return _k.grouped_matmul_forward(x, weight, offsets)

    @staticmethod
    def backward(ctx, dy):
        x, weight, offsets = ctx.saved_tensors
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = _k.grouped_matmul_backward_input(dy, weight, offsets)
            dx = _first_order(dx, "grouped_matmul", dy.requires_grad, weight.requires_grad)
        if ctx.needs_input_grad[1]:
            dw = _k.grouped_matmul_backward_weight(dy, x, offsets)
            dw = _first_order(dw, "grouped_matmul", dy.requires_grad, x.requires_grad)
        return dx, dw, None


def _inference_only(name: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"mhc: {name} has no backward; call it under torch.no_grad()")
    # a launcher reads a dual tensor's values and would drop its tangent
    if not torch.compiler.is_compiling() and any(t is not None and unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"mhc: {name} has no forward-mode derivative")


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``h / sqrt(mean(h^2) + eps) * weight`` over the last dimension (at most 16384), in x's dtype.

    Without a residual ``h`` is x and the result is ``y``.  With one, of x's shape and dtype, ``h`` is
    ``x + residual`` rounded to their dtype and the result is ``(y, h)``: h is the residual stream that goes
    on, and y is the norm of what is stored.  ``weight`` (dim,) may have any floating dtype; None means ones.
    """
    if torch.compiler.is_compiling():
        return _l.rms_norm(x, weight, residual, float(eps))
    if x.is_cuda:
        out = _lib.native().rms_norm(x, weight, residual, float(eps))
        if out is not None:
            return out
    return _RmsNorm.apply(x, weight, residual, float(eps))


def rms_norm_mx(x: torch.Tensor, weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                eps: float = 1e-6):
    """``rms_norm`` with y in 8 bits, for ``grouped_matmul_mx``: ``(q, scales)`` or, with a residual,
    ``(q, scales, h)``.

    ``q`` (float8_e4m3fn, x's shape) holds y over its block's scale, a block being 32 neighbours of a row;
    ``scales`` (float8_e8m0fnu, (..., 4 * ceil(dim / 128))) the powers of two, the smallest that keep a
    block's largest magnitude at or below 448 (the row is filled up with the smallest scale).  A block with
    an infinity or a NaN has scale NaN.  No backward.
    """
    _inference_only("rms_norm_mx", x, weight, residual)
    if torch.compiler.is_compiling():
        return _l.rms_norm_mx(x, weight, residual, float(eps))
    q, scales, h = _k.rms_norm_mx(x, weight, residual, float(eps))
    return (q, scales) if h is None else (q, scales, h)


def quantize_mx(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows (..., dim), dim a multiple of 32, in 8 bits: ``(q, scales)`` as ``rms_norm_mx`` returns them.
    Experts' weights (experts, out, in) are quantised with it once.  No backward."""
    _inference_only("quantize_mx", x)
    if torch.compiler.is_compiling():
        return _l.quantize_mx(x)
    return _k.quantize_mx(x)


def grouped_matmul(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """Each row of x (rows, in) times its expert's weight (experts, out, in): (rows, out) in x's dtype.

    Rows are sorted by expert: expert e has rows ``offsets[e-1]`` to ``offsets[e]`` (``offsets[-1]`` counting as 0),
    the running sum of the experts' row counts, int32 on the GPU (int64 is narrowed, two more launches).  It is read there
    only, so any split, experts without rows among them, serves a captured graph.  Rows past the last offset
    belong to no expert: they give zeros and get zero gradients; offsets out of range count clamped, offsets that
    run backwards as their running maximum.  Differentiable in x and weight.

    Both operands are read as they lie when contiguous; any other view, weights stored (experts, in, out) and passed
    transposed among them, is copied whole at every call.
    """
    if torch.compiler.is_compiling():
        return _l.grouped_matmul(x, weight, offsets)
    if x.is_cuda:
        y = _lib.native().grouped_matmul(x, weight, offsets)
        if y is not None:
            return y
    return _GroupedMatmul.apply(x, weight, offsets)


def grouped_matmul_mx(q: torch.Tensor, scales: torch.Tensor, weight_q: torch.Tensor, weight_scales: torch.Tensor,
                      offsets: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``grouped_matmul`` of 8-bit rows and weights, each with its scales as ``quantize_mx`` gives them; the
    result is in ``out_dtype``, bfloat16 or float16 (the 8-bit matrix instruction's sums fall short of fp32).
    No backward."""
    _inference_only("grouped_matmul_mx", q, scales, weight_q, weight_scales)
    if torch.compiler.is_compiling():
        return _l.grouped_matmul_mx(q, scales, weight_q, weight_scales, offsets, out_dtype)
    return _k.grouped_matmul_mx(q, scales, weight_q, weight_scales, offsets, out_dtype)


def dropout(x: torch.Tensor, p: float, rng: Rng, residual: Optional[torch.Tensor] = None,
            training: bool = True) -> torch.Tensor:
    """``residual + dropout(x)``: each element of x is dropped with probability p and the others are scaled to keep
    the mean.  The mask follows from ``rng`` and the element's index alone (Philox4x32-10) and is never
    stored.

    ``rng`` is (seed, offset): two ints, or an int64 tensor of two on the GPU, which a captured graph reads
    at each replay.  The same pair gives the same mask: add one to the offset for each call.  p is rounded
    to a multiple of 2^-16.  Not training, or p = 0: x + residual without a mask.
    """
    if not training:
        p = 0.0
    if torch.compiler.is_compiling():
        return _l.dropout(x, float(p), rng, residual)
    if x.is_cuda:
        y = _lib.native().dropout(x, residual, float(p), rng)
        if y is not None:
            return y
    return _Dropout.apply(x, residual, float(p), rng)
