"""torch.library registrations of ``mhc.branch`` (namespace ``mhc_branch``), for torch.compile.

As in ``_library.py``: each launcher is an opaque custom op with a fake kernel, the differentiable ones
carry their backward, and the functions below are what ``mhc.branch`` calls when it is traced.
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import Tensor

from . import _branch as _k

_F32 = torch.float32


def _op(name: str):
    return torch.library.custom_op(f"mhc_branch::{name}", mutates_args=(), device_types="cuda")


# --------------------------------------------------------------------------
# RMS norm
# --------------------------------------------------------------------------

@_op("norm")
def _norm(x: Tensor, weight: Optional[Tensor], eps: float) -> Tuple[Tensor, Tensor]:
    y, _, rstd = _k.rms_norm_forward(x, weight, None, eps)
    return y, rstd


@_norm.register_fake
def _(x, weight, eps):
    return x.new_empty(x.shape), x.new_empty(x.shape[:-1], dtype=_F32)


@_op("add_norm")
def _add_norm(x: Tensor, weight: Optional[Tensor], residual: Tensor, eps: float) -> Tuple[Tensor, Tensor, Tensor]:
    return _k.rms_norm_forward(x, weight, residual, eps)


@_add_norm.register_fake
def _(x, weight, residual, eps):
    return x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty(x.shape[:-1], dtype=_F32)


@_op("norm_backward")
def _norm_backward(dy: Tensor, h: Tensor, dh: Optional[Tensor], weight: Optional[Tensor], rstd: Tensor,
                   need_dw: bool) -> Tuple[Tensor, Tensor]:
    dx, dw = _k.rms_norm_backward(dy, h, dh, weight, rstd, True, need_dw)
    return dx, rstd.new_empty(0) if dw is None else dw


@_norm_backward.register_fake
def _(dy, h, dh, weight, rstd, need_dw):
    return h.new_empty(h.shape), rstd.new_empty(h.shape[-1] if need_dw else 0)


def _norm_grads(ctx, dy, dh):
    h, weight, rstd = ctx.saved_tensors
    if dy is None:
        return dh, None
    need_dw = weight is not None and ctx.needs_input_grad[1]
    dx, dw = torch.ops.mhc_branch.norm_backward(dy, h, dh, weight, rstd, need_dw)
    return dx, dw.to(weight.dtype) if need_dw else None


def _norm_setup(ctx, inputs, output):
    x, weight, _ = inputs
    ctx.save_for_backward(x, weight, output[1])
    ctx.set_materialize_grads(False)


def _add_norm_setup(ctx, inputs, output):
    ctx.save_for_backward(output[1], inputs[1], output[2])
    ctx.set_materialize_grads(False)


def _norm_bwd(ctx, dy, _):
    dx, dw = _norm_grads(ctx, dy, None)
    return dx, dw, None


def _add_norm_bwd(ctx, dy, dh, _):
    dx, dw = _norm_grads(ctx, dy, dh)
    return dx, dw, dx, None


torch.library.register_autograd("mhc_branch::norm", _norm_bwd, setup_context=_norm_setup)
torch.library.register_autograd("mhc_branch::add_norm", _add_norm_bwd, setup_context=_add_norm_setup)


def rms_norm(x, weight, residual, eps):
    if residual is None:
        return torch.ops.mhc_branch.norm(x, weight, eps)[0]
    y, h, _ = torch.ops.mhc_branch.add_norm(x, weight, residual, eps)
    return y, h


# --------------------------------------------------------------------------
# The 8-bit format
# --------------------------------------------------------------------------

def _mx_fake(x):
    return (x.new_empty(x.shape, dtype=_k.F8),
            x.new_empty((*x.shape[:-1], _k.scale_width(x.shape[-1])), dtype=_k.E8))


@_op("norm_mx")
def _norm_mx(x: Tensor, weight: Optional[Tensor], residual: Optional[Tensor], eps: float) -> List[Tensor]:
    q, scales, h = _k.rms_norm_mx(x, weight, residual, eps)
    return [q, scales] if h is None else [q, scales, h]


@_norm_mx.register_fake
def _(x, weight, residual, eps):
    out = list(_mx_fake(x))
    return out if residual is None else out + [x.new_empty(x.shape)]


@_op("quantize_mx")
def _quantize_mx(x: Tensor) -> Tuple[Tensor, Tensor]:
    return _k.quantize_mx(x)


@_quantize_mx.register_fake
def _(x):
    return _mx_fake(x)


def rms_norm_mx(x, weight, residual, eps):
    return tuple(torch.ops.mhc_branch.norm_mx(x, weight, residual, eps))


def quantize_mx(x):
    return torch.ops.mhc_branch.quantize_mx(x)


# --------------------------------------------------------------------------
# Products grouped by expert
# --------------------------------------------------------------------------

@_op("grouped_matmul")
def _grouped_matmul(x: Tensor, weight: Tensor, offsets: Tensor) -> Tensor:
    return _k.grouped_matmul_forward(x, weight, offsets)


@_grouped_matmul.register_fake
def _(x, weight, offsets):
    return x.new_empty(x.shape[0], weight.shape[1])


@_op("grouped_matmul_backward_input")
def _grouped_matmul_backward_input(dy: Tensor, weight: Tensor, offsets: Tensor) -> Tensor:
    return _k.grouped_matmul_backward_input(dy, weight, offsets)


@_grouped_matmul_backward_input.register_fake
def _(dy, weight, offsets):
    return dy.new_empty(dy.shape[0], weight.shape[2])


@_op("grouped_matmul_backward_weight")
def _grouped_matmul_backward_weight(dy: Tensor, x: Tensor, offsets: Tensor) -> Tensor:
    return _k.grouped_matmul_backward_weight(dy, x, offsets)


@_grouped_matmul_backward_weight.register_fake
def _(dy, x, offsets):
    return x.new_empty(offsets.shape[0], dy.shape[1], x.shape[1])


def _grouped_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _grouped_bwd(ctx, dy):
    x, weight, offsets = ctx.saved_tensors
    dx = torch.ops.mhc_branch.grouped_matmul_backward_input(dy, weight, offsets) if ctx.needs_input_grad[0] else None
    dw = torch.ops.mhc_branch.grouped_matmul_backward_weight(dy, x, offsets) if ctx.needs_input_grad[1] else None
    return dx, dw, None


torch.library.register_autograd("mhc_branch::grouped_matmul", _grouped_bwd, setup_context=_grouped_setup)


def grouped_matmul(x, weight, offsets):
    return torch.ops.mhc_branch.grouped_matmul(x, weight, offsets)


@_op("grouped_matmul_mx")
def _grouped_matmul_mx(q: Tensor, scales: Tensor, weight_q: Tensor, weight_scales: Tensor, offsets: Tensor,
                       out_dtype: torch.dtype) -> Tensor:
    return _k.grouped_matmul_mx(q, scales, weight_q, weight_scales, offsets, out_dtype)


@_grouped_matmul_mx.register_fake
def _(q, scales, weight_q, weight_scales, offsets, out_dtype):
    return q.new_empty((q.shape[0], weight_q.shape[1]), dtype=out_dtype)


def grouped_matmul_mx(q, scales, weight_q, weight_scales, offsets, out_dtype):
    return torch.ops.mhc_branch.grouped_matmul_mx(q, scales, weight_q, weight_scales, offsets, out_dtype)


# --------------------------------------------------------------------------
# Dropout
# --------------------------------------------------------------------------

# rng: a device state, or None and the words of a pair of ints (low and high 32 bits of the seed, of the offset):
# traced ints are symbols, and one past int64 can neither pass a schema nor enter a graph whole.

@_op("dropout")
def _dropout(x: Tensor, residual: Optional[Tensor], p: float, rng: Optional[Tensor],
             words: List[int]) -> Tuple[Tensor, Tensor]:
    if rng is None:
        rng = (words[0] | words[1] << 32, words[2] | words[3] << 32)
    return _k.dropout(x, p, rng, residual, want_used=True)


@_dropout.register_fake
def _(x, residual, p, rng, words):
    return x.new_empty(x.shape), x.new_empty(2, dtype=torch.int64)


def _dropout_setup(ctx, inputs, output):
    ctx.p = inputs[2]
    ctx.save_for_backward(output[1])


def _dropout_bwd(ctx, dy, _):
    used, = ctx.saved_tensors
    dx = torch.ops.mhc_branch.dropout(dy, None, ctx.p, used, [])[0] if ctx.needs_input_grad[0] else None
    return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


torch.library.register_autograd("mhc_branch::dropout", _dropout_bwd, setup_context=_dropout_setup)


def dropout(x, p, rng, residual):
    words = []
    if not isinstance(rng, Tensor):
        _k.check_rng(x, rng)
        words = [w for v in rng for w in (v & 0xFFFFFFFF, v >> 32)]
        rng = None
    return torch.ops.mhc_branch.dropout(x, residual, p, rng, words)[0]
