"""torch.library registrations of the operators that mix tokens (namespace ``mhc_mixer``), for torch.compile.

As in ``_branch_library.py``: each launcher is an opaque custom op with a fake kernel, the differentiable ones carry
their backward, and the functions below are what ``mhc.branch`` calls when it is traced.  An output that a call does
not have is empty.
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import Tensor

from . import _mixer as _k

_F32 = torch.float32


def _op(name: str, mutates=()):
    return torch.library.custom_op(f"mhc_mixer::{name}", mutates_args=mutates, device_types="cuda")


def _or_empty(t: Optional[Tensor], like: Tensor) -> Tensor:
    return like.new_empty(0) if t is None else t


# --------------------------------------------------------------------------
# Rotary positions
# --------------------------------------------------------------------------

@_op("rotary")
def _rotary(q: Tensor, k: Optional[Tensor], positions: Tensor, frequencies: Tensor, interleaved: bool, magnitude: float,
            inverse: bool) -> Tuple[Tensor, Tensor]:
    a, b = _k.rotary(q, k, positions, frequencies, interleaved, magnitude, inverse)
    return a, _or_empty(b, a)


@_rotary.register_fake
def _(q, k, positions, frequencies, interleaved, magnitude, inverse):
    return q.new_empty(q.shape), q.new_empty(0 if k is None else k.shape)


def _rotary_setup(ctx, inputs, output):
    _, k, positions, frequencies, ctx.interleaved, ctx.magnitude, ctx.inverse = inputs
    ctx.has_k = k is not None
    ctx.save_for_backward(positions, frequencies)


def _rotary_bwd(ctx, dq, dk):
    dq, dk = torch.ops.mhc_mixer.rotary(dq, dk if ctx.has_k else None, *ctx.saved_tensors, ctx.interleaved, ctx.magnitude,
                                        not ctx.inverse)
    return dq, dk if ctx.has_k else None, None, None, None, None, None


torch.library.register_autograd("mhc_mixer::rotary", _rotary_bwd, setup_context=_rotary_setup)


def rotary(q, k, positions, frequencies, interleaved, magnitude):
    a, b = torch.ops.mhc_mixer.rotary(q, k, positions, frequencies, interleaved, magnitude, False)
    return a if k is None else (a, b)


# --------------------------------------------------------------------------
# Decay attention
# --------------------------------------------------------------------------

def _state_shape(q, v, offsets):
    return (q.shape[0] if offsets is None else offsets.shape[0], *q.shape[-2:], v.shape[-1])


@_op("decay_attention")
def _decay_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, offsets: Optional[Tensor],
                     initial_state: Optional[Tensor], scale: float) -> Tuple[Tensor, Tensor]:
    return _k.decay_attention_forward(q, k, v, log_decay, offsets, initial_state, scale, True)[:2]


@_decay_attention.register_fake
def _(q, k, v, log_decay, offsets, initial_state, scale):
    return v.new_empty(v.shape), v.new_empty(_state_shape(q, v, offsets), dtype=_F32)


@_op("decay_attention_backward")
def _decay_attention_backward(q: Tensor, k: Tensor, v: Tensor, do: Tensor, log_decay: Tensor, offsets: Optional[Tensor],
                              initial_state: Optional[Tensor], d_state: Optional[Tensor], scale: float,
                              need: List[bool]) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    got = _k.decay_attention_backward(q, k, v, do, log_decay, offsets, initial_state, None, d_state, scale, tuple(need))
    return tuple(_or_empty(g, t) for g, t in zip(got, (q, k, v, log_decay)))


@_decay_attention_backward.register_fake
def _(q, k, v, do, log_decay, offsets, initial_state, d_state, scale, need):
    out = [t.new_empty(t.shape if n else 0) for t, n in zip((q, k, v), need)]
    state = q.new_empty(_state_shape(q, v, offsets), dtype=_F32) if need[3] else log_decay.new_empty(0)
    return (*out, state)


def _decay_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:6])
    ctx.scale = inputs[6]
    ctx.set_materialize_grads(False)


def _decay_bwd(ctx, do, d_state):
    q, k, v, log_decay, offsets, initial = ctx.saved_tensors
    need = [*ctx.needs_input_grad[:3], ctx.needs_input_grad[5]]
    if do is None:
        do = v.new_zeros(v.shape)
    got = torch.ops.mhc_mixer.decay_attention_backward(q, k, v, do, log_decay, offsets, initial, d_state, ctx.scale, need)
    dq, dk, dv, ds = (g if n else None for g, n in zip(got, need))
    return dq, dk, dv, None, None, ds, None


torch.library.register_autograd("mhc_mixer::decay_attention", _decay_bwd, setup_context=_decay_setup)


def decay_attention(q, k, v, log_decay, offsets, initial_state, scale):
    """(o, state).  The state is always made and the segments' states are not kept for the backward, which makes them again."""
    return torch.ops.mhc_mixer.decay_attention(q, k, v, log_decay, offsets, initial_state, scale)


@_op("decay_attention_step", ("state",))
def _decay_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, slots: Optional[Tensor],
                          scale: float) -> Tensor:
    return _k.decay_attention_step(q, k, v, log_decay, state, slots, scale, None)


@_decay_attention_step.register_fake
def _(q, k, v, log_decay, state, slots, scale):
    return v.new_empty(v.shape)


@_op("decay_attention_step_out", ("state_out",))
def _decay_attention_step_out(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, slots: Optional[Tensor],
                              scale: float, state_out: Tensor) -> Tensor:
    return _k.decay_attention_step(q, k, v, log_decay, state, slots, scale, state_out)


@_decay_attention_step_out.register_fake
def _(q, k, v, log_decay, state, slots, scale, state_out):
    return v.new_empty(v.shape)


def decay_attention_step(q, k, v, log_decay, state, slots, scale, state_out):
    if state_out is None:
        return torch.ops.mhc_mixer.decay_attention_step(q, k, v, log_decay, state, slots, scale)
    return torch.ops.mhc_mixer.decay_attention_step_out(q, k, v, log_decay, state, slots, scale, state_out)


# --------------------------------------------------------------------------
# Gated products
# --------------------------------------------------------------------------

@_op("gated_matmul")
def _gated_matmul(x: Tensor, weight: Tensor, offsets: Optional[Tensor], activation: str, keep: bool) -> Tuple[Tensor, Tensor]:
    y, saved = _k.gated_matmul_forward(x, weight, offsets, activation, keep)
    return y, x.new_empty(0, dtype=_F32) if saved is None else saved


@_gated_matmul.register_fake
def _(x, weight, offsets, activation, keep):
    R, N = x.shape[0], weight.shape[-2] // 2
    return x.new_empty(R, N), x.new_empty((R, 2 * N) if keep else (0,), dtype=_F32)


@_op("gated_matmul_backward")
def _gated_matmul_backward(dy: Tensor, saved: Tensor, x: Tensor, weight: Tensor, offsets: Optional[Tensor], activation: str,
                           need_dx: bool, need_dw: bool) -> Tuple[Tensor, Tensor]:
    dx, dw = _k.gated_matmul_backward(dy, saved, x, weight, offsets, activation, need_dx, need_dw)
    return _or_empty(dx, x), _or_empty(dw, weight)


@_gated_matmul_backward.register_fake
def _(dy, saved, x, weight, offsets, activation, need_dx, need_dw):
    return x.new_empty(x.shape if need_dx else 0), weight.new_empty(weight.shape if need_dw else 0)


def _gated_setup(ctx, inputs, output):
    x, weight, offsets, ctx.activation, keep = inputs
    ctx.kept = keep
    ctx.save_for_backward(x, weight, offsets, output[1])


def _gated_bwd(ctx, dy, _):
    if not ctx.kept:
        raise RuntimeError("mhc: gated_matmul was traced without its backward")
    x, weight, offsets, saved = ctx.saved_tensors
    need = ctx.needs_input_grad[:2]
    dx, dw = torch.ops.mhc_mixer.gated_matmul_backward(dy, saved, x, weight, offsets, ctx.activation, *need)
    return dx if need[0] else None, dw if need[1] else None, None, None, None


torch.library.register_autograd("mhc_mixer::gated_matmul", _gated_bwd, setup_context=_gated_setup)


def gated_matmul(x, weight, offsets, activation):
    keep = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)
    return torch.ops.mhc_mixer.gated_matmul(x, weight, offsets, activation, keep)[0]
