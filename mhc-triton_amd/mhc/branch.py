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

A branch that mixes tokens, and a feed-forward that begins with a gated product:

    q, k = rotary(q, k, positions, rotary_frequencies(dim))  # (batch, tokens, heads, dim)
    o, state = decay_attention(q, k, v, log_decay, return_state=True)
    o = decay_attention_step(q, k, v, log_decay, state)      # the next token of each sequence, (batch, heads, dim)
    x = gated_matmul(y, w_gate_up, offsets)                  # act(y gate) * (y up), or without offsets of one weight

``examples/decay_layer.py`` is the whole of it, training, prompts and decoding.

Tensors are fp32, bf16 or fp16 on a ROCm GPU and are computed in fp32; each op runs on the current stream,
waits for nothing on the host and may be captured in a HIP graph.  Gradients are of the first order in reverse
mode; second derivatives and, in eager calls, forward mode raise.  Not part of ``mhc.__all__``, which stays the reference's.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _branch as _k
from . import _branch_library as _l
from . import _lib
from . import _mixer as _m
from . import _mixer_library as _ml
from ._branch import Rng

__all__ = ["rms_norm", "rms_norm_mx", "quantize_mx", "grouped_matmul", "grouped_matmul_mx", "dropout",
           "rotary", "rotary_frequencies", "decay_attention", "decay_attention_step", "gated_matmul"]


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


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, frequencies, interleaved: bool, magnitude: float):
        ctx.save_for_backward(positions, frequencies)
        ctx.how = interleaved, magnitude
        ctx.set_materialize_grads(False)
        a, b = _m.rotary(q, k, positions, frequencies, interleaved, magnitude)
        return a if k is None else (a, b)

    @staticmethod
    def backward(ctx, dq, dk=None):
        grads = [dq if ctx.needs_input_grad[0] else None, dk if ctx.needs_input_grad[1] else None]
        have = [i for i in (0, 1) if grads[i] is not None]
        if have:  # both in one launch
            got = _m.rotary(grads[have[0]], grads[1] if len(have) == 2 else None, *ctx.saved_tensors, *ctx.how, True)
            for i, g in zip(have, got):
                grads[i] = _first_order(g, "rotary", grads[i].requires_grad)
        return (*grads, None, None, None, None)


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, offsets, initial_state, scale: float, return_state: bool):
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        o, state, kept = _m.decay_attention_forward(q, k, v, log_decay, offsets, initial_state, scale, return_state)
        ctx.save_for_backward(q, k, v, log_decay, offsets, initial_state, kept if ctx.needs_input_grad[0] else None)
        return (o, state) if return_state else o

    @staticmethod
    def backward(ctx, do, d_state=None):
        q, k, v, log_decay, offsets, initial, kept = ctx.saved_tensors
        need = (*ctx.needs_input_grad[:3], ctx.needs_input_grad[5])
        if do is None and d_state is None:
            return (None,) * 8
        if do is None:
            do = torch.zeros_like(v, memory_format=torch.contiguous_format)
        got = _m.decay_attention_backward(q, k, v, do, log_decay, offsets, initial, kept, d_state, ctx.scale, need)
        graph = [t is not None and t.requires_grad for t in (do, d_state, q, k, v, initial)]
        dq, dk, dv, ds = (_first_order(g, "decay_attention", *graph) for g in got)
        return dq, dk, dv, None, None, ds, None, None


class _GatedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets, activation: str):
        y, saved = _m.gated_matmul_forward(x, weight, offsets, activation, want_saved=any(ctx.needs_input_grad))
        ctx.save_for_backward(x, weight, offsets, saved)
        ctx.activation = activation
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, offsets, saved = ctx.saved_tensors
        need = ctx.needs_input_grad[:2]
        dx, dw = _m.gated_matmul_backward(dy, saved, x, weight, offsets, ctx.activation, *need)
        graph = (dy.requires_grad, x.requires_grad, weight.requires_grad)
        return _first_order(dx, "gated_matmul", *graph), _first_order(dw, "gated_matmul", *graph), None, None


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


def rotary_frequencies(dim: int, base: float = 10000.0, factor: float = 1.0, original_length: Optional[int] = None,
                       fast: float = 32.0, slow: float = 1.0, device=None) -> torch.Tensor:
    """Radians a position for each of the dim / 2 pairs that ``rotary`` turns, in fp64: ``base ** (-2 i / dim)``.

    For contexts ``factor`` times as long as the trained ones every frequency is divided by factor; with
    ``original_length``, the trained length, only those that turn fewer than ``slow`` times over it are, those that
    turn more than ``fast`` times stay, and between them the share that stays falls off linearly in the pair's index (between
    the whole numbers around the two ends, which may lie before the first pair and behind the last).  (Such a
    context usually takes ``magnitude = 0.1 * log(factor) + 1`` in ``rotary``, too.)"""
    if dim < 0 or dim % 2:
        raise ValueError(f"dim must be even, got {dim}")
    if not (base > 0 and factor > 0):
        raise ValueError(f"base and factor must be positive, got {base} and {factor}")
    i = torch.arange(dim // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / max(dim, 1))
    if original_length is None:
        f = f / factor
    elif factor != 1.0:
        if not (original_length > 0 and fast > slow > 0 and base > 1):
            raise ValueError(f"original_length, fast > slow and base > 1 must be positive, got {original_length}, {fast}, "
                             f"{slow}, {base}")

        def pair_of(turns):  # the index, not whole, of the pair that turns so often over the trained length
            return dim * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        lo, hi = math.floor(pair_of(fast)), math.ceil(pair_of(slow))  # the ramp's ends, whether or not there are such pairs
        stretched = ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        f = f * (1.0 - stretched) + f / factor * stretched
    return f.to(device) if device is not None else f


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor,
           interleaved: bool = False, magnitude: float = 1.0) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Rotary positions of q (..., heads, dim) and k (..., its own number of heads, dim): ``(q, k)``, or with k None q
    alone.  A pair (a, b) of a head becomes ``magnitude * (a cos t - b sin t, b cos t + a sin t)``,
    ``t = position * frequency``.

    ``frequencies`` (pairs,) are radians a position, one for each pair of the head's first 2 * pairs elements (at most
    4096); the others go through.  Pair i is (i, pairs + i), or (2 i, 2 i + 1) when ``interleaved``.  ``positions``
    (int32 or int64) has q's leading dimensions or the last of them, (tokens,) for (batch, tokens, heads, dim).
    Angles are taken in fp64: they are exact to 2^-52 of their size however far the position (int64 up to 2^53).

    q and k are read where they lie if a head's elements are neighbours and one stride leads from row to row, parts of
    a fused projection's output among them; others are copied.  The results are contiguous.  Differentiable in q and k.
    """
    _no_gradient("rotary", "frequencies", frequencies)
    if torch.compiler.is_compiling():
        return _ml.rotary(q, k, positions, frequencies, bool(interleaved), float(magnitude))
    if q.is_cuda:
        out = _lib.native().rotary(q, k, positions, frequencies, bool(interleaved), float(magnitude))
        if out is not None:
            return out
    return _Rotary.apply(q, k, positions, frequencies, bool(interleaved), float(magnitude))


def _no_gradient(name: str, what: str, t: torch.Tensor) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"mhc: {name} has no gradient of {what}; detach it")


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                    initial_state: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None, return_state: bool = False):
    """Linear attention with a decay for each head: ``S_t = exp(log_decay) S_{t-1} + k_t^T v_t``,
    ``o_t = scale * q_t S_t``; o as v, or ``(o, state)`` with ``return_state``.

    q and k are (batch, tokens, heads, key dim), v (batch, tokens, heads, value dim), dims from 1 to 128.  With
    ``offsets`` (sequences,) int32 on the GPU (int64 is narrowed) they are packed, (tokens, heads, dim), and sequence n
    has tokens ``offsets[n-1]`` to ``offsets[n]``; offsets count clamped and as their running maximum, and are read on the
    GPU only, so a captured graph serves every split.  Tokens past the last offset give zeros and get zero gradients.
    ``initial_state`` and the state are (sequences, heads, key dim, value dim) fp32; a sequence without tokens hands its own on.
    ``log_decay`` (heads,) has no gradient; above 0 it counts as 0.  ``scale`` defaults to ``key dim ** -0.5``.

    Differentiable in q, k, v and initial_state.  Inputs are read where they lie as ``rotary`` reads them (rows at most
    2^22 elements apart), heads that are one expanded among them.  Sums are fp32; products are of bf16 parts whose sum
    is the operand, exactly for inputs.  A value that is not finite reaches its own and later tokens of its sequence and
    head, no others; which of them are infinite and which NaN may differ from the recurrence's (fp32 magnitudes that round
    to no bf16, from 3.39e38 on, count as not finite).  What is computed (weights, states) enters the products as two bf16
    parts for 16-bit types, 2^-16 of itself or better, three for fp32.  With ``return_state``, and in traced calls, weighted values have a
    part more than without, so that the last bits of o may differ.
    """
    _no_gradient("decay_attention", "log_decay", log_decay)
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    if torch.compiler.is_compiling():
        out = _ml.decay_attention(q, k, v, log_decay, offsets, initial_state, scale)
        return out if return_state else out[0]
    if q.is_cuda:
        out = _lib.native().decay_attention(q, k, v, log_decay, initial_state, offsets, scale, bool(return_state))
        if out is not None:
            return out
    return _DecayAttention.apply(q, k, v, log_decay, offsets, initial_state, scale, bool(return_state))


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor,
                         slots: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                         state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``decay_attention`` of one more token for each row of q, k (rows, heads, key dim) and v (rows, heads, value dim):
    o as v, and ``state`` (states, heads, key dim, value dim) fp32, contiguous, moved on in place.

    Row r has state ``slots[r]`` (int32 or int64 on the GPU, read there only), or state r without slots.  Rows with the same
    slot are tokens of one sequence in their order; a row whose slot is outside the pool (negative: padding of a batch)
    gives zeros and touches no state, and states of no row stay as they are.  With ``state_out`` the rows' new states go
    there and ``state`` stays: the one before is kept for tokens that may be taken back.  No backward.
    """
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    compiling = torch.compiler.is_compiling()
    if q.is_cuda and not compiling:
        o = _lib.native().decay_attention_step(q, k, v, log_decay, state, slots, scale, state_out)
        if o is not None:
            return o
    _inference_only("decay_attention_step", q, k, v, log_decay, state, state_out)
    if compiling:
        return _ml.decay_attention_step(q, k, v, log_decay, state, slots, scale, state_out)
    o = _m.decay_attention_step(q, k, v, log_decay, state, slots, scale, state_out)
    out = state if state_out is None else state_out
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)
    return o


def gated_matmul(x: torch.Tensor, weight: torch.Tensor, offsets: Optional[torch.Tensor] = None,
                 activation: str = "silu") -> torch.Tensor:
    """``act(x gate^T) * (x up^T)``: the gated product that a feed-forward begins with, (rows, out) in x's dtype.

    ``weight`` is (2 * out, in), the gate's rows and then the up projection's, for all rows of x (rows, in); with
    ``offsets`` it is (experts, 2 * out, in) and x's rows are sorted by expert, exactly as in ``grouped_matmul``.
    ``activation`` is "silu", "gelu" (by the error function) or "gelu_tanh".  Both products are summed, activated and
    multiplied in fp32 and rounded once.  Differentiable in x and weight; for the backward both products are kept
    in fp32 (8 * rows * out bytes).  Gradients are rounded twice: the gradients of the two products, computed in fp32, to x's
    dtype before their own products, and the results.
    """
    if torch.compiler.is_compiling():
        return _ml.gated_matmul(x, weight, offsets, activation)
    if x.is_cuda:
        y = _lib.native().gated_matmul(x, weight, offsets, activation)
        if y is not None:
            return y
    return _GatedMatmul.apply(x, weight, offsets, activation)
