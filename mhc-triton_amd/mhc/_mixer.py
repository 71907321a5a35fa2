"""Launchers of the operators that mix tokens (``mhc.branch``: rotary, decay attention, gated products) over the C ABI.

Like ``_branch.py``: argument checks, output allocation, one C-ABI call.  They know nothing of autograd.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._branch import _offsets
from ._kernels import ShapeError, _f32

#: Widest head of decay attention (a head's state stays in registers).
MAX_HEAD_DIM = 128
#: Widest head of rotary positions (its angles stay in LDS).
MAX_ROTARY_DIM = 4096
#: Rows are at most this many elements apart; others are copied.
MAX_ROW_STRIDE = 1 << 22
#: Activations of gated products and their codes.
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


class _Heads:
    """Rows (..., heads, dim) as the kernels read them: a head's elements neighbours, rows and heads anywhere.  What no
    one row stride describes is copied."""

    __slots__ = ("t", "R", "H", "D", "row", "head")

    def __init__(self, t: torch.Tensor):
        H, D = t.shape[-2:]
        if t.dim() == 2:
            t = t.unsqueeze(0)
        elif t.dim() > 3:
            t = t.flatten(0, -3)
        if (D > 1 and t.stride(2) != 1) or (t.shape[0] > 1 and t.stride(0) > MAX_ROW_STRIDE):
            t = t.contiguous()
        self.t, self.R, self.H, self.D = t, t.shape[0], H, D
        self.row = t.stride(0) if self.R > 1 else H * D
        self.head = t.stride(1) if H > 1 else D

    def args(self):
        return self.t.data_ptr(), self.row, self.head


_NONE = (None, 0, 0)


def _same_dtype(name: str, t: torch.Tensor, like: torch.Tensor) -> None:
    if t.dtype != like.dtype:
        raise TypeError(f"mhc: {name} must be {like.dtype}, got {t.dtype}")


# --------------------------------------------------------------------------
# Rotary positions
# --------------------------------------------------------------------------

def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor,
           interleaved: bool, magnitude: float, inverse: bool = False):
    """(q, k) turned by position * frequency, or back."""
    for name, t in (("q", q), ("k", k)):
        if t is not None and t.dim() < 2:
            raise ShapeError(f"{name} must be (..., heads, dim), got {tuple(t.shape)}")
    lead, D = q.shape[:-2], q.shape[-1]
    if k is not None:
        if k.shape[:-2] != lead or k.shape[-1] != D:
            raise ShapeError(f"k must be {(*lead, 'heads', D)}, got {tuple(k.shape)}")
        _same_dtype("k", k, q)
    if positions.dim() > len(lead) or positions.shape != lead[len(lead) - positions.dim():]:
        raise ShapeError(f"positions must have the last of the dimensions {tuple(lead)}, got {tuple(positions.shape)}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"mhc: positions must be int32 or int64, got {positions.dtype}")
    if frequencies.dim() != 1 or 2 * frequencies.shape[0] > D or D > MAX_ROTARY_DIM:
        raise ShapeError(f"frequencies must be one for each of at most {D // 2} pairs of heads of at most "
                         f"{MAX_ROTARY_DIM}, got {tuple(frequencies.shape)}")
    if not frequencies.is_floating_point():
        raise TypeError(f"mhc: frequencies must be floating point, got {frequencies.dtype}")
    dev = _lib.require_gpu(q, k, positions, frequencies)
    code = _lib.dtype_code(q)
    positions, frequencies = positions.contiguous(), frequencies.to(torch.float64).contiguous()
    a = _Heads(q)
    b = None if k is None else _Heads(k)
    q_out = torch.empty(q.shape, device=dev, dtype=q.dtype)
    k_out = None if k is None else torch.empty(k.shape, device=dev, dtype=k.dtype)
    if q_out.numel() == 0 and (k_out is None or k_out.numel() == 0):
        return q_out, k_out
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.mhc_rotary(*a.args(), q_out.data_ptr(), a.H, *(_NONE if b is None else b.args()), _lib.ptr(k_out),
                                  0 if b is None else b.H, code, positions.data_ptr(),
                                  int(positions.dtype == torch.int64), positions.numel(), frequencies.data_ptr(),
                                  frequencies.shape[0], a.R, D, float(magnitude), int(interleaved), int(inverse),
                                  _lib.stream(dev)), "rotary")
    return q_out, k_out


# --------------------------------------------------------------------------
# Decay attention
# --------------------------------------------------------------------------

def _head_dims(q, k, v) -> Tuple[int, int, int]:
    if q.dim() < 3 or k.shape != q.shape or v.shape[:-1] != q.shape[:-1]:
        raise ShapeError(f"q and k must be (..., heads, dim) and v (..., heads, dim of its own), got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    H, Dk, Dv = *q.shape[-2:], v.shape[-1]
    if not (1 <= Dk <= MAX_HEAD_DIM and 1 <= Dv <= MAX_HEAD_DIM):
        raise ShapeError(f"heads of {Dk} and {Dv} elements; 1 to {MAX_HEAD_DIM}")
    _same_dtype("k", k, q)
    _same_dtype("v", v, q)
    return H, Dk, Dv


def _check_decay(log_decay, H):
    if tuple(log_decay.shape) != (H,):
        raise ShapeError(f"log_decay must be ({H},), got {tuple(log_decay.shape)}")
    if not log_decay.is_floating_point():
        raise TypeError(f"mhc: log_decay must be floating point, got {log_decay.dtype}")


def _check_state(name, state, shape):
    if state is None:
        return
    if tuple(state.shape) != shape:
        raise ShapeError(f"{name} must be {shape}, got {tuple(state.shape)}")
    if state.dtype != torch.float32:
        raise TypeError(f"mhc: {name} must be torch.float32, got {state.dtype}")


def _sequences(q, offsets) -> int:
    """N of (N, T, heads, dim) or of packed rows (tokens, heads, dim) with their ends."""
    if offsets is None:
        if q.dim() != 4:
            raise ShapeError(f"q must be (batch, tokens, heads, dim) without offsets, got {tuple(q.shape)}")
        return q.shape[0]
    if q.dim() != 3 or offsets.dim() != 1:
        raise ShapeError(f"q and offsets must be (tokens, heads, dim) and (sequences,), got {tuple(q.shape)}, "
                         f"{tuple(offsets.shape)}")
    return offsets.shape[0]


def _decay_args(q, k, v, log_decay, offsets, *states):
    H, Dk, Dv = _head_dims(q, k, v)
    _check_decay(log_decay, H)
    N = _sequences(q, offsets)
    for name, s in states:
        _check_state(name, s, (N, H, Dk, Dv))
    dev = _lib.require_gpu(q, k, v, log_decay, offsets, *(s for _, s in states))
    return dev, N, H, Dk, Dv, None if offsets is None else _offsets(offsets, N)


def decay_attention_forward(q, k, v, log_decay, offsets, initial_state, scale: float, want_state: bool):
    """(o, state, kept): o as v; state (N, H, Dk, Dv) fp32 after each sequence, None unless wanted; kept, or None, spares
    the backward a pass over k and v."""
    dev, N, H, Dk, Dv, offsets = _decay_args(q, k, v, log_decay, offsets, ("initial_state", initial_state))
    code, log_decay = _lib.dtype_code(q), _f32(log_decay)
    first = None if initial_state is None else initial_state.contiguous()
    a, b, c = _Heads(q), _Heads(k), _Heads(v)
    o = torch.empty(v.shape, device=dev, dtype=v.dtype)
    last = torch.empty((N, H, Dk, Dv), device=dev, dtype=torch.float32) if want_state else None
    lib = _lib.load()
    ws = _lib.workspace(lib.mhc_decay_attention_workspace_bytes(a.R, N, H, Dk, Dv, int(offsets is not None), code), dev)
    with _lib.on_device(dev):
        _lib.check(lib.mhc_decay_attention_forward(*a.args(), *b.args(), *c.args(), code, log_decay.data_ptr(),
                                                   _lib.ptr(offsets), _lib.ptr(first), o.data_ptr(), _lib.ptr(last), a.R, N,
                                                   H, Dk, Dv, float(scale), _lib.ptr(ws), 0 if ws is None else ws.numel(),
                                                   _lib.stream(dev)), "decay_attention_forward")
    return o, last, ws


def decay_attention_backward(q, k, v, do, log_decay, offsets, initial_state, kept, d_state, scale: float,
                             need: Tuple[bool, bool, bool, bool]):
    """(dq, dk, dv, d_initial): None for what is not needed.  kept: the forward's third result, or None."""
    dev, N, H, Dk, Dv, offsets = _decay_args(q, k, v, log_decay, offsets, ("initial_state", initial_state),
                                             ("the state's gradient", d_state))
    if do.shape != v.shape:
        raise ShapeError(f"the output's gradient must be {tuple(v.shape)}, got {tuple(do.shape)}")
    _same_dtype("the output's gradient", do, q)
    _lib.require_gpu(q, do, kept)
    code, log_decay = _lib.dtype_code(q), _f32(log_decay)
    first = None if initial_state is None else initial_state.contiguous()
    d_last = None if d_state is None else d_state.contiguous()
    a, b, c, d = _Heads(q), _Heads(k), _Heads(v), _Heads(do)
    out = [torch.empty(t.shape, device=dev, dtype=t.dtype) if n else None for t, n in zip((q, k, v), need)]
    d_first = torch.empty((N, H, Dk, Dv), device=dev, dtype=torch.float32) if need[3] else None
    lib = _lib.load()
    packed = int(offsets is not None)
    states = lib.mhc_decay_attention_workspace_bytes(a.R, N, H, Dk, Dv, packed, code)
    if kept is not None:  # a saved-tensor hook may have changed it
        if kept.dtype != torch.uint8 or kept.numel() != states:
            raise ShapeError(f"kept must be the forward's, got {tuple(kept.shape)} {kept.dtype}")
        kept = kept.contiguous()
    ws = _lib.workspace(states if kept is not None else
                        lib.mhc_decay_attention_backward_workspace_bytes(a.R, N, H, Dk, Dv, packed, code), dev)
    with _lib.on_device(dev):
        _lib.check(lib.mhc_decay_attention_backward(*a.args(), *b.args(), *c.args(), *d.args(), code, log_decay.data_ptr(),
                                                    _lib.ptr(offsets), _lib.ptr(first), _lib.ptr(kept), _lib.ptr(d_last),
                                                    *(_lib.ptr(t) for t in out), _lib.ptr(d_first), a.R, N, H, Dk, Dv,
                                                    float(scale), _lib.ptr(ws), 0 if ws is None else ws.numel(),
                                                    _lib.stream(dev)), "decay_attention_backward")
    return (*out, d_first)


def check_step(q, k, v, log_decay, state, slots, state_out) -> torch.device:
    H, Dk, Dv = _head_dims(q, k, v)
    if q.dim() != 3:
        raise ShapeError(f"q must be (rows, heads, dim), got {tuple(q.shape)}")
    _check_decay(log_decay, H)
    if state.dim() != 4:
        raise ShapeError(f"state must be (states, {H}, {Dk}, {Dv}), got {tuple(state.shape)}")
    R, pool = q.shape[0], state.shape[0]
    for name, s in (("state", state), ("state_out", state_out)):
        _check_state(name, s, (pool, H, Dk, Dv))
        if s is not None and not s.is_contiguous():
            raise ShapeError(f"{name} must be contiguous: it is updated in place")
    if slots is None:
        if R > pool:
            raise ShapeError(f"{R} rows without slots for {pool} states")
    else:
        if tuple(slots.shape) != (R,):
            raise ShapeError(f"slots must be ({R},), got {tuple(slots.shape)}")
        if slots.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"mhc: slots must be int32 or int64, got {slots.dtype}")
    dev = _lib.require_gpu(q, k, v, log_decay, state, slots, state_out)
    if state_out is not None and state.numel():
        lo, hi = sorted((state.data_ptr(), state_out.data_ptr()))
        if lo != hi and lo + state.numel() * 4 > hi:
            raise ValueError("mhc: state and state_out must be the same or apart")
    return dev


def decay_attention_step(q, k, v, log_decay, state, slots, scale: float, state_out) -> torch.Tensor:
    """o (R, H, Dv); the rows' states go to state_out (state itself unless given)."""
    dev = check_step(q, k, v, log_decay, state, slots, state_out)
    R, H, Dk, Dv = *q.shape, v.shape[2]
    out = state if state_out is None else state_out
    code, log_decay = _lib.dtype_code(q), _f32(log_decay)
    if slots is not None:  # outside 32 bits is outside the pool, on either side
        slots = slots.clamp(-1, (1 << 31) - 1).int() if slots.dtype == torch.int64 else slots
        slots = slots.contiguous()
    a, b, c = _Heads(q), _Heads(k), _Heads(v)
    o = torch.empty(v.shape, device=dev, dtype=v.dtype)
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.mhc_decay_attention_step(*a.args(), *b.args(), *c.args(), code, log_decay.data_ptr(),
                                                _lib.ptr(slots), state.data_ptr(), out.data_ptr(), o.data_ptr(), R,
                                                state.shape[0], H, Dk, Dv, float(scale), _lib.stream(dev)),
                   "decay_attention_step")
    return o


# --------------------------------------------------------------------------
# Gated products
# --------------------------------------------------------------------------

def _gated_args(x, weight, offsets, activation):
    """(device, R, K, N, E, offsets, code of the activation)."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    want = 2 if offsets is None else 3
    if weight.dim() != want or weight.shape[-2] % 2:
        raise ShapeError(f"weight must be ({'' if want == 2 else 'experts, '}2 * out, in), got {tuple(weight.shape)}")
    E, N, K = (1 if want == 2 else weight.shape[0]), weight.shape[-2] // 2, weight.shape[-1]
    if x.dim() != 2 or x.shape[1] != K:
        raise ShapeError(f"x must be (rows, {K}), got {tuple(x.shape)}")
    _same_dtype("weight", weight, x)
    dev = _lib.require_gpu(x, weight, offsets)
    return dev, x.shape[0], K, N, E, None if offsets is None else _offsets(offsets, E), ACTIVATIONS[activation]


def gated_matmul_forward(x, weight, offsets, activation: str, want_saved: bool = True):
    """(y, saved): saved [R, 2 N] fp32 holds both products for the backward, None unless wanted."""
    dev, R, K, N, E, offsets, act = _gated_args(x, weight, offsets, activation)
    x, weight = x.contiguous(), weight.contiguous()
    y = torch.empty(R, N, device=dev, dtype=x.dtype)
    saved = torch.empty(R, 2 * N, device=dev, dtype=torch.float32) if want_saved else None
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.mhc_gated_matmul_forward(x.data_ptr(), weight.data_ptr(), _lib.dtype_code(x), _lib.ptr(offsets),
                                                act, y.data_ptr(), _lib.ptr(saved), R, K, N, E, _lib.stream(dev)),
                   "gated_matmul_forward")
    return y, saved


def gated_matmul_backward(dy, saved, x, weight, offsets, activation: str, need_dx: bool = True, need_dw: bool = True):
    """(dx, dweight): None for what is not needed."""
    dev, R, K, N, E, offsets, act = _gated_args(x, weight, offsets, activation)
    if tuple(dy.shape) != (R, N) or tuple(saved.shape) != (R, 2 * N) or saved.dtype != torch.float32:
        raise ShapeError(f"dy and saved must be ({R}, {N}) and ({R}, {2 * N}) fp32, got {tuple(dy.shape)}, "
                         f"{tuple(saved.shape)} {saved.dtype}")
    _same_dtype("dy", dy, x)
    _lib.require_gpu(x, dy, saved)
    if not (need_dx or need_dw):
        return None, None
    x, weight, dy, saved = x.contiguous(), weight.contiguous(), dy.contiguous(), saved.contiguous()
    code = _lib.dtype_code(x)
    dx = torch.empty_like(x) if need_dx else None
    dw = torch.empty_like(weight) if need_dw else None
    lib = _lib.load()
    ws = _lib.workspace(lib.mhc_gated_matmul_backward_workspace_bytes(R, N, code), dev)
    with _lib.on_device(dev):
        _lib.check(lib.mhc_gated_matmul_backward(dy.data_ptr(), saved.data_ptr(), x.data_ptr(), weight.data_ptr(), code,
                                                 _lib.ptr(offsets), act, _lib.ptr(dx), _lib.ptr(dw), R, K, N, E,
                                                 _lib.ptr(ws), 0 if ws is None else ws.numel(), _lib.stream(dev)),
                   "gated_matmul_backward")
    return dx, dw
