"""Launchers of the operators inside a branch (``mhc.branch``) over the C ABI.

Like ``_kernels.py``: argument checks, output allocation, one C-ABI call.  They know nothing of autograd.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib
from ._kernels import ShapeError, _f32

F8 = torch.float8_e4m3fn
E8 = torch.float8_e8m0fnu

#: Widest row of the norms (they hold a row in registers).
MAX_NORM_DIM = 16384
#: Values that share a scale in the 8-bit format.
MX_BLOCK = 32

Rng = Union[Tuple[int, int], torch.Tensor]


def _rows(x: torch.Tensor) -> Tuple[int, int]:
    if x.dim() < 1:
        raise ShapeError("expected at least one dimension (..., dim)")
    D = x.shape[-1]
    return (x.numel() // D if D else 0), D


def _same(x: torch.Tensor, t: Optional[torch.Tensor], name: str) -> None:
    if t is None:
        return
    if t.shape != x.shape:
        raise ShapeError(f"{name} must have the shape {tuple(x.shape)}, got {tuple(t.shape)}")
    if t.dtype != x.dtype:
        raise TypeError(f"mhc: {name} must be {x.dtype}, got {t.dtype}")


def _norm_args(x, weight, residual):
    _, D = _rows(x)
    if D > MAX_NORM_DIM:
        raise ShapeError(f"rows of {D} elements; at most {MAX_NORM_DIM}")
    if weight is not None and tuple(weight.shape) != (D,):
        raise ShapeError(f"weight must be ({D},), got {tuple(weight.shape)}")
    _same(x, residual, "residual")
    return _lib.require_gpu(x, weight, residual)


def scale_width(dim: int) -> int:
    """Bytes of a row's scales: one for each 32 values, filled up to a multiple of 4."""
    return -(-dim // 128) * 4


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def rms_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor], eps: float,
                     want_rstd: bool = True):
    """(y, h, rstd): h = x + residual, None without a residual; rstd [rows] fp32, None unless wanted."""
    dev = _norm_args(x, weight, residual)
    R, D = _rows(x)
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    weight = None if weight is None else _f32(weight)
    y = torch.empty_like(x)
    h = None if residual is None else torch.empty_like(x)
    rstd = torch.empty(x.shape[:-1], device=dev, dtype=torch.float32) if want_rstd else None
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.mhc_rms_norm_forward(x.data_ptr(), _lib.ptr(residual), _lib.dtype_code(x), _lib.ptr(weight),
                                            y.data_ptr(), _lib.ptr(h), _lib.ptr(rstd), R, D, float(eps),
                                            _lib.stream(dev)), "rms_norm_forward")
    return y, h, rstd


def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, dh: Optional[torch.Tensor],
                      weight: Optional[torch.Tensor], rstd: torch.Tensor, need_dx: bool = True,
                      need_dw: bool = True):
    """(dx, dweight): dweight [dim] fp32; None for what is not needed."""
    dev = _norm_args(h, weight, None)
    _same(h, dy, "dy")
    _same(h, dh, "dh")
    _lib.require_gpu(h, dy, dh, rstd)
    R, D = _rows(h)
    if rstd.shape != h.shape[:-1] or rstd.dtype != torch.float32:
        raise ShapeError(f"rstd must be {tuple(h.shape[:-1])} fp32, got {tuple(rstd.shape)} {rstd.dtype}")
    if not (need_dx or need_dw):
        return None, None
    h, dy, rstd = h.contiguous(), dy.contiguous(), rstd.contiguous()
    dh = None if dh is None else dh.contiguous()
    weight = None if weight is None else _f32(weight)
    dx = torch.empty_like(h) if need_dx else None
    dw = torch.empty(D, device=dev, dtype=torch.float32) if need_dw else None
    lib = _lib.load()
    ws = _lib.workspace(lib.mhc_rms_norm_backward_workspace_bytes(R, D), dev) if need_dw else None
    with _lib.on_device(dev):
        _lib.check(lib.mhc_rms_norm_backward(dy.data_ptr(), h.data_ptr(), _lib.ptr(dh), _lib.dtype_code(h),
                                             _lib.ptr(weight), rstd.data_ptr(), _lib.ptr(dx), _lib.ptr(dw), R, D,
                                             _lib.ptr(ws), 0 if ws is None else ws.numel(), _lib.stream(dev)),
                   "rms_norm_backward")
    return dx, dw


def _mx_outputs(x: torch.Tensor):
    D = x.shape[-1] if x.dim() else 0
    if x.dim() < 1 or D % MX_BLOCK:
        raise ShapeError(f"the 8-bit format needs rows of whole blocks of {MX_BLOCK}, got {tuple(x.shape)}")
    q = torch.empty(x.shape, device=x.device, dtype=F8)
    scales = torch.empty(*x.shape[:-1], scale_width(D), device=x.device, dtype=E8)
    return q, scales


def rms_norm_mx(x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor], eps: float):
    """(q, scales, h): the normalised rows in 8 bits; h None without a residual."""
    dev = _norm_args(x, weight, residual)
    R, D = _rows(x)
    q, scales = _mx_outputs(x)
    x = _aligned(x)
    residual = None if residual is None else _aligned(residual)
    weight = None if weight is None else _f32(weight)
    h = None if residual is None else torch.empty_like(x)
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.mhc_rms_norm_mx_forward(x.data_ptr(), _lib.ptr(residual), _lib.dtype_code(x),
                                               _lib.ptr(weight), q.data_ptr(), scales.data_ptr(), _lib.ptr(h), R, D,
                                               float(eps), _lib.stream(dev)), "rms_norm_mx_forward")
    return q, scales, h


def quantize_mx(x: torch.Tensor):
    """(q, scales) of rows (..., dim)."""
    dev = _lib.require_gpu(x)
    R, D = _rows(x)
    q, scales = _mx_outputs(x)
    x = _aligned(x)
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.mhc_quantize_mx(x.data_ptr(), _lib.dtype_code(x), q.data_ptr(), scales.data_ptr(), R, D,
                                       _lib.stream(dev)), "quantize_mx")
    return q, scales


def check_rng(x: torch.Tensor, rng: Rng) -> None:
    if isinstance(rng, torch.Tensor):
        if tuple(rng.shape) != (2,) or rng.dtype != torch.int64:
            raise ShapeError(f"rng must be two int64 values (seed, offset), got {tuple(rng.shape)} {rng.dtype}")
        _lib.require_gpu(x, rng)
        return
    if not (isinstance(rng, (tuple, list)) and len(rng) == 2 and all(isinstance(v, int) for v in rng)):
        raise TypeError("mhc: rng must be (seed, offset) as two ints or an int64 tensor of two on the GPU")
    if not all(0 <= v < 1 << 64 for v in rng):
        raise ValueError(f"seed and offset must be in [0, 2^64), got {tuple(rng)}")


def dropout(x: torch.Tensor, p: float, rng: Rng, residual: Optional[torch.Tensor] = None,
            want_used: bool = False):
    """(y, used): used holds the (seed, offset) that were drawn from, None unless wanted."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    check_rng(x, rng)
    _same(x, residual, "residual")
    dev = _lib.require_gpu(x, residual)
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    y = torch.empty_like(x)
    used = torch.empty(2, device=dev, dtype=torch.int64) if want_used else None
    state = rng.contiguous() if isinstance(rng, torch.Tensor) else None
    seed, offset = (0, 0) if state is not None else rng
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.mhc_dropout(x.data_ptr(), _lib.ptr(residual), _lib.dtype_code(x), y.data_ptr(), x.numel(),
                                   float(p), seed, offset, _lib.ptr(state), _lib.ptr(used), _lib.stream(dev)),
                   "dropout")
    return y, used


def _offsets(offsets: torch.Tensor, E: int) -> torch.Tensor:
    if tuple(offsets.shape) != (E,):
        raise ShapeError(f"offsets must be ({E},), the end of each expert's rows, got {tuple(offsets.shape)}")
    if offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"mhc: offsets must be int32 or int64, got {offsets.dtype}")
    if offsets.dtype == torch.int64:  # narrowed to the nearest: the kernels clamp what is out of range
        offsets = offsets.clamp(-(1 << 31), (1 << 31) - 1)
    return offsets.to(torch.int32).contiguous()


def _grouped_args(rows: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, width: int, name: str):
    """Checks rows [R, .] against weight [E, N, K] (axis `width` of it); returns (device, R, K, N, E)."""
    if weight.dim() != 3:
        raise ShapeError(f"weight must be (experts, out, in), got {tuple(weight.shape)}")
    E, N, K = weight.shape
    if rows.dim() != 2 or rows.shape[1] != weight.shape[width]:
        raise ShapeError(f"{name} must be (rows, {weight.shape[width]}), got {tuple(rows.shape)}")
    return _lib.require_gpu(rows, weight, offsets), rows.shape[0], K, N, E


def grouped_matmul_forward(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """y [R, N]: each row times its expert's weight."""
    dev, R, K, N, E = _grouped_args(x, weight, offsets, 2, "x")
    if weight.dtype != x.dtype:
        raise TypeError(f"mhc: weight must be {x.dtype}, got {weight.dtype}")
    offsets = _offsets(offsets, E)
    x, weight = x.contiguous(), weight.contiguous()
    y = torch.empty(R, N, device=dev, dtype=x.dtype)
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.mhc_grouped_matmul_forward(x.data_ptr(), weight.data_ptr(), _lib.dtype_code(x),
                                                  offsets.data_ptr(), y.data_ptr(), R, K, N, E, _lib.stream(dev)),
                   "grouped_matmul_forward")
    return y


def grouped_matmul_backward_input(dy: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """dx [R, K]."""
    dev, R, K, N, E = _grouped_args(dy, weight, offsets, 1, "dy")
    if weight.dtype != dy.dtype:
        raise TypeError(f"mhc: dy must be {weight.dtype}, got {dy.dtype}")
    offsets = _offsets(offsets, E)
    dy, weight = dy.contiguous(), weight.contiguous()
    dx = torch.empty(R, K, device=dev, dtype=dy.dtype)
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.mhc_grouped_matmul_backward_input(dy.data_ptr(), weight.data_ptr(), _lib.dtype_code(dy),
                                                         offsets.data_ptr(), dx.data_ptr(), R, K, N, E,
                                                         _lib.stream(dev)), "grouped_matmul_backward_input")
    return dx


def grouped_matmul_backward_weight(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """dweight [E, N, K] in x's dtype, one expert for each entry of offsets."""
    if dy.dim() != 2 or x.dim() != 2 or dy.shape[0] != x.shape[0] or offsets.dim() != 1:
        raise ShapeError(f"dy, x and offsets must be (rows, out), (rows, in) and (experts,), got {tuple(dy.shape)}, "
                         f"{tuple(x.shape)}, {tuple(offsets.shape)}")
    if dy.dtype != x.dtype:
        raise TypeError(f"mhc: dy must be {x.dtype}, got {dy.dtype}")
    dev = _lib.require_gpu(dy, x, offsets)
    (R, N), K, E = dy.shape, x.shape[1], offsets.shape[0]
    offsets = _offsets(offsets, E)
    dy, x = dy.contiguous(), x.contiguous()
    dw = torch.empty(E, N, K, device=dev, dtype=x.dtype)
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.mhc_grouped_matmul_backward_weight(dy.data_ptr(), x.data_ptr(), _lib.dtype_code(x),
                                                          offsets.data_ptr(), dw.data_ptr(), R, K, N, E,
                                                          _lib.stream(dev)), "grouped_matmul_backward_weight")
    return dw


def grouped_matmul_mx(q: torch.Tensor, scales: torch.Tensor, weight_q: torch.Tensor, weight_scales: torch.Tensor,
                      offsets: torch.Tensor, out_dtype: torch.dtype) -> torch.Tensor:
    """y [R, N] of 8-bit rows and weights."""
    if q.dtype != F8 or weight_q.dtype != F8 or scales.dtype != E8 or weight_scales.dtype != E8:
        raise TypeError(f"mhc: 8-bit values must be {F8} and scales {E8}, got {q.dtype}, {weight_q.dtype}, "
                        f"{scales.dtype}, {weight_scales.dtype}")
    if out_dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"mhc: out_dtype must be bfloat16 or float16, got {out_dtype}")
    dev, R, K, N, E = _grouped_args(q, weight_q, offsets, 2, "q")
    if K % MX_BLOCK:
        raise ShapeError(f"the 8-bit format needs rows of whole blocks of {MX_BLOCK}, got {K}")
    ns = scale_width(K)
    if tuple(scales.shape) != (R, ns) or tuple(weight_scales.shape) != (E, N, ns):
        raise ShapeError(f"scales must be ({R}, {ns}) and weight_scales ({E}, {N}, {ns}); got {tuple(scales.shape)}, "
                         f"{tuple(weight_scales.shape)}")
    _lib.require_gpu(q, scales, weight_q, weight_scales)
    offsets = _offsets(offsets, E)
    y = torch.empty(R, N, device=dev, dtype=out_dtype)
    code = _lib.dtype_code(y)
    q, scales, weight_q, weight_scales = (_aligned(t) for t in (q, scales, weight_q, weight_scales))
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.mhc_grouped_matmul_mx(q.data_ptr(), scales.data_ptr(), weight_q.data_ptr(),
                                             weight_scales.data_ptr(), offsets.data_ptr(), y.data_ptr(), code, R, K,
                                             N, E, _lib.stream(dev)), "grouped_matmul_mx")
    return y
