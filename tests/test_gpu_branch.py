"""``mhc.branch`` on the GPU against the float64 oracle (oracle/branch_oracle.py).

Tolerances.  Every op computes in fp32 from its stored inputs and rounds once.  An fp32 sum of n terms, in
any order, is within n 2^-24 of the sum of their magnitudes; the norms add in trees (depth below 32), the
products in chains of at most K terms plus what the matrix instruction does inside (2^-23 allows for it).
16-bit outputs are checked with helpers.assert_rounded_once, whose allowance is one unit in the last place and
2^-21 of the terms' magnitudes.
"""

import numpy as np
import pytest
import torch

from helpers import assert_rounded_once, to_np
from test_gpu_native_nodes import both, same
from mhc import _branch, branch
from oracle import branch_oracle as O

pytestmark = pytest.mark.gpu

DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rand(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def close(got, ref, size, tol, what=""):
    """|got - ref| <= tol * size + one rounding to got's dtype, everywhere."""
    got_np = to_np(got)
    allowed = tol * np.abs(size) + 1.01 * HALF_ULP[got.dtype] * np.abs(ref) + 1e-37
    if got.dtype == torch.float16:
        allowed = allowed + 2.0 ** -25  # subnormal spacing
    assert got_np.shape == ref.shape, what
    worst = float((np.abs(got_np - ref) / allowed).max()) if ref.size else 0.0
    print(f"{what}: worst/allowed {worst:.3f}", flush=True)
    assert worst <= 1.0, (what, worst)


# --------------------------------------------------------------------------
# RMS norm
# --------------------------------------------------------------------------

# widths around a vector, a wave's and a workgroup's reach, odd ones among them
WIDTHS = [1, 3, 7, 8, 64, 100, 500, 512, 1024, 1500, 2050, 4096, 7168, 8191, 16384]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("D", WIDTHS)
def test_rms_norm_forward_and_backward(D, residual, dtype):
    R, dt = (37 if D < 4096 else 5), DT[dtype]
    x = rand(R, D, seed=1, dtype=dt, scale=1.5).requires_grad_()
    w = rand(D, seed=2).add_(1.0).requires_grad_()
    dy = rand(R, D, seed=4, dtype=dt)
    if residual:
        res = rand(R, D, seed=3, dtype=dt).requires_grad_()
        dh = rand(R, D, seed=5, dtype=dt)
        y, h = branch.rms_norm(x, w, residual=res)
        assert torch.equal(h, x + res)
        dx, dres, dw = torch.autograd.grad((y, h), (x, res, w), (dy, dh))
        assert torch.equal(dx, dres)
    else:
        h, dh = x, None
        y = branch.rms_norm(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
    ref, _ = O.rms_norm(to_np(h), to_np(w))
    rx, rw, sx, sw = O.rms_norm_backward(to_np(dy), to_np(h), None if dh is None else to_np(dh), to_np(w))
    assert dw.dtype == torch.float32 and dx.dtype == dt and y.dtype == dt
    close(y, ref, ref, 2.0 ** -20, "y")
    close(dx, rx, sx, 2.0 ** -19, "dx")
    close(dw, rw, sw, 2.0 ** -19, "dw")
    with torch.no_grad():  # the forward alone gives the same bits
        out = branch.rms_norm(x, w, residual=res if residual else None)
        assert torch.equal(out[0] if residual else out, y)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_rms_norm_rounds_once(dtype):
    x, w = rand(64, 2048, seed=1, dtype=DT[dtype]), rand(2048, seed=2)
    y = branch.rms_norm(x, w)
    ref = torch.from_numpy(O.rms_norm(to_np(x), to_np(w))[0])
    assert_rounded_once(y.cpu(), ref, ref.abs(), "rms_norm")


@pytest.mark.parametrize("D", [512, 1500, 8192])
def test_rms_norm_gradient_against_differences(D):
    """Central differences along a random direction, in fp32: t^2 / 6 of the third derivative (of order one
    here, per unit of direction) and the outputs' 2^-22 over t bound the error; t = 2^-6."""
    R, t = 8, 2.0 ** -6
    x, w, res = rand(R, D, seed=1), rand(D, seed=2).add_(1.0), rand(R, D, seed=3)
    dy, dh = rand(R, D, seed=4), rand(R, D, seed=5)
    leaves = [v.clone().requires_grad_() for v in (x, w, res)]
    y, h = branch.rms_norm(leaves[0], leaves[1], residual=leaves[2])
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))

    def loss(x, w, res):
        y, h = branch.rms_norm(x, w, residual=res)
        return float((y.double() * dy.double()).sum() + (h.double() * dh.double()).sum())

    for i, (leaf, g) in enumerate(zip((x, w, res), grads)):
        v = rand(*leaf.shape, seed=10 + i)
        up, down = [[u + s * t * v if j == i else u for j, u in enumerate((x, w, res))] for s in (1, -1)]
        diff = (loss(*up) - loss(*down)) / (2 * t)
        # the same number of terms of order one as the inner product has
        scale = float((g.double() * v.double()).square().sum().sqrt()) + (R * D) ** 0.5
        assert abs(diff - float((g.double() * v.double()).sum())) < 1e-2 * scale, i


def test_rms_norm_optional_weight_and_needed_gradients():
    x, dy = rand(9, 256, seed=1, dtype=torch.bfloat16).requires_grad_(), rand(9, 256, seed=2, dtype=torch.bfloat16)
    y = branch.rms_norm(x)
    dx, = torch.autograd.grad(y, x, dy)
    rx, _, sx, _ = O.rms_norm_backward(to_np(dy), to_np(x))
    close(y, O.rms_norm(to_np(x))[0], 1.0, 2.0 ** -20, "y")
    close(dx, rx, sx, 2.0 ** -19, "dx")
    # only the weight's gradient, in the weight's own dtype and shape
    w = rand(256, seed=3, dtype=torch.bfloat16).requires_grad_()
    y = branch.rms_norm(x.detach(), w)
    dw, = torch.autograd.grad(y, w, dy)
    _, rw, _, sw = O.rms_norm_backward(to_np(dy), to_np(x), None, to_np(w))
    assert dw.dtype == torch.bfloat16
    close(dw, rw, sw, 2.0 ** -19, "dw")
    # only h is used: its gradient passes through
    res = rand(9, 256, seed=4, dtype=torch.bfloat16).requires_grad_()
    _, h = branch.rms_norm(x, w, residual=res)
    dx, dres = torch.autograd.grad(h, (x, res), dy)
    assert torch.equal(dx, dy) and torch.equal(dres, dy)
    # only y is used
    y, _ = branch.rms_norm(x, w, residual=res)
    dx, = torch.autograd.grad(y, x, dy)
    rx, _, sx, _ = O.rms_norm_backward(to_np(dy), to_np((x + res)), None, to_np(w))
    close(dx, rx, sx, 2.0 ** -19, "dx of y")


def test_rms_norm_extremes():
    z = torch.zeros(3, 64, device=DEV)
    assert torch.equal(branch.rms_norm(z), z)  # eps carries a row of zeros
    x = rand(4, 1500, seed=1)
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    y = branch.rms_norm(x)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, 9]) and not y[2, :9].any()
    assert torch.equal(y[[0, 3]], branch.rms_norm(x[[0, 3]]))  # other rows untouched
    for shape in ((0, 64), (4, 0), (2, 0, 64)):
        e = torch.zeros(shape, device=DEV, requires_grad=True)
        w = torch.ones(shape[-1], device=DEV, requires_grad=True)
        y = branch.rms_norm(e, w)
        assert y.shape == e.shape
        dx, dw = torch.autograd.grad(y.sum(), (e, w))
        assert dx.shape == e.shape and not dw.any()


def test_rms_norm_strides_and_alignment():
    base = rand(6, 2, 520, seed=1, dtype=torch.bfloat16)
    ref = branch.rms_norm(base[:, 1, :512].contiguous())
    assert torch.equal(branch.rms_norm(base[:, 1, :512]), ref)  # strided rows
    flat = rand(4 * 512 + 1, seed=2, dtype=torch.bfloat16)
    x = flat[1:].view(4, 512)  # two bytes past a 16-byte boundary
    y, h = branch.rms_norm(x, residual=x)
    want, wh = branch.rms_norm(x.clone(), residual=x.clone())
    assert torch.equal(h, wh)
    close(y, O.rms_norm(to_np(h))[0], 1.0, 2.0 ** -20, "unaligned")
    assert float((y.float() - want.float()).abs().max()) <= 2.0 ** -6  # a bf16 step of values below 4
    q, s = branch.rms_norm_mx(x)
    qa, sa = branch.rms_norm_mx(x.clone())
    assert torch.equal(q.view(torch.uint8), qa.view(torch.uint8)) and torch.equal(s.view(torch.uint8), sa.view(torch.uint8))
    t = rand(512, 6, seed=3)
    assert torch.equal(branch.rms_norm(t.T), branch.rms_norm(t.T.contiguous()))


@pytest.mark.parametrize("R", [1, 64, 65, 511, 513, 4099])
def test_rms_norm_row_counts_and_repeatability(R):
    """More rows than the backward has workgroups, fewer, few and one: the same bits each time."""
    D = 250
    x, w = rand(R, D, seed=1, dtype=torch.bfloat16).requires_grad_(), rand(D, seed=2).requires_grad_()
    dy = rand(R, D, seed=3, dtype=torch.bfloat16)
    runs = []
    for _ in range(3):
        y = branch.rms_norm(x, w)
        runs.append((y.detach(), *torch.autograd.grad(y, (x, w), dy)))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
    rx, rw, sx, sw = O.rms_norm_backward(to_np(dy), to_np(x), None, to_np(w))
    close(runs[0][1], rx, sx, 2.0 ** -19, "dx")
    close(runs[0][2], rw, sw, 2.0 ** -19, "dw")


# --------------------------------------------------------------------------
# 8 bits
# --------------------------------------------------------------------------

def mx_values(q, scales):
    n = q.shape[-1] // 32
    k = to_np(scales.view(torch.uint8))[..., :n] - 127.0
    v = to_np(q.float()).reshape(*q.shape[:-1], n, 32) * np.exp2(k)[..., None]
    return v.reshape(q.shape)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(1, 32), (5, 64), (3, 7, 160), (2, 4096), (1000, 96)])
def test_quantize_mx_bits(shape, dtype):
    x = rand(*shape, seed=1, dtype=DT[dtype])
    x *= torch.exp2(torch.arange(shape[-1], device=DEV) % 23 - 11).to(x.dtype)
    flat = x.view(-1)
    flat[:4] = torch.tensor([448.0, -448.0, 0.0, 1.75], device=DEV).to(x.dtype)
    q, s = branch.quantize_mx(x)
    k = O.mx_exponents(to_np(x))
    n = shape[-1] // 32
    assert s.shape == (*shape[:-1], -(-shape[-1] // 128) * 4)
    bytes_ = s.view(torch.uint8).cpu().numpy()
    assert np.array_equal(bytes_[..., :n], k + 127) and not bytes_[..., n:].any()
    ref = O.e4m3_round(to_np(x).reshape(*shape[:-1], n, 32) / np.exp2(k.astype(float))[..., None])
    assert np.array_equal(to_np(q.float()).reshape(ref.shape), ref)


def test_quantize_mx_extremes():
    x = torch.zeros(6, 64, device=DEV)
    x[1, 3] = float("nan")
    x[2, 40] = -float("inf")
    x[3, 5] = torch.finfo(torch.float32).max
    x[4, 6] = 1e-45
    q, s = branch.quantize_mx(x)
    b = s.view(torch.uint8).cpu()
    assert not q[0].float().any() and b[0].tolist() == [0, 0, 0, 0]
    assert b[1].tolist() == [255, 0, 0, 0] and torch.isnan(q[1, :32].float()).all() and not q[1, 32:].float().any()
    assert b[2].tolist() == [0, 255, 0, 0] and torch.isnan(q[2, 32:].float()).all()
    assert b[3, 0] == 127 + 120 and float(q[3, 5].float()) == 256.0  # just below 2^128
    assert b[4, 0] == 0 and float(q[4, 6].float()) == 0.0  # 2^-149 over 2^-127
    assert branch.quantize_mx(torch.zeros(0, 64, device=DEV))[0].shape == (0, 64)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("D", [32, 96, 512, 1504, 4096, 7168, 16384])
def test_rms_norm_mx(D, residual, dtype):
    R, dt = 19, DT[dtype]
    x, w = rand(R, D, seed=1, dtype=dt), rand(D, seed=2).add_(1.0)
    res = rand(R, D, seed=3, dtype=dt) if residual else None
    out = branch.rms_norm_mx(x, w, residual=res)
    h = out[2] if residual else x
    if residual:
        assert torch.equal(h, x + res)
    ref, _ = O.rms_norm(to_np(h), to_np(w))
    q, s = out[0], out[1]
    n = D // 32
    b = s.view(torch.uint8).cpu().numpy().astype(int)
    assert not b[..., n:].any()
    # a scale may differ only where the block's largest value is within the fp32 error of a boundary
    top = np.abs(ref).reshape(R, n, 32).max(-1)
    lo, hi = O.mx_exponent(top * (1 - 2.0 ** -20)), O.mx_exponent(top * (1 + 2.0 ** -20))
    assert ((b[:, :n] - 127 >= lo) & (b[:, :n] - 127 <= hi)).all()
    # half a step: 2^-4 of the value, or 2^-10 of the scale where the format has fixed steps
    scale = np.repeat(np.exp2(b[:, :n] - 127.0), 32, -1)
    err = np.abs(mx_values(q, s) - ref)
    assert (err <= (np.abs(ref) * 2.0 ** -4 + 2.0 ** -10 * scale) * (1 + 2.0 ** -18)).all()


# --------------------------------------------------------------------------
# Dropout
# --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 2048, 100003])
def test_dropout(n, residual, dtype):
    dt, p, seed, offset = DT[dtype], 0.3, 0x123456789ABCDEF0, 5
    x = rand(n, seed=1, dtype=dt).requires_grad_()
    res = rand(n, seed=2, dtype=dt).requires_grad_() if residual else None
    dy = rand(n, seed=3, dtype=dt)
    f = O.dropout_factors(n, p, seed, offset)
    y = branch.dropout(x, p, (seed, offset), residual=res)
    ref = to_np(x) * f
    size = np.abs(ref)
    if residual:
        ref, size = ref + to_np(res), size + np.abs(to_np(res))
    close(y, ref, size, 2.0 ** -23, "y")
    if residual:
        dx, dres = torch.autograd.grad(y, (x, res), dy)
        assert torch.equal(dres, dy)
    else:
        dx, = torch.autograd.grad(y, x, dy)
        assert np.array_equal(to_np(y) == 0, (f == 0) | (to_np(x) == 0))
    close(dx, to_np(dy) * f, to_np(dy) * f, 2.0 ** -23, "dx")


def test_dropout_mask_depends_on_seed_offset_and_index_only():
    x = torch.ones(64, 513, device=DEV)
    y = branch.dropout(x, 0.5, (7, 1))
    assert torch.equal(y, branch.dropout(x, 0.5, (7, 1)))
    assert not torch.equal(y, branch.dropout(x, 0.5, (7, 2))) and not torch.equal(y, branch.dropout(x, 0.5, (8, 1)))
    assert torch.equal(y.view(-1), branch.dropout(x.view(-1), 0.5, (7, 1)))
    assert torch.equal(y != 0, branch.dropout(x.to(torch.bfloat16), 0.5, (7, 1)) != 0)
    wide = torch.ones(64, 600, device=DEV)[:, :513]  # strided rows count as their logical order
    assert torch.equal(y, branch.dropout(wide, 0.5, (7, 1)))
    off = torch.ones(64 * 513 + 1, device=DEV)[1:]  # unaligned
    assert torch.equal(y.view(-1), branch.dropout(off, 0.5, (7, 1)))
    state = torch.tensor([7, 1], device=DEV)
    assert torch.equal(y, branch.dropout(x, 0.5, state))
    big = (2 ** 64 - 1, 2 ** 63 + 5)
    f = O.dropout_factors(x.numel(), 0.5, *big)
    assert np.array_equal(to_np(branch.dropout(x, 0.5, big)).reshape(-1), f)
    signed = torch.tensor([-1, 5 - 2 ** 63], device=DEV)
    assert np.array_equal(to_np(branch.dropout(x, 0.5, signed)).reshape(-1), f)


def test_dropout_probabilities():
    x = rand(1 << 20, seed=1)
    for p in (0.0, 0.1, 0.5, 0.9, 1.0, 1e-7):
        y = branch.dropout(x, p, (3, 4))
        kept = float((y != 0).double().mean())
        q = round((1 - p) * 65536) / 65536
        assert abs(kept - q) <= 5 * (q * (1 - q) / x.numel()) ** 0.5 + 1e-9, p  # five deviations
        if p in (0.0, 1e-7):
            assert torch.equal(y, x)
        if p == 1.0:
            assert not y.any()
    assert torch.equal(branch.dropout(x, 0.7, (3, 4), training=False), x)
    assert torch.equal(branch.dropout(x, 0.7, (3, 4), residual=x, training=False), x + x)
    bad = x[:1024].clone()
    bad[:] = float("nan")
    y = branch.dropout(bad, 0.5, (3, 4))
    f = O.dropout_factors(1024, 0.5, 3, 4)
    assert np.array_equal(np.isnan(to_np(y)), f != 0) and not to_np(y)[f == 0].any()
    assert branch.dropout(x[:0], 0.5, (3, 4)).shape == (0,)


def test_dropout_backward_uses_the_state_of_its_forward():
    x = torch.ones(4096, device=DEV, requires_grad=True)
    state = torch.tensor([11, 0], device=DEV)
    ys = []
    for _ in range(3):
        ys.append(branch.dropout(x, 0.5, state))
        state[1] += 1
    for y in ys:
        dx, = torch.autograd.grad(y.sum(), x)
        assert torch.equal(dx, y.detach())
    assert not torch.equal(ys[0], ys[1])


# --------------------------------------------------------------------------
# Products grouped by expert
# --------------------------------------------------------------------------

SPLITS = {
    "even": lambda R, E: [R * (i + 1) // E for i in range(E)],
    "one has all": lambda R, E: [0] * (E // 2) + [R] * (E - E // 2),
    "empty ends": lambda R, E: [0] + [R * i // E for i in range(1, E - 1)] + [R * (E - 2) // E],  # rows past the last
    "none": lambda R, E: [0] * E,
    "single rows": lambda R, E: [min(i + 1, R) for i in range(E - 1)] + [R],
}


def offsets_of(split, R, E, dtype=torch.int32):
    return torch.tensor(SPLITS[split](R, E), dtype=dtype, device=DEV)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("R,K,N,E,split", [
    (1, 8, 8, 1, "even"), (1, 64, 64, 3, "one has all"), (7, 1, 1, 2, "even"), (5, 3, 130, 4, "single rows"),
    (64, 128, 256, 8, "even"), (300, 72, 136, 5, "empty ends"), (300, 129, 65, 5, "one has all"),
    (1000, 256, 200, 70, "single rows"), (257, 500, 1001, 3, "even"), (130, 96, 64, 4, "none"),
    (700, 640, 384, 130, "even"), (1024, 1024, 512, 4, "empty ends"), (90, 2048, 264, 6, "empty ends"),
    (2000, 512, 768, 2, "one has all"), (300, 136, 2056, 4, "even"), (1100, 1032, 1048, 5, "empty ends"),
    (2100, 1032, 2056, 5, "empty ends"), (4100, 264, 2048, 3, "one has all"), (1500, 1026, 1030, 6, "even"),
    (4100, 264, 4104, 3, "even"), (4100, 4104, 264, 3, "empty ends"), (600, 2056, 2312, 3, "even"),
    (4360, 136, 4104, 16, "single rows"),
])
def test_grouped_matmul(R, K, N, E, split, dtype):
    dt = DT[dtype]
    x = rand(R, K, seed=1, dtype=dt).requires_grad_()
    w = rand(E, N, K, seed=2, dtype=dt, scale=K ** -0.5).requires_grad_()
    dy = rand(R, N, seed=3, dtype=dt)
    off = offsets_of(split, R, E)
    y = branch.grouped_matmul(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    o = off.tolist()
    ref, size = O.grouped_matmul(to_np(x), to_np(w), o)
    rx, rw, sx, sw = O.grouped_matmul_backward(to_np(dy), to_np(x), to_np(w), o)
    assert y.dtype == dx.dtype == dw.dtype == dt
    close(y, ref, size, (K + 8) * 2.0 ** -23, "y")
    close(dx, rx, sx, (N + 8) * 2.0 ** -23, "dx")
    close(dw, rw, sw, (R + 8) * 2.0 ** -23, "dw")
    with torch.no_grad():
        assert torch.equal(branch.grouped_matmul(x, w, off.long()), y)


@pytest.mark.parametrize("R,K,N,E", [(40, 64, 96, 3), (600, 256, 384, 4), (33, 100, 77, 2)])
def test_grouped_matmul_gradient_against_differences(R, K, N, E):
    """The product is linear in each operand: differences are exact but for the fp32 sums."""
    x, w, dy = rand(R, K, seed=1), rand(E, N, K, seed=2), rand(R, N, seed=3)
    off = offsets_of("even", R, E)
    lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(branch.grouped_matmul(lx, lw, off), (lx, lw), dy)
    vx, vw = rand(R, K, seed=4), rand(E, N, K, seed=5)
    loss = lambda x, w: float((branch.grouped_matmul(x, w, off).double() * dy.double()).sum())  # noqa: E731
    n = (R * N * K) ** 0.5  # the loss's typical size; 2^-18 of it is far above the sums' errors
    assert abs((loss(x + vx, w) - loss(x - vx, w)) / 2 - float((dx.double() * vx.double()).sum())) < 2.0 ** -18 * n * 4
    assert abs((loss(x, w + vw) - loss(x, w - vw)) / 2 - float((dw.double() * vw.double()).sum())) < 2.0 ** -18 * n * 4


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_grouped_matmul_rows_of_other_experts_do_not_leak(dtype):
    """NaN and infinity in one expert's rows and weights, and in the rows of none, stay there."""
    dt, (R, K, N, E) = DT[dtype], (200, 72, 136, 4)
    off = torch.tensor([50, 90, 91, 150], dtype=torch.int32, device=DEV)
    x, w, dy = rand(R, K, seed=1, dtype=dt), rand(E, N, K, seed=2, dtype=dt), rand(R, N, seed=3, dtype=dt)
    clean = [t.clone().requires_grad_() for t in (x, w)]
    y0 = branch.grouped_matmul(*clean, off)
    g0 = torch.autograd.grad(y0, clean, dy)
    for t in (x, dy):
        t[50:90] = float("nan")
        t[150:] = float("inf")
    w[1] = float("inf")
    dirty = [t.clone().requires_grad_() for t in (x, w)]
    y1 = branch.grouped_matmul(*dirty, off)
    g1 = torch.autograd.grad(y1, dirty, dy)
    keep = [i for i in range(R) if not 50 <= i < 90]
    assert torch.equal(y0[keep], y1[keep]) and torch.equal(g0[0][keep], g1[0][keep])
    assert not y1[150:].any() and not g1[0][150:].any()
    assert torch.equal(g0[1][[0, 2, 3]], g1[1][[0, 2, 3]])
    assert torch.isnan(y1[50:90]).all() and torch.isnan(g1[1][1]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_grouped_matmul_large_tiles_do_not_leak(dtype):
    """The same where experts end inside the largest tiles, one of them has no rows and K ends inside a slab."""
    dt, (R, K, N, E) = DT[dtype], (2500, 2056, 4104, 4)
    ends = [1000, 1000, 1277, 2300]
    off = torch.tensor(ends, dtype=torch.int32, device=DEV)
    x, w, dy = rand(R, K, seed=1, dtype=dt), rand(E, N, K, seed=2, dtype=dt), rand(R, N, seed=3, dtype=dt)
    clean = [t.clone().requires_grad_() for t in (x, w)]
    y0 = branch.grouped_matmul(*clean, off)
    g0 = torch.autograd.grad(y0, clean, dy)
    for t in (x, dy):
        t[1000:1277] = float("nan")
        t[2300:] = float("inf")
    w[1:3] = float("inf")
    dirty = [t.clone().requires_grad_() for t in (x, w)]
    y1 = branch.grouped_matmul(*dirty, off)
    g1 = torch.autograd.grad(y1, dirty, dy)
    for a, b in ((y0, y1), (g0[0], g1[0])):
        assert torch.equal(a[:1000], b[:1000]) and torch.equal(a[1277:2300], b[1277:2300])
        assert torch.isnan(b[1000:1277]).all() and not b[2300:].any()
    assert torch.equal(g0[1][[0, 3]], g1[1][[0, 3]])
    assert not g1[1][1].any() and torch.isnan(g1[1][2]).all()


def test_grouped_matmul_offsets_out_of_range_are_clamped():
    x, w = rand(20, 32, seed=1), rand(3, 16, 32, seed=2)
    want = branch.grouped_matmul(x, w, torch.tensor([0, 20, 20], dtype=torch.int32, device=DEV))
    got = branch.grouped_matmul(x, w, torch.tensor([-5, 1000, 2000], dtype=torch.int32, device=DEV))
    assert torch.equal(want, got)


@pytest.mark.parametrize("R,K", [(60, 32), (3000, 32), (3000, 33)])
def test_grouped_matmul_offsets_that_run_backwards(R, K):
    """They count as their running maximum, in whatever kernel: experts share no row and leave none out."""
    x, w = rand(R, K, seed=1), rand(3, 40, K, seed=2)
    y = branch.grouped_matmul(x, w, torch.tensor([R * 2 // 3, R // 6, R], dtype=torch.int32, device=DEV))
    for rows, e in ((slice(0, R // 6), 0), (slice(R * 2 // 3, R), 2)):
        ref, size = O.grouped_matmul(to_np(x[rows]), to_np(w[e:e + 1]), [x[rows].shape[0]])
        close(y[rows], ref, size, (K + 8) * 2.0 ** -23, "y")


@pytest.mark.parametrize("E", [5, 70, 200])
@pytest.mark.parametrize("K", [32, 33])
def test_grouped_matmul_offsets_count_as_their_running_maximum(K, E):
    R, N = 900, 40
    x, w = rand(R, K, seed=1).requires_grad_(), rand(E, N, K, seed=2).requires_grad_()
    dy = rand(R, N, seed=3)
    off = torch.from_numpy(np.random.default_rng(4).integers(-50, R // 2, E).astype(np.int32)).to(DEV)
    off[E // 2:] += R // 2 + 20
    got = [branch.grouped_matmul(x, w, o) for o in (off, off.clamp(0, R).cummax(0).values.int())]
    grads = [torch.autograd.grad(y, (x, w), dy) for y in got]
    assert torch.equal(*got) and all(torch.equal(a, b) for a, b in zip(*grads))


def test_grouped_matmul_empty_sizes():
    off = torch.zeros(3, dtype=torch.int32, device=DEV)
    for R, K, N in ((0, 8, 8), (4, 0, 8), (4, 8, 0)):
        x = torch.ones(R, K, device=DEV, requires_grad=True)
        w = torch.ones(3, N, K, device=DEV, requires_grad=True)
        o = torch.tensor([R // 2, R, R], dtype=torch.int32, device=DEV)
        y = branch.grouped_matmul(x, w, o)
        assert y.shape == (R, N) and not y.any()
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == x.shape and dw.shape == w.shape and not dx.any() and not dw.any()
    y = branch.grouped_matmul(torch.ones(4, 8, device=DEV), torch.ones(0, 8, 8, device=DEV), off[:0])
    assert y.shape == (4, 8) and not y.any()


def test_grouped_matmul_strides_alignment_and_repeatability():
    R, K, N, E = 70, 96, 80, 3
    off = offsets_of("even", R, E)
    x, w, dy = (rand(*s, seed=i, dtype=torch.bfloat16) for i, s in enumerate([(R, K), (E, N, K), (R, N)]))
    y = branch.grouped_matmul(x, w, off)
    assert torch.equal(branch.grouped_matmul(x, w, off), y)
    xs = torch.zeros(R, 2 * K, device=DEV, dtype=x.dtype)[:, ::2]
    xs.copy_(x)
    ws = w.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(branch.grouped_matmul(xs, ws, off), y)
    flat = torch.zeros(R * K + 1, device=DEV, dtype=x.dtype)
    flat[1:] = x.view(-1)
    xu = flat[1:].view(R, K)  # two bytes past a 16-byte boundary
    ref, size = O.grouped_matmul(to_np(x), to_np(w), off.tolist())
    close(branch.grouped_matmul(xu, w, off), ref, size, (K + 8) * 2.0 ** -23, "unaligned")
    lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = branch.grouped_matmul(lx, lw, off)
    a = torch.autograd.grad(out, (lx, lw), dy, retain_graph=True)
    b = torch.autograd.grad(out, (lx, lw), dy.T.contiguous().T)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # a broadcast gradient, as sum() gives it
    c = torch.autograd.grad(branch.grouped_matmul(lx, lw, off).sum(), (lx, lw))
    d = torch.autograd.grad(branch.grouped_matmul(lx, lw, off), (lx, lw), torch.ones_like(dy))
    assert torch.equal(c[0], d[0]) and torch.equal(c[1], d[1])


@pytest.mark.parametrize("out", ["bf16", "fp16"])  # fp32 is refused
@pytest.mark.parametrize("R,K,N,E,split", [
    (1, 32, 8, 1, "even"), (3, 96, 33, 2, "even"), (64, 128, 128, 8, "even"), (129, 160, 257, 5, "empty ends"),
    (40, 1024, 64, 40, "single rows"), (600, 512, 384, 3, "one has all"), (16, 4096, 72, 4, "even"),
    (77, 64, 100, 3, "none"), (900, 416, 1100, 5, "empty ends"), (4200, 288, 2056, 3, "empty ends"),
    (4200, 288, 4104, 3, "empty ends"),
])
def test_grouped_matmul_mx(R, K, N, E, split, out):
    x, w = rand(R, K, seed=1), rand(E, N, K, seed=2, scale=K ** -0.5)
    # block scales far apart
    x *= torch.exp2((torch.arange(K, device=DEV) // 32) % 7 - 3.0)
    w *= torch.exp2((torch.arange(N, device=DEV) % 5) - 2.0)[None, :, None]
    q, s = branch.quantize_mx(x)
    wq, ws = branch.quantize_mx(w)
    off = offsets_of(split, R, E)
    y = branch.grouped_matmul_mx(q, s, wq, ws, off, out_dtype=DT[out])
    ref, size = O.grouped_matmul(mx_values(q, s), mx_values(wq, ws), off.tolist())
    assert y.dtype == DT[out]
    close(y, ref, size, (K + 8) * 2.0 ** -23, "y")


def test_grouped_matmul_mx_one_slab():
    """The largest tiles at the shortest K, 18 million results.  The instruction cuts each of a group's 16 products,
    but the largest, at 2^-13 of that one: 15 * 2^-13 of the groups' largest products, which the bound of the test above
    leaves out (34 of these results are past it).  Bit by bit the tiles of every size agree."""
    R, K, N, E = 4200, 128, 4360, 3
    x, w = rand(R, K, seed=1), rand(E, N, K, seed=2, scale=K ** -0.5)
    x *= torch.exp2((torch.arange(K, device=DEV) // 32) % 7 - 3.0)
    w *= torch.exp2((torch.arange(N, device=DEV) % 5) - 2.0)[None, :, None]
    q, s = branch.quantize_mx(x)
    wq, ws = branch.quantize_mx(w)
    y = branch.grouped_matmul_mx(q, s, wq, ws, offsets_of("one has all", R, E), out_dtype=torch.bfloat16)
    for rows in (40, 600):  # 64-tiles and 128-tiles
        for i in range(0, R, rows):
            c = slice(i, i + rows)
            part = branch.grouped_matmul_mx(q[c], s[c], wq[1:2], ws[1:2], offsets_of("even", rows, 1), out_dtype=torch.bfloat16)
            assert torch.equal(part, y[c])
    xv, wv = torch.from_numpy(mx_values(q, s)).to(DEV), torch.from_numpy(mx_values(wq, ws)).to(DEV)[1]
    cut = torch.zeros(R, N, dtype=torch.float64, device=DEV)
    for g in range(0, K, 16):
        largest = torch.zeros_like(cut)
        for k in range(g, g + 16):
            largest = torch.maximum(largest, xv[:, k, None].abs() * wv[None, :, k].abs())
        cut += 15 * 2.0 ** -13 * largest
    ref = xv @ wv.T
    allowed = cut + (K + 8) * 2.0 ** -23 * (xv.abs() @ wv.abs().T) + 1.01 * HALF_ULP[torch.bfloat16] * ref.abs()
    assert bool(((y.double() - ref).abs() <= allowed).all())


def test_grouped_matmul_mx_special_scales():
    """A NaN block makes its row (or column) NaN and no other; the filling of a scale row is not read as values."""
    R, K, N, E = 20, 96, 40, 2
    x, w = rand(R, K, seed=1), rand(E, N, K, seed=2)
    off = offsets_of("even", R, E)
    clean = branch.grouped_matmul_mx(*branch.quantize_mx(x), *branch.quantize_mx(w), off, out_dtype=torch.bfloat16)
    x[3, 70] = float("inf")
    w[1, 5, 0] = float("nan")
    q, s = branch.quantize_mx(x)
    wq, ws = branch.quantize_mx(w)
    s.view(torch.uint8)[:, 3:] = 255
    ws.view(torch.uint8)[..., 3:] = 255
    y = branch.grouped_matmul_mx(q, s, wq, ws, off, out_dtype=torch.bfloat16)
    bad = torch.zeros(R, N, dtype=torch.bool, device=DEV)
    bad[3] = True
    bad[10:, 5] = True
    assert torch.equal(torch.isnan(y), bad) and torch.equal(y[~bad], clean[~bad])


# --------------------------------------------------------------------------
# Large tensors, streams, graphs, compile
# --------------------------------------------------------------------------

def test_offsets_past_32_bits():
    """Elements past 2^31: the last rows against the same rows alone."""
    D = 4096
    R = (1 << 31) // D + 300
    x = torch.empty(R, D, device=DEV, dtype=torch.bfloat16)
    x[-300:] = rand(300, D, seed=1, dtype=torch.bfloat16)
    x[:-300] = 0.5
    y = branch.rms_norm(x)
    assert torch.equal(y[-300:], branch.rms_norm(x[-300:]))
    del y
    z = branch.dropout(x, 0.25, (9, 9))
    first = (R - 300) * D
    f = O.dropout_factors(300 * D, 0.25, 9, 9, first=first)
    assert np.array_equal(to_np(z[-300:]).reshape(-1) != 0, (f != 0) & (to_np(x[-300:]).reshape(-1) != 0))
    del z
    q, s = branch.quantize_mx(x)
    qt, st = branch.quantize_mx(x[-300:])
    assert torch.equal(q[-300:].view(torch.uint8), qt.view(torch.uint8))
    assert torch.equal(s[-300:].view(torch.uint8), st.view(torch.uint8))
    w = rand(2, 64, D, seed=2, dtype=torch.bfloat16, scale=D ** -0.5)
    off = torch.tensor([R - 290, R], dtype=torch.int32, device=DEV)
    y = branch.grouped_matmul(x, w, off)
    want = branch.grouped_matmul(x[-300:], w, torch.tensor([10, 300], dtype=torch.int32, device=DEV))
    ref, size = O.grouped_matmul(to_np(x[-300:]), to_np(w), [10, 300])
    close(y[-300:], ref, size, (D + 8) * 2.0 ** -23, "last rows")
    close(want, ref, size, (D + 8) * 2.0 ** -23, "alone")
    ym = branch.grouped_matmul_mx(q, s, *branch.quantize_mx(w), off)
    wm = branch.grouped_matmul_mx(qt, st, *branch.quantize_mx(w), torch.tensor([10, 300], dtype=torch.int32, device=DEV))
    assert float((ym[-300:].float() - wm.float()).abs().max()) <= 2.0 ** -5  # a bf16 step of values below 8


def _step(x, res, w, wt, off, state, dy):
    y, h = branch.rms_norm(x, w, residual=res)
    z = branch.grouped_matmul(y, wt, off)
    z = branch.dropout(z, 0.2, state, residual=h)
    return (z, *torch.autograd.grad(z, (x, res, w, wt), dy))


def _step_inputs():
    R, D, E = 192, 128, 4
    bf = torch.bfloat16
    x, res = (rand(R, D, seed=i, dtype=bf).requires_grad_() for i in (1, 2))
    w, wt = rand(D, seed=3).requires_grad_(), rand(E, D, D, seed=4, dtype=bf, scale=D ** -0.5).requires_grad_()
    off = torch.tensor([50, 50, 120, 192], dtype=torch.int32, device=DEV)
    return x, res, w, wt, off, torch.tensor([5, 0], device=DEV), rand(R, D, seed=6, dtype=bf)


def test_another_stream():
    args = _step_inputs()
    want = _step(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _step(*args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_graph_replays_follow_offsets_and_state():
    x, res, w, wt, off, state, dy = _step_inputs()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(x, res, w, wt, off, state, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(x, res, w, wt, off, state, dy)
    for i, split in enumerate(([50, 50, 120, 192], [0, 0, 0, 192], [10, 20, 30, 100], [192, 192, 192, 192])):
        off.copy_(torch.tensor(split, dtype=torch.int32))
        state[1] = i
        with torch.no_grad():
            x.copy_(rand(*x.shape, seed=20 + i, dtype=x.dtype))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = _step(x, res, w, wt, off, state, dy)  # eager work between the replays
        assert all(torch.equal(a, b) for a, b in zip(want, got)), i


def test_compiled_equals_eager():
    args = _step_inputs()

    def f(x, res, w, wt, off, state):
        y, h = branch.rms_norm(x, w, residual=res)
        z = branch.grouped_matmul(y, wt, off)
        return branch.dropout(z, 0.2, state, residual=h) + branch.rms_norm(x)

    def grads(fn):
        z = fn(*args[:-1])
        return (z, *torch.autograd.grad(z, args[:4], args[-1]))

    want = grads(f)
    got = grads(torch.compile(f, fullgraph=True, backend="aot_eager"))
    assert all(torch.equal(a, b) for a, b in zip(want, got))

    @torch.no_grad()
    def g(x, res, w, wt, off):
        q, s, h = branch.rms_norm_mx(x, w, residual=res)
        return branch.grouped_matmul_mx(q, s, *branch.quantize_mx(wt), off), h

    assert all(torch.equal(a, b) for a, b in zip(g(*args[:5]), torch.compile(g, fullgraph=True, backend="aot_eager")(*args[:5])))


@pytest.mark.parametrize("grads", [(), ("x",), ("w",), ("res",), ("wt",), ("x", "w", "res", "wt")])
@pytest.mark.parametrize("state", [False, True])
def test_native_and_python_nodes_agree(monkeypatch, grads, state):
    """The C++ nodes and the Python nodes make the same launches: the same bits."""
    leaves = {"x": rand(40, 128, seed=1, dtype=torch.bfloat16), "w": rand(128, seed=2, dtype=torch.float16),
              "res": rand(40, 128, seed=3, dtype=torch.bfloat16), "wt": rand(3, 128, 128, seed=4, dtype=torch.bfloat16)}
    off = torch.tensor([7, 7, 40], device=DEV)
    dy = rand(40, 128, seed=5, dtype=torch.bfloat16).T.contiguous().T

    def step():
        for n, t in leaves.items():
            t.requires_grad_(n in grads)
        y, h = branch.rms_norm(leaves["x"], leaves["w"], residual=leaves["res"])
        y = branch.grouped_matmul(branch.rms_norm(y), leaves["wt"], off)
        y = branch.dropout(y, 0.3, torch.tensor([3, 4], device=DEV) if state else (3, 4), residual=h)
        return [y.detach(), *(torch.autograd.grad(y, [leaves[n] for n in grads], dy) if grads else ())]

    got, want = both(monkeypatch, step)
    same(got, want)


def test_calls_the_native_nodes_leave_alone():
    from mhc import _lib

    n = _lib.native()
    x, w = torch.ones(4, 8, device=DEV), torch.ones(2, 8, 8, device=DEV)
    off = torch.tensor([2, 4], dtype=torch.int32, device=DEV)
    assert n.rms_norm(x, None, None, 1e-6) is not None and n.grouped_matmul(x, w, off) is not None
    for out in (n.rms_norm(x, x, None, 1e-6), n.rms_norm(x.double(), None, None, 1e-6), n.rms_norm(x, None, x[:2], 1e-6),
                n.rms_norm(x, None, None, 1), n.dropout(x, None, 0.5, (-1, 0)), n.dropout(x, None, 1.5, (0, 0)),
                n.dropout(x, None, 0.5, (0, 1 << 64)), n.dropout(x, None, 0.5, off), n.dropout(x, None, 0.5, None),
                n.grouped_matmul(x, w[0], off), n.grouped_matmul(x, w, off[:1]), n.grouped_matmul(x, w, off.cpu()),
                n.grouped_matmul(x, w.half(), off), n.grouped_matmul(x.cpu(), w, off)):
        assert out is None


def test_wrong_devices_and_dtypes_are_refused():
    x, w = torch.zeros(4, 64, device=DEV), torch.zeros(2, 8, 64, device=DEV)
    off = torch.zeros(2, dtype=torch.int32, device=DEV)
    for error, call in (
        (RuntimeError, lambda: branch.grouped_matmul(x, w, off.cpu())),
        (RuntimeError, lambda: branch.rms_norm(x, torch.ones(64))),
        (TypeError, lambda: branch.grouped_matmul(x, w.to(torch.bfloat16), off)),
        (TypeError, lambda: branch.rms_norm(x.double())),
        (TypeError, lambda: branch.dropout(x.long(), 0.5, (0, 0))),
        (TypeError, lambda: branch.grouped_matmul_mx(x, off, w, off, off)),
        (TypeError, lambda: branch.grouped_matmul_mx(*branch.quantize_mx(x), *branch.quantize_mx(w), off, torch.float32)),
        (ValueError, lambda: branch.quantize_mx(x[:, :40])),
        (RuntimeError, lambda: branch.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))),
    ):
        with pytest.raises(error):
            call()


def test_saved_tensors_changed_in_place_are_noticed():
    x, w = rand(8, 64).requires_grad_(), torch.ones(64, device=DEV)
    h = x * 1
    y = branch.rms_norm(h, w)
    h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
