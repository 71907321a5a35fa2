"""``mhc.branch`` on the GPU, beside test_gpu_branch.py: calls and kernels that its cases do not reach."""

import pytest
import torch

from test_branch_cpu import OPS, SECOND_ORDER, _forward_mode_calls, forward_mode_is_refused, second_derivatives_raise
from helpers import to_np
from test_gpu_branch import DT, HALF_ULP, close, mx_values, offsets_of, rand
from test_gpu_native_nodes import both, same
from mhc import branch
from oracle import branch_oracle as O

pytestmark = pytest.mark.gpu

DEV = "cuda"


def against_oracle(y, dx, dw, x, w, dy, offsets):
    """The bounds of fp32 sums of as many terms, as in test_gpu_branch.py; rows of no expert are zeros."""
    (R, K), N = x.shape, w.shape[1]
    o = list(offsets)
    ref, size = O.grouped_matmul(to_np(x), to_np(w), o)
    rx, rw, sx, sw = O.grouped_matmul_backward(to_np(dy), to_np(x), to_np(w), o)
    close(y, ref, size, (K + 8) * 2.0 ** -23, "y")
    close(dx, rx, sx, (N + 8) * 2.0 ** -23, "dx")
    close(dw, rw, sw, (R + 8) * 2.0 ** -23, "dw")
    end = max(0, max(o)) if o else 0
    assert not y[end:].any() and not dx[end:].any()


@pytest.mark.parametrize("name", list(_forward_mode_calls("cpu")))
def test_forward_mode_is_refused(name):
    forward_mode_is_refused(name, DEV)


@pytest.mark.parametrize("wide", [[-2 ** 31 - 1, 3, 2 ** 32, 2 ** 40], [2 ** 32, 2 ** 32 + 5, 2 ** 63 - 1, 4], [-2 ** 32, -2 ** 40, 5, 2 ** 31]])
def test_int64_offsets_outside_32_bits_are_clamped(monkeypatch, wide):
    """Forward, both gradients and 8 bits, from the C++ nodes and from the Python ones."""
    R, K, N, E = 20, 64, 24, 4
    x, w, dy = rand(R, K, seed=1).requires_grad_(), rand(E, N, K, seed=2).requires_grad_(), rand(R, N, seed=3)
    wide = torch.tensor(wide, device=DEV)
    in_range = wide.clamp(0, R).int()

    def step(off):
        y = branch.grouped_matmul(x, w, off)
        with torch.no_grad():
            mx = branch.grouped_matmul_mx(*branch.quantize_mx(x), *branch.quantize_mx(w), off)
        return [y.detach(), *torch.autograd.grad(y, (x, w), dy), mx]

    want = step(in_range)
    for got in both(monkeypatch, lambda: step(wide)):
        same(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("R,K,N,E", [
    (60, 32, 40, 8), (60, 33, 40, 8),         # few rows: whole chunks, any alignment
    (600, 96, 72, 3), (600, 97, 71, 3),       # small tiles
    (3000, 256, 5000, 3), (3000, 5000, 264, 3),  # the largest tiles, with quarters (of y, of dx)
])
def test_offsets_that_run_backwards_against_the_oracle(R, K, N, E, dtype):
    """Every row and both gradients: the rows belong to the running maximum's experts."""
    dt = DT[dtype]
    x, w = rand(R, K, seed=1, dtype=dt).requires_grad_(), rand(E, N, K, seed=2, dtype=dt, scale=K ** -0.5).requires_grad_()
    dy = rand(R, N, seed=3, dtype=dt)
    o = [R // 3, R // 6, -R, R * 5 // 6, R // 2, R * 2 // 3, R - 7, R - 9][:E - 1] + [R - 4]
    off = torch.tensor(o, dtype=torch.int32, device=DEV)
    y = branch.grouped_matmul(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    against_oracle(y, dx, dw, x, w, dy, o)


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_compiled_dropout_from_pairs_of_ints(backend):
    """The same mask as eager, forward and backward, also once the ints have become symbols and past 2^63."""
    x, res, dy = rand(64, 96, seed=1).requires_grad_(), rand(64, 96, seed=2).requires_grad_(), rand(64, 96, seed=3)

    def f(x, res, rng):
        return branch.dropout(x, 0.3, rng, residual=res)

    torch._dynamo.reset()
    compiled = torch.compile(f, fullgraph=True, backend=backend)
    for pair in [(7, 0), (7, 1), (8, 2), (2 ** 63 + 5, 3), (2 ** 64 - 1, 2 ** 64 - 2), (2 ** 31, 2 ** 32)]:
        want, got = f(x, res, pair), compiled(x, res, pair)
        assert torch.equal(got, want)
        for a, b in zip(torch.autograd.grad(got, (x, res), dy), torch.autograd.grad(want, (x, res), dy)):
            assert torch.equal(a, b)
    torch._dynamo.reset()


def test_more_rows_than_a_launch_has_workgroups():
    """Workgroups of 1024 threads come to 2^32 work items at 2^22 rows: a launch holds fewer and loops."""
    D, R = 15392, (1 << 22) + 5
    torch.cuda.empty_cache()
    need = R * D * 3 + R * 4 * 121 + (4 << 30)
    if torch.cuda.mem_get_info()[0] < need:
        pytest.skip(f"needs {need >> 30} GiB of GPU memory")
    x = torch.empty(R, D, device=DEV, dtype=torch.bfloat16).fill_(0.5)
    x[-9:] = rand(9, D, seed=1, dtype=torch.bfloat16)
    x[:3] = rand(3, D, seed=2, dtype=torch.bfloat16)
    q, s = (t.view(torch.uint8) for t in branch.rms_norm_mx(x))
    for rows in (slice(0, 4), slice(R // 2, R // 2 + 2), slice(R - 9, R)):
        qa, sa = (t.view(torch.uint8) for t in branch.rms_norm_mx(x[rows].clone()))
        assert torch.equal(q[rows], qa) and torch.equal(s[rows], sa)
    del x, q, s
    torch.cuda.empty_cache()


@pytest.mark.parametrize("op,need,dy_grad,graph", SECOND_ORDER)
def test_second_derivatives_raise(monkeypatch, op, need, dy_grad, graph):
    both(monkeypatch, lambda: second_derivatives_raise(op, need, dy_grad, graph, DEV))


# --------------------------------------------------------------------------
# RMS norm of more than 64 rows: partial weight gradients, rows in a loop
# --------------------------------------------------------------------------
# Bounds.  A sum over a row adds at most 16 terms a lane, six levels in a wave and 16 waves: 38 roundings of 2^-24 of
# the terms' magnitudes, and half of that in rstd; with the roundings around it y is within 24 * 2^-24 of itself.  dx has
# rstd three times and two sums: below 128 * 2^-24 of its terms.  The weight gradient adds few rows in fp32 and
# the rest in fp64: 32 * 2^-24.
Y_TOL, DX_TOL, DW_TOL = 2.0 ** -19, 2.0 ** -17, 2.0 ** -19


def check_norm(x, w, res, dy, dh):
    leaves = [t for t in (x, w, res) if t is not None]
    out = branch.rms_norm(x, w, residual=res)
    y, h = (out, x) if res is None else out
    if res is not None:
        assert torch.equal(h, x + res)
    grads = torch.autograd.grad((y,) if res is None else (y, h), leaves, (dy,) if res is None else (dy, dh))
    if res is not None:
        assert torch.equal(grads[0], grads[2])
    ref, _ = O.rms_norm(to_np(h), to_np(w))
    rx, rw, sx, sw = O.rms_norm_backward(to_np(dy), to_np(h), None if res is None else to_np(dh), to_np(w))
    close(y, ref, ref, Y_TOL, "y")
    close(grads[0], rx, sx, DX_TOL, "dx")
    close(grads[1], rw, sw, DW_TOL, "dw")


# a row in a wave of one, two and four vectors a lane, in workgroups of every width, below one vector
NORM_WIDTHS = {
    "16": [3, 7, 504, 513, 1024, 1030, 1500, 2048, 2050, 4096, 4099, 7168, 8191, 16383, 16384],
    "32": [1, 3, 256, 258, 512, 750, 1022, 1024, 1026, 4096, 8190, 8192, 8193, 12290, 16383, 16384],
}


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype,D", [(t, D) for t in DT for D in NORM_WIDTHS["32" if t == "fp32" else "16"]])
def test_rms_norm_of_many_rows(D, dtype, residual):
    R, dt = (2101 if D <= 2048 else 1100 if D <= 4100 else 1027 if D < 8193 else 517), DT[dtype]
    x, dy = rand(R, D, seed=1, dtype=dt, scale=1.5).requires_grad_(), rand(R, D, seed=4, dtype=dt)
    w = rand(D, seed=2).add_(1.0).requires_grad_()
    res = rand(R, D, seed=3, dtype=dt).requires_grad_() if residual else None
    check_norm(x, w, res, dy, rand(R, D, seed=5, dtype=dt) if residual else None)


@pytest.mark.parametrize("dtype,D", [("bf16", 512), ("fp16", 2048), ("bf16", 4096), ("fp32", 1024), ("fp32", 8192), ("fp32", 12288)])
def test_rms_norm_of_many_unaligned_rows(dtype, D):
    """Rows of whole vectors, an element past a 16-byte boundary."""
    R, dt = 300, DT[dtype]
    off = lambda seed: rand(R * D + 1, seed=seed, dtype=dt)[1:].view(R, D)  # noqa: E731
    x, res, dy, dh = off(1).requires_grad_(), off(3).requires_grad_(), off(4), off(5)
    check_norm(x, rand(D, seed=2).add_(1.0).requires_grad_(), res, dy, dh)


@pytest.mark.parametrize("R", [65, 1100])
@pytest.mark.parametrize("dtype,D", [("bf16", 512), ("bf16", 1500), ("fp16", 2050), ("bf16", 4096), ("fp32", 1000), ("fp32", 9001)])
def test_rms_norm_of_many_rows_each_gradient_alone(dtype, D, R):
    """dx without dw and dw without dx: the bits that both together have."""
    dt = DT[dtype]
    x, dy, w = rand(R, D, seed=1, dtype=dt), rand(R, D, seed=4, dtype=dt), rand(D, seed=2)
    lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(branch.rms_norm(lx, lw), (lx, lw), dy)
    assert torch.equal(torch.autograd.grad(branch.rms_norm(lx, w), lx, dy)[0], dx)
    assert torch.equal(torch.autograd.grad(branch.rms_norm(x, lw), lw, dy)[0], dw)


# --------------------------------------------------------------------------
# Expert products: few rows an expert, unaligned tiles
# --------------------------------------------------------------------------

FEW_SPLITS = ["even", "one has all", "empty ends", "single rows", "none"]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("split", FEW_SPLITS)
@pytest.mark.parametrize("R,K,N,E", [(100, 1001, 37, 16), (100, 1500, 65, 16), (100, 1504, 72, 16), (128, 200, 130, 16),
                                     (500, 260, 34, 70)])
def test_grouped_matmul_of_few_rows(R, K, N, E, split, dtype):
    """At most eight rows an expert on average: several tiles of one expert, experts without any, rows of none; rows
    of whole chunks, and of any alignment over several units of 128 bytes."""
    dt = DT[dtype]
    x = rand(R, K, seed=1, dtype=dt).requires_grad_()
    w = rand(E, N, K, seed=2, dtype=dt, scale=K ** -0.5).requires_grad_()
    dy = rand(R, N, seed=3, dtype=dt)
    off = offsets_of(split, R, E)
    y = branch.grouped_matmul(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    against_oracle(y, dx, dw, x, w, dy, off.tolist())


def test_grouped_matmul_of_few_rows_does_not_leak():
    """NaN and infinity in one expert's rows and weights and in the rows of none stay there."""
    R, N, E = 100, 37, 16
    off = torch.tensor([5, 5, 31, 40] + [40 + 4 * i for i in range(11)] + [90], dtype=torch.int32, device=DEV)
    for K in (1001, 1500, 1504):
        for dt in DT.values():
            x, w = rand(R, K, seed=1, dtype=dt), rand(E, N, K, seed=2, dtype=dt)
            want = branch.grouped_matmul(x, w, off)
            x[5:31], x[90:] = float("nan"), float("inf")
            w[1:3] = float("inf")
            got = branch.grouped_matmul(x, w, off)
            assert torch.equal(got[:5], want[:5]) and torch.equal(got[31:90], want[31:90])
            assert torch.isnan(got[5:31]).all() and not got[90:].any()


@pytest.mark.parametrize("out", ["bf16", "fp16"])
@pytest.mark.parametrize("split", FEW_SPLITS)
@pytest.mark.parametrize("K,N", [(2048, 40), (2080, 33), (4128, 257), (4224, 100)])
def test_grouped_matmul_mx_of_few_rows(K, N, split, out):
    """8 bits: the last unit and the last scales of a row partial, odd widths, NaN in the scales' filling.  The bound is
    the instruction's: of 16 products all but the largest are cut at 2^-13 of that one."""
    R, E = 100, 16
    x, w = rand(R, K, seed=1), rand(E, N, K, seed=2, scale=K ** -0.5)
    x *= torch.exp2((torch.arange(K, device=DEV) // 32) % 7 - 3.0)
    w *= torch.exp2((torch.arange(N, device=DEV) % 5) - 2.0)[None, :, None]
    (q, s), (wq, ws) = branch.quantize_mx(x), branch.quantize_mx(w)
    xv, wv = (torch.from_numpy(mx_values(*t)).to(DEV) for t in ((q, s), (wq, ws)))
    for t in (s, ws):
        t.view(torch.uint8)[..., K // 32:] = 255
    off = offsets_of(split, R, E)
    y = branch.grouped_matmul_mx(q, s, wq, ws, off, out_dtype=DT[out])
    ref, allowed = torch.zeros(R, N, dtype=torch.float64, device=DEV), torch.zeros(R, N, dtype=torch.float64, device=DEV)
    for e, lo, hi in O.groups(off.tolist(), R):
        for r in range(lo, hi):
            terms = xv[r] * wv[e]
            ref[r] = terms.sum(1)
            cut = 15 * 2.0 ** -13 * terms.abs().view(N, -1, 16).amax(2).sum(1)
            allowed[r] = cut + (K + 8) * 2.0 ** -23 * terms.abs().sum(1)
    allowed += 1.01 * HALF_ULP[DT[out]] * ref.abs() + (2.0 ** -25 if out == "fp16" else 0.0)
    assert y.dtype == DT[out]
    assert bool(((y.double() - ref).abs() <= allowed).all())
    end = max(off.tolist())
    assert not y[end:].any()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("R,K,N", [(2900, 129, 2801), (2900, 2801, 129), (2900, 2801, 136), (300, 2801, 2901), (301, 2800, 2901)])
def test_grouped_matmul_unaligned_large_tiles(R, K, N, dtype):
    """Unaligned rows and enough tiles of 128 x 128 (22 x 24, 66 x 23 of the weight gradient) for two a CU: y, dx and dw
    each, one operand of whole chunks beside an odd one, an expert without rows, rows of none."""
    dt, E = DT[dtype], 3
    x = rand(R, K, seed=1, dtype=dt).requires_grad_()
    w = rand(E, N, K, seed=2, dtype=dt, scale=K ** -0.5).requires_grad_()
    dy = rand(R, N, seed=3, dtype=dt)
    o = [R * 2 // 5, R * 2 // 5, R - 13]
    y = branch.grouped_matmul(x, w, torch.tensor(o, dtype=torch.int32, device=DEV))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    against_oracle(y, dx, dw, x, w, dy, o)


# --------------------------------------------------------------------------
# Registrations, uninitialised memory
# --------------------------------------------------------------------------

def _registered_ops():
    """name -> arguments of each op; several of one op side by side."""
    bf = torch.bfloat16
    x, res, w, dy = (rand(6, 64, seed=i, dtype=bf) for i in (1, 2, 3, 4))
    w, off, wt = rand(64, seed=3), torch.tensor([2, 2, 5], dtype=torch.int32, device=DEV), rand(3, 16, 64, seed=5, dtype=bf)
    rstd, state = rand(6, seed=6).abs(), torch.tensor([3, 4], device=DEV)
    (q, s), (wq, ws) = branch.quantize_mx(x), branch.quantize_mx(wt)
    rg = lambda t: t.clone().requires_grad_()  # noqa: E731
    return [
        ("norm", (rg(x.float()), rg(w), 1e-6)), ("norm", (x, None, 1e-6)),
        ("add_norm", (rg(x.float()), rg(w), rg(res.float()), 1e-6)),
        ("norm_backward", (dy, x, res, w, rstd, True)), ("norm_backward", (dy, x, None, None, rstd, False)),
        ("norm_mx", (x, w, res, 1e-6)), ("norm_mx", (x, None, None, 1e-6)), ("quantize_mx", (x,)),
        ("grouped_matmul", (rg(x.float()), rg(wt.float()), off)),
        ("grouped_matmul_backward_input", (rand(6, 16, seed=7, dtype=bf), wt, off)),
        ("grouped_matmul_backward_weight", (rand(6, 16, seed=7, dtype=bf), x, off)),
        ("grouped_matmul_mx", (q, s, wq, ws, off, torch.float16)),
        ("dropout", (rg(x.float()), rg(res.float()), 0.3, state, [])), ("dropout", (rg(x.float()), None, 0.3, None, [1, 2, 3, 4])),
    ]


@pytest.mark.parametrize("i", range(14))
def test_opcheck(i):
    cases = _registered_ops()
    assert len(cases) == 14 and {n for n, _ in cases} == OPS
    name, args = cases[i]
    checks = ("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")
    # the schema check compares inputs before and after with products, which torch does not have in 8 bits
    torch.library.opcheck(getattr(torch.ops.mhc_branch, name).default, args, test_utils=checks[name == "grouped_matmul_mx":])


def test_outputs_and_workspaces_are_written_before_they_are_read(monkeypatch):
    """With every new tensor's bytes set to 0xFF (NaN in each type) the results are the same."""
    from mhc import _lib

    def run():
        out = []
        for R, D, dt in ((3, 7, torch.float32), (70, 500, torch.bfloat16), (200, 2050, torch.float16), (600, 96, torch.float32)):
            x, res, dy = (rand(R, D, seed=i, dtype=dt).requires_grad_() for i in (1, 2, 3))
            w = rand(D, seed=4).requires_grad_()
            y, h = branch.rms_norm(x, w, residual=res)
            out += [y, h, *torch.autograd.grad((y, h), (x, res, w), (dy, dy))]
            y = branch.dropout(x, 0.4, torch.tensor([1, 2], device=DEV), residual=res)
            out += [y, *torch.autograd.grad(y, (x, res), dy)]
            E, N = 5, 40
            wt, g = rand(E, N, D, seed=5, dtype=dt).requires_grad_(), rand(R, N, seed=6, dtype=dt)
            off = torch.tensor([R // 3, R // 3, R // 2, R // 2, R - 2], dtype=torch.int32, device=DEV)
            y = branch.grouped_matmul(x, wt, off)
            out += [y, *torch.autograd.grad(y, (x, wt), g)]
        with torch.no_grad():
            for R, D, E in ((5, 32, 2), (60, 2080, 9), (300, 416, 3)):
                x, w = rand(R, D, seed=1, dtype=torch.bfloat16), rand(E, 24, D, seed=2, dtype=torch.bfloat16)
                q, s, h = branch.rms_norm_mx(x, residual=x)
                wq, ws = branch.quantize_mx(w)
                off = torch.tensor([R // 3] * (E - 1) + [R - 2], dtype=torch.int32, device=DEV)
                out += [q, s, h, wq, ws, branch.grouped_matmul_mx(q, s, wq, ws, off)]
        return [t.detach().contiguous().view(torch.uint8) for t in out]

    class Off:
        def __getattr__(self, name):
            return lambda *a: None

    monkeypatch.setattr(_lib, "native", lambda: Off())
    want = run()
    for owner, name in ((torch, "empty"), (torch, "empty_like"), (torch.Tensor, "new_empty")):
        def poisoned(*a, _make=getattr(owner, name), **k):
            t = _make(*a, **k)
            if t.is_cuda and t.numel() and t.is_contiguous():
                t.view(torch.uint8).fill_(0xFF)
            return t
        monkeypatch.setattr(owner, name, poisoned)
    got = run()
    monkeypatch.undo()
    same(got, want)


def test_quantize_mx_of_more_elements_than_a_launch_has_work_items():
    D, R = 8192, (1 << 22) + 5  # eight elements a work item
    torch.cuda.empty_cache()
    need = R * D * 3 + R * 256 + (4 << 30)
    if torch.cuda.mem_get_info()[0] < need:
        pytest.skip(f"needs {need >> 30} GiB of GPU memory")
    x = torch.empty(R, D, device=DEV, dtype=torch.bfloat16).fill_(0.5)
    x[-9:] = rand(9, D, seed=1, dtype=torch.bfloat16)
    x[:3] = rand(3, D, seed=2, dtype=torch.bfloat16)
    q, s = (t.view(torch.uint8) for t in branch.quantize_mx(x))
    for rows in (slice(0, 4), slice(R // 2, R // 2 + 2), slice(R - 9, R)):
        qa, sa = (t.view(torch.uint8) for t in branch.quantize_mx(x[rows].clone()))
        assert torch.equal(q[rows], qa) and torch.equal(s[rows], sa)
    del x, q, s
    torch.cuda.empty_cache()
