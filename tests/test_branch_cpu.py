"""``mhc.branch`` without a GPU: the oracle's pins, refusals, the C ABI's host-side checks, and the
torch.library fakes."""

import numpy as np
import pytest
import torch

from mhc import _branch, branch
from oracle import branch_oracle as O

BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("ctr,key,out", [
    # known answers published with the generator
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_oracle_philox_known_answers(ctr, key, out):
    got = O.philox([ctr[0]], [ctr[1]], ctr[2] | ctr[3] << 32, key[0] | key[1] << 32)
    assert tuple(int(w[0]) for w in got) == out


def test_oracle_e4m3_and_scales():
    v = torch.tensor([0.0, 448.0, 440.0, 1.0, 1.0625, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, 0.3, -27.0, 2.0 ** -6])
    assert np.array_equal(O.e4m3_round(v.numpy()), v.to(torch.float8_e4m3fn).double().numpy())
    assert O.mx_exponent([448.0, 448.0001, 224.0, 0.0, 1e-45, 1.0, 1.75, 1.7500001]).tolist() == [
        0, 1, -1, -127, -127, -8, -8, -7]
    for k, top in enumerate((448.0, 3.0, 1e30, 2.0 ** -100)):
        e = float(O.mx_exponent(top))
        assert top / 2 ** e <= 448 < top / 2 ** (e - 1), k


def test_oracle_gradients_against_differences():
    r = np.random.default_rng(0)
    h, dy, dh, w = r.standard_normal((3, 5)), r.standard_normal((3, 5)), r.standard_normal((3, 5)), r.standard_normal(5)
    dx, dw, _, _ = O.rms_norm_backward(dy, h, dh, w)
    loss = lambda h, w: (O.rms_norm(h, w)[0] * dy).sum() + (h * dh).sum()  # noqa: E731
    v, u, t = r.standard_normal(h.shape), r.standard_normal(5), 1e-6
    assert abs((loss(h + t * v, w) - loss(h - t * v, w)) / (2 * t) - (dx * v).sum()) < 1e-8
    assert abs((loss(h, w + t * u) - loss(h, w - t * u)) / (2 * t) - (dw * u).sum()) < 1e-8
    x, wt, g = r.standard_normal((7, 4)), r.standard_normal((3, 6, 4)), r.standard_normal((7, 6))
    off = [2, 2, 6]
    dx, dw, _, _ = O.grouped_matmul_backward(g, x, wt, off)
    vx, vw = r.standard_normal(x.shape), r.standard_normal(wt.shape)
    f = lambda x, w: (O.grouped_matmul(x, w, off)[0] * g).sum()  # noqa: E731
    assert abs((f(x + vx, wt) - f(x - vx, wt)) / 2 - (dx * vx).sum()) < 1e-10
    assert abs((f(x, wt + vw) - f(x, wt - vw)) / 2 - (dw * vw).sum()) < 1e-10
    assert not dw[1].any() and not dx[6].any()


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 32)
    off = torch.tensor([2, 4], dtype=torch.int32)
    for call in (lambda: branch.rms_norm(x), lambda: branch.rms_norm_mx(x), lambda: branch.quantize_mx(x),
                 lambda: branch.dropout(x, 0.1, (1, 2)), lambda: branch.grouped_matmul(x, torch.randn(2, 8, 32), off)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


def _refusals():
    x = torch.zeros(4, 64)
    off = torch.zeros(2, dtype=torch.int32)
    w = torch.zeros(2, 8, 64)
    q, s = torch.zeros(4, 64).to(_branch.F8), torch.zeros(4, 4, dtype=torch.uint8).view(_branch.E8)
    wq, ws = torch.zeros(2, 8, 64).to(_branch.F8), torch.zeros(2, 8, 4, dtype=torch.uint8).view(_branch.E8)
    mx = lambda **k: branch.grouped_matmul_mx(*{**dict(q=q, s=s, wq=wq, ws=ws, off=off), **k}.values())  # noqa: E731
    return [
        ("weight width", AssertionError, lambda: branch.rms_norm(x, torch.ones(63))),
        ("scalar", AssertionError, lambda: branch.rms_norm(torch.zeros(()))),
        ("row too wide", ValueError, lambda: branch.rms_norm(torch.zeros(1, 16385))),
        ("residual shape", AssertionError, lambda: branch.rms_norm(x, residual=torch.zeros(64))),
        ("residual dtype", TypeError, lambda: branch.rms_norm(x, residual=x.to(BF))),
        ("not whole blocks", ValueError, lambda: _branch._mx_outputs(torch.zeros(4, 48))),
        ("p", ValueError, lambda: branch.dropout(x, 1.5, (0, 0))),
        ("p nan", ValueError, lambda: branch.dropout(x, float("nan"), (0, 0))),
        ("seed range", ValueError, lambda: branch.dropout(x, 0.5, (-1, 0))),
        ("seed type", TypeError, lambda: branch.dropout(x, 0.5, 7)),
        ("rng shape", AssertionError, lambda: branch.dropout(x, 0.5, torch.zeros(3, dtype=torch.int64))),
        ("dropout residual", AssertionError, lambda: branch.dropout(x, 0.5, (0, 0), residual=x[:2])),
        ("weight dims", AssertionError, lambda: branch.grouped_matmul(x, w[0], off)),
        ("in width", AssertionError, lambda: branch.grouped_matmul(x[:, :32], w, off)),
        ("rows dims", AssertionError, lambda: branch.grouped_matmul(x[None], w, off)),
        ("offsets count", AssertionError, lambda: _branch._offsets(off, 3)),
        ("offsets dtype", TypeError, lambda: _branch._offsets(off.float(), 2)),
        ("8-bit types", TypeError, lambda: mx(q=x)),
        ("grad needed", RuntimeError, lambda: branch.quantize_mx(x.clone().requires_grad_())),
        ("grad needed", RuntimeError, lambda: branch.rms_norm_mx(x, torch.ones(64, requires_grad=True))),
    ]


@pytest.mark.parametrize("i", range(20))
def test_refusals(i):
    cases = _refusals()
    assert len(cases) == 20
    name, error, call = cases[i]
    with pytest.raises(error):
        call()


def test_abi_refusals_before_any_device_work():
    from mhc import _lib

    lib = _lib.load()
    assert lib.mhc_rms_norm_forward(None, None, 1, None, None, None, None, 4, 64, 1e-6, None) == 1
    assert lib.mhc_rms_norm_forward(None, None, 1, None, None, None, None, 0, 64, 1e-6, None) == 0
    assert lib.mhc_rms_norm_forward(16, 16, 1, None, 16, None, None, 4, 64, 1e-6, None) == 1  # residual without h
    assert lib.mhc_rms_norm_forward(16, None, 1, None, 16, None, None, 4, 16385, 1e-6, None) == 1
    assert b"16384" in lib.mhc_last_error()
    assert lib.mhc_rms_norm_forward(16, None, 9, None, 16, None, None, 4, 64, 1e-6, None) == 2
    assert lib.mhc_rms_norm_mx_forward(16, None, 1, None, 16, 16, None, 4, 48, 1e-6, None) == 1
    assert lib.mhc_rms_norm_mx_forward(24, None, 1, None, 16, 16, None, 4, 64, 1e-6, None) == 1  # alignment
    assert lib.mhc_rms_norm_backward(16, 16, None, 1, None, 16, 16, 16, 100, 64, None, 0, None) == 3
    need = lib.mhc_rms_norm_backward_workspace_bytes(100, 64)
    assert need == 50 * 64 * 4 and lib.mhc_rms_norm_backward_workspace_bytes(64, 64) == 0
    assert lib.mhc_rms_norm_backward(16, 16, None, 1, None, 16, 16, 16, 100, 64, 256, need - 1, None) == 3
    assert lib.mhc_quantize_mx(16, 1, 16, 16, 4, 33, None) == 1
    assert lib.mhc_dropout(None, None, 1, None, -1, 0.1, 0, 0, None, None, None) == 1
    assert lib.mhc_dropout(None, None, 1, None, 8, 0.1, 0, 0, None, None, None) == 1
    assert lib.mhc_dropout(16, None, 1, 16, 8, 1.1, 0, 0, None, None, None) == 1
    assert lib.mhc_dropout(None, None, 1, None, 0, 0.1, 0, 0, None, None, None) == 0
    for name in ("forward", "backward_input", "backward_weight"):
        fn = getattr(lib, f"mhc_grouped_matmul_{name}")
        assert fn(None, None, 1, None, None, 4, 8, 8, 2, None) == 1
        assert fn(16, 16, 1, 16, 16, 4, -8, 8, 2, None) == 1
        assert fn(16, 16, 1, 16, 16, 1 << 31, 8, 8, 2, None) == 1
        assert fn(16, 16, 1, 16, 16, 4, 8, 8, 4097, None) == 1
        assert fn(None, None, 1, None, None, 0, 0, 8, 2, None) == 0
        assert fn(16, 16, 5, 16, 16, 4, 8, 8, 2, None) == 2
    assert lib.mhc_grouped_matmul_mx(16, 16, 16, 16, 16, 16, 1, 4, 48, 8, 2, None) == 1
    assert lib.mhc_grouped_matmul_mx(24, 16, 16, 16, 16, 16, 1, 4, 64, 8, 2, None) == 1
    assert b"aligned" in lib.mhc_last_error()
    assert lib.mhc_grouped_matmul_mx(16, 16, 16, 16, 16, 16, 0, 4, 64, 8, 2, None) == 2  # no fp32 results


OPS = {"norm", "add_norm", "norm_backward", "norm_mx", "quantize_mx", "grouped_matmul",
       "grouped_matmul_backward_input", "grouped_matmul_backward_weight", "grouped_matmul_mx", "dropout"}


def test_every_launcher_is_registered():
    assert {n for n in dir(torch.ops.mhc_branch) if not n.startswith("_") and n != "name"} == OPS
    for n in OPS:
        assert torch._C._dispatch_has_kernel_for_dispatch_key(f"mhc_branch::{n}", "CUDA"), n
        assert not torch._C._dispatch_has_kernel_for_dispatch_key(f"mhc_branch::{n}", "CPU"), n


def test_fakes_and_traced_gradients():
    """Meta tensors through the traced functions: every gradient has its input's shape and dtype."""
    from mhc import _branch_library as L

    e = lambda *s, dt=BF: torch.empty(*s, device="meta", dtype=dt).requires_grad_(dt in (BF, F32))  # noqa: E731
    x, res, w = e(6, 64), e(6, 64), e(64, dt=F32)
    y, h = L.rms_norm(x, w, res, 1e-6)
    assert y.shape == h.shape == x.shape and y.dtype == h.dtype == BF
    g = torch.autograd.grad((y.sum() + h.sum()), (x, w, res))
    assert [(t.shape, t.dtype) for t in g] == [(t.shape, t.dtype) for t in (x, w, res)]
    y = L.rms_norm(x, None, None, 1e-6)
    assert torch.autograd.grad(y.sum(), x)[0].shape == x.shape
    q, s, h = L.rms_norm_mx(x.detach(), w.detach(), res.detach(), 1e-6)
    assert (q.dtype, s.dtype, s.shape, h.dtype) == (_branch.F8, _branch.E8, (6, 4), BF)
    assert L.quantize_mx(e(3, 5, 160).detach())[1].shape == (3, 5, 8)
    wt, off = e(3, 16, 64), e(3, dt=torch.int32)
    y = L.grouped_matmul(x, wt, off)
    assert y.shape == (6, 16) and y.dtype == BF
    g = torch.autograd.grad(y.sum(), (x, wt))
    assert [(t.shape, t.dtype) for t in g] == [(t.shape, t.dtype) for t in (x, wt)]
    wq, ws = L.quantize_mx(wt.detach())
    assert L.grouped_matmul_mx(q, s, wq, ws, off, torch.float16).dtype == torch.float16
    y = L.dropout(x, 0.1, e(2, dt=torch.int64), res)
    g = torch.autograd.grad(y.sum(), (x, res))
    assert [(t.shape, t.dtype) for t in g] == [(t.shape, t.dtype) for t in (x, res)]


def _forward_mode_calls(device):
    """name -> call on tensors of which f makes one dual (forward-mode AD)."""
    x, w, off = torch.ones(4, 64, device=device), torch.ones(64, device=device), torch.tensor([2, 4], device=device)
    wt = torch.ones(2, 64, 64, device=device)
    q, s = x.to(_branch.F8), torch.full((4, 4), 127, dtype=torch.uint8, device=device).view(_branch.E8)
    wq, ws = wt.to(_branch.F8), torch.full((2, 64, 4), 127, dtype=torch.uint8, device=device).view(_branch.E8)
    return {
        "norm": lambda f: branch.rms_norm(f(x)),
        "norm weight": lambda f: branch.rms_norm(x, f(w)),
        "norm residual": lambda f: branch.rms_norm(x, w, residual=f(x)),
        "norm mx": lambda f: branch.rms_norm_mx(f(x)),
        "norm mx weight": lambda f: branch.rms_norm_mx(x, f(w)),
        "quantize": lambda f: branch.quantize_mx(f(x)),
        "dropout": lambda f: branch.dropout(f(x), 0.5, (1, 2)),
        "grouped": lambda f: branch.grouped_matmul(f(x), wt, off),
        "grouped weight": lambda f: branch.grouped_matmul(x, f(wt), off),
        "grouped mx": lambda f: branch.grouped_matmul_mx(f(q), s, wq, ws, off),
        "grouped mx weight": lambda f: branch.grouped_matmul_mx(q, s, f(wq), ws, off),
    }


def forward_mode_is_refused(name, device):
    """No operator has a forward-mode derivative: a dual tensor is refused, not computed without its tangent.
    Without one the same call runs, with gradients off and with them on."""
    from torch.autograd.forward_ad import dual_level, make_dual

    call = _forward_mode_calls(device)[name]
    for mode in (torch.no_grad, torch.enable_grad):
        with mode(), dual_level():
            call(lambda t: t)
            with pytest.raises(NotImplementedError):
                call(lambda t: make_dual(t, t.clone()))


@pytest.mark.parametrize("name", list(_forward_mode_calls("cpu")))
def test_forward_mode_is_refused(monkeypatch, name):
    """Stand-in launchers that, as the real ones do, read the values and return new tensors."""
    new = torch.empty_like
    monkeypatch.setattr(_branch, "rms_norm_forward", lambda x, w, res, eps, want_rstd=True: (
        new(x), None if res is None else new(x), new(x) if want_rstd else None))
    monkeypatch.setattr(_branch, "rms_norm_mx", lambda x, w, res, eps: (new(x), new(x), None))
    monkeypatch.setattr(_branch, "quantize_mx", lambda x: (new(x), new(x)))
    monkeypatch.setattr(_branch, "dropout", lambda x, p, rng, res, want_used: (new(x), None))
    monkeypatch.setattr(_branch, "grouped_matmul_forward", lambda x, w, off: new(x))
    monkeypatch.setattr(_branch, "grouped_matmul_mx", lambda q, *rest: new(q))
    forward_mode_is_refused(name, "cpu")


def test_8_bit_products_refuse_operands_that_need_gradients():
    q, s = torch.zeros(4, 64).to(_branch.F8), torch.zeros(4, 4, dtype=torch.uint8).view(_branch.E8)
    wq, ws = torch.zeros(2, 8, 64).to(_branch.F8), torch.zeros(2, 8, 4, dtype=torch.uint8).view(_branch.E8)
    with pytest.raises(RuntimeError, match="no backward"):
        branch.grouped_matmul_mx(q.requires_grad_(), s, wq, ws, torch.zeros(2, dtype=torch.int32))


def test_wide_offsets_are_narrowed_to_the_nearest():
    """int64 offsets outside 32 bits stay out of range, on the side on which they were."""
    wide = torch.tensor([-2 ** 40, -2 ** 31 - 1, -2 ** 31, 7, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 3, 2 ** 63 - 1])
    got = _branch._offsets(wide, 9)
    assert got.dtype == torch.int32
    assert got.tolist() == [-2 ** 31] * 3 + [7] + [2 ** 31 - 1] * 5


@pytest.mark.parametrize("offsets,want", [
    ([2, 2, 6], [(0, 0, 2), (1, 2, 2), (2, 2, 6)]),
    ([5, 3, 8], [(0, 0, 5), (1, 5, 5), (2, 5, 8)]),
    ([-4, 20, 1], [(0, 0, 0), (1, 0, 8), (2, 8, 8)]),
    ([6, -1, 2, 7], [(0, 0, 6), (1, 6, 6), (2, 6, 6), (3, 6, 7)]),
])
def test_oracle_offsets_count_as_their_running_maximum(offsets, want):
    assert O.groups(offsets, 8) == want


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_traced_dropout_takes_every_pair_of_ints(backend):
    """Traced ints become symbols once they change between calls; the pairs still reach the op whole, and its
    backward draws from what the forward drew from.  A stand-in op writes down what it got."""
    seen = []

    def op(x, residual, p, rng, words):
        u64 = (1 << 64) - 1
        if rng is None:
            rng = torch.tensor([v - (1 << 64) if v >> 63 else v for v in (words[0] | words[1] << 32, words[2] | words[3] << 32)])
        seen.append(tuple(v & u64 for v in rng.tolist()))
        return x.clone(), rng.clone()

    torch._dynamo.reset()
    with torch.library._scoped_library("mhc_branch", "IMPL") as lib:
        lib.impl("dropout", op, "CPU")
        f = torch.compile(lambda x, rng: branch.dropout(x, 0.5, rng), fullgraph=True, backend=backend)
        for pair in [(7, 0), (7, 1), (8, 2), (2 ** 63 + 5, 3), (9, 2 ** 64 - 1), (2 ** 64 - 1, 2 ** 63), (2 ** 31, 2 ** 32), (0, 0)]:
            x = torch.ones(8, requires_grad=True)
            f(x, pair).sum().backward()
            assert seen == [pair, pair]
            seen.clear()
        for pair in ((-1, 0), (0, 2 ** 64)):
            with pytest.raises(Exception, match=r"2\^64"):
                f(torch.ones(8), pair)
    torch._dynamo.reset()


def _leaf(*shape, device, grad=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(device).requires_grad_(grad)


# (operator, which of its inputs need gradients, whether dy depends on something differentiated, gradients that go on)
SECOND_ORDER = [
    ("norm", "x", False, "x"), ("norm", "w", False, ""), ("norm", "w", True, "w"), ("norm", "xw", False, "xw"),
    ("norm", "xwr", True, "xwr"), ("norm", "r", False, "r"),
    ("dropout", "x", False, ""), ("dropout", "x", True, "x"), ("dropout", "xr", True, "xr"),
    ("grouped", "x", False, ""), ("grouped", "w", False, ""), ("grouped", "xw", False, "xw"), ("grouped", "x", True, "x"),
]


def second_derivatives_raise(op, need, dy_grad, graph, device):
    """Under create_graph a gradient that depends on something differentiated has a graph, and going back through
    the operator's part of it raises; one that depends on nothing has none.  The values are the same."""
    x, r = (_leaf(8, 32, device=device, grad=n in need, seed=i) for i, n in enumerate("xr"))
    w = _leaf(*((2, 32, 32) if op == "grouped" else (32,)), device=device, grad="w" in need, seed=3)
    dy = _leaf(8, 32, device=device, grad=dy_grad, seed=4)
    res = r if "r" in need else None
    if op == "norm":
        y = branch.rms_norm(x, w, residual=res)
        y = y if res is None else y[0]
    elif op == "dropout":
        y = branch.dropout(x, 0.5, (1, 2), residual=res)
    else:
        y = branch.grouped_matmul(x, w, torch.tensor([3, 8], dtype=torch.int32, device=device))
    leaves = {n: t for n, t in zip("xwr", (x, w, r)) if n in need}
    plain = torch.autograd.grad(y, list(leaves.values()), dy, retain_graph=True)
    grads = torch.autograd.grad(y, list(leaves.values()), dy, create_graph=True)
    for n, g, p in zip(leaves, grads, plain):
        assert torch.equal(g, p) and g.dtype == leaves[n].dtype
        assert g.requires_grad == (n in graph), n
        if op == "dropout" and n == "r":  # dy itself
            assert torch.equal(torch.autograd.grad(g.sum(), dy)[0], torch.ones_like(dy))
        elif n in graph:
            with pytest.raises(RuntimeError, match="no second derivative"):
                (g.square().sum() + x.sum()).backward()


@pytest.mark.parametrize("op,need,dy_grad,graph", SECOND_ORDER)
def test_second_derivatives_raise(monkeypatch, op, need, dy_grad, graph):
    """The Python nodes, with stand-in launchers that return new tensors."""
    one = lambda t: torch.ones(t.shape)  # noqa: E731
    monkeypatch.setattr(_branch, "rms_norm_forward", lambda x, w, res, eps, want_rstd=True: (
        one(x), None if res is None else one(x), torch.ones(8)))
    monkeypatch.setattr(_branch, "rms_norm_backward", lambda dy, h, dh, w, rstd, need_dx=True, need_dw=True: (
        one(h) if need_dx else None, one(w) if need_dw else None))
    monkeypatch.setattr(_branch, "dropout", lambda x, p, rng, res=None, want_used=False: (one(x), None))
    monkeypatch.setattr(_branch, "grouped_matmul_forward", lambda x, w, off: one(x))
    monkeypatch.setattr(_branch, "grouped_matmul_backward_input", lambda dy, w, off: one(dy))
    monkeypatch.setattr(_branch, "grouped_matmul_backward_weight", lambda dy, x, off: torch.ones(2, 32, 32))
    second_derivatives_raise(op, need, dy_grad, graph, "cpu")
