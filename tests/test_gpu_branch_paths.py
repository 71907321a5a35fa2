"""``mhc.branch`` on the GPU, beside test_gpu_branch.py: calls and kernels that its cases do not reach."""

import pytest
import torch

from test_branch_cpu import SECOND_ORDER, _forward_mode_calls, forward_mode_is_refused, second_derivatives_raise
from helpers import to_np
from test_gpu_branch import DT, close, rand
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
