"""``mhc.branch`` on the GPU, beside test_gpu_branch.py: calls and kernels that its cases do not reach."""

import pytest
import torch

from test_branch_cpu import _forward_mode_calls, forward_mode_is_refused
from test_gpu_branch import rand
from test_gpu_native_nodes import both, same
from mhc import branch

pytestmark = pytest.mark.gpu

DEV = "cuda"


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
