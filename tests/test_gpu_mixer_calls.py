"""The operators that mix tokens on the GPU: calls that their documentation allows and that test_gpu_mixer.py and
test_gpu_mixer_paths.py do not make."""

import pytest
import torch

from test_gpu_branch import DT, rand
from test_gpu_mixer import check_decay, decays

pytestmark = pytest.mark.gpu

DEV = "cuda"


# --------------------------------------------------------------------------
# Rows that share memory
# --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("which", ["kv", "qd", "qkvd"])
@pytest.mark.parametrize("B,T,D", [(1, 100, 64), (2, 1, 64), (2, 70, 128), (1, 300, 40)])
def test_tokens_that_are_one_expanded(B, T, D, which, dtype):
    """Operands and gradients of row stride 0, whole chunks and short ones."""
    dt, H = DT[dtype], 2
    t = {n: (rand(H, D, seed=i, dtype=dt).expand(B, T, H, D) if n in which else rand(B, T, H, D, seed=i, dtype=dt))
         for i, n in enumerate("qkvd")}
    q, k, v = (t[n].detach().requires_grad_() for n in "qkv")
    first, d_last = rand(B, H, D, D, seed=5).requires_grad_(), rand(B, H, D, D, seed=6)
    check_decay(q, k, v, decays(H), None, first, t["d"], d_last, 0.1, [(n * T, (n + 1) * T) for n in range(B)])


@pytest.mark.parametrize("dtype", list(DT))
def test_tokens_that_are_windows_of_one_row(dtype):
    """Rows 8 elements apart, which overlap."""
    dt, T, H, D = DT[dtype], 90, 2, 64
    q, k, v, do = (rand(8 * T + H * D, seed=i, dtype=dt).as_strided((T, H, D), (8, D, 1)) for i in range(4))
    off = torch.tensor([30, 85], device=DEV)
    first, d_last = rand(2, H, D, D, seed=5).requires_grad_(), rand(2, H, D, D, seed=6)
    check_decay(*(t.detach().requires_grad_() for t in (q, k, v)), decays(H), off, first, do, d_last, 0.1, [(0, 30), (30, 85)])
