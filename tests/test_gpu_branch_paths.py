"""``mhc.branch`` on the GPU, beside test_gpu_branch.py: calls and kernels that its cases do not reach."""

import pytest
import torch

from test_branch_cpu import _forward_mode_calls, forward_mode_is_refused

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("name", list(_forward_mode_calls("cpu")))
def test_forward_mode_is_refused(name):
    forward_mode_is_refused(name, DEV)
