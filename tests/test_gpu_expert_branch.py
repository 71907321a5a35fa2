"""examples/expert_branch.py: the branch's operators together, as a user has them."""

import importlib.util
import os

import numpy as np
import pytest
import torch

from helpers import rel_err, to_np
from oracle import branch_oracle as O

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("expert_branch", os.path.join(ROOT, "examples", "expert_branch.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def reference(branch, x, rng):
    """The branch in float64 torch on the CPU, from the definition; returns (out, leaves)."""
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in branch.named_parameters()}
    x = x.detach().double().cpu().requires_grad_()
    tokens = x.flatten(0, 1)
    mixed = torch.cat((torch.zeros_like(x[:, :1]), x[:, :-1]), 1) * p["shift"]
    h = tokens + mixed.flatten(0, 1)
    y = h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * p["norm"]
    gates, chosen = (h @ p["router"]).softmax(-1).topk(branch.top_k, -1)
    gates = gates / gates.sum(-1, keepdim=True)
    out = torch.zeros_like(h)
    for e in range(branch.experts):
        u = y @ p["up"][e].T
        gate, value = u.chunk(2, -1)
        z = (torch.nn.functional.silu(gate) * value) @ p["down"][e].T
        out = out + z * (gates * (chosen == e)).sum(-1, keepdim=True)
    f = torch.from_numpy(O.dropout_factors(out.numel(), branch.p, *rng)).view(out.shape)
    return (h + out * f).view_as(x), {"x": x, **p}


def test_branch_against_its_definition(example):
    """fp32: the longest chain is five products and sums of up to 96 terms, each within 2^-17 of its terms'
    magnitudes; 1e-4 of the largest value leaves room for how they add up."""
    torch.manual_seed(0)
    B, S, D = 2, 37, 96
    branch = example.ExpertBranch(D, 64, 6, top_k=2, p=0.25).cuda()
    x = torch.randn(B, S, D, device="cuda", requires_grad=True)
    dy = torch.randn(B, S, D, device="cuda")
    rng = (11, 3)
    out = branch(x, rng)
    grads = torch.autograd.grad(out, [x, *branch.parameters()], dy)
    ref, leaves = reference(branch, x, rng)
    want = torch.autograd.grad(ref, [leaves["x"], *(leaves[n] for n, _ in branch.named_parameters())], dy.double().cpu())
    assert rel_err(to_np(out), ref.detach().numpy()) < 1e-4
    for name, g, w in zip(["x", *(n for n, _ in branch.named_parameters())], grads, want):
        assert rel_err(to_np(g), w.numpy()) < 1e-4, name


def test_example_trains_and_serves(example):
    got = example.main(["--dim", "128", "--hidden", "64", "--experts", "4", "--batch", "4", "--seq", "64", "--steps", "40"])
    first, last = np.mean(got["losses"][:5]), np.mean(got["losses"][-5:])
    assert np.isfinite(got["losses"]).all() and last < 0.8 * first
    assert got["off"] < 0.1  # 4 significant bits an operand
