"""examples/decay_layer.py: the operators that mix tokens together, as a user has them."""

import importlib.util
import os

import numpy as np
import pytest
import torch

from helpers import rel_err, to_np

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("decay_layer", os.path.join(ROOT, "examples", "decay_layer.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def norm(x, w):
    return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w


def mixer_reference(m, x):
    """The mixing branch in float64 torch on the CPU, from the definition, token by token; (out, leaves)."""
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in m.named_parameters()}
    x = x.detach().double().cpu().requires_grad_()
    B, T, _ = x.shape
    q, k, v = (norm(x, p["norm"]) @ p["qkv"].T).view(B, T, 3, m.heads, m.head_dim).unbind(2)
    angle = torch.arange(T, dtype=torch.float64)[:, None] * m.frequencies.cpu()
    c, s = angle.cos()[:, None], angle.sin()[:, None]

    def turned(t):
        a, b = t.chunk(2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    q, k, keep = turned(q), turned(k), m.log_decay.double().cpu().exp()[:, None, None]
    state, rows = torch.zeros(B, m.heads, m.head_dim, m.head_dim, dtype=torch.float64), []
    for t in range(T):
        state = keep * state + k[:, t].unsqueeze(-1) * v[:, t].unsqueeze(-2)
        rows.append((q[:, t].unsqueeze(-2) @ state).squeeze(-2) * m.head_dim ** -0.5)
    return torch.stack(rows, 1).flatten(-2) @ p["out"].T, {"x": x, **p}


def ff_reference(m, x):
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in m.named_parameters()}
    x = x.detach().double().cpu().requires_grad_()
    gate, value = (norm(x, p["norm"]) @ p["up"].T).chunk(2, -1)
    return (torch.nn.functional.silu(gate) * value) @ p["down"].T, {"x": x, **p}


@pytest.mark.parametrize("kind", ["mixer", "feed-forward"])
def test_branches_against_their_definitions(example, kind):
    """fp32: the longest chain is five products and sums of up to 96 terms, each within 2^-17 of its terms' magnitudes, and the
    state's; 1e-4 of the largest value leaves room for how they add up."""
    torch.manual_seed(0)
    m = (example.DecayMixer(96, 3) if kind == "mixer" else example.GatedFeedForward(96, 80)).cuda()
    x = torch.randn(2, 70, 96, device="cuda", requires_grad=True)
    dy = torch.randn(2, 70, 96, device="cuda")
    out = m(x)
    grads = torch.autograd.grad(out, [x, *m.parameters()], dy)
    ref, leaves = (mixer_reference if kind == "mixer" else ff_reference)(m, x)
    want = torch.autograd.grad(ref, [leaves["x"], *(leaves[n] for n, _ in m.named_parameters())], dy.double().cpu())
    assert rel_err(to_np(out), ref.detach().numpy()) < 1e-4
    for name, g, w in zip(["x", *(n for n, _ in m.named_parameters())], grads, want):
        assert rel_err(to_np(g), w.numpy()) < 1e-4, name


def test_casts_leave_decays_and_frequencies(example):
    m = example.DecayMixer(96, 3).cuda().to(torch.bfloat16)
    assert m.log_decay.dtype == torch.float32 and m.frequencies.dtype == torch.float64 and m.frequencies.is_cuda
    assert m.qkv.dtype == torch.bfloat16


def test_packed_sequences_are_the_sequences(example):
    """Several sequences packed give what each gives by itself, in fp32 to rounding."""
    torch.manual_seed(0)
    model = example.Stack(64, 2, 96, 2).cuda()
    parts = [torch.randn(n, 64, device="cuda") for n in (5, 70, 1, 33)]
    with torch.no_grad():
        out = model(torch.cat(parts), torch.tensor([5, 75, 76, 109], dtype=torch.int32, device="cuda"))
        want = torch.cat([model(p[None])[0] for p in parts])
    assert rel_err(to_np(out), to_np(want)) < 1e-5


def test_example_trains_and_serves(example):
    got = example.main(["--dim", "128", "--heads", "4", "--hidden", "192", "--batch", "4", "--seq", "96", "--steps", "6"])
    assert np.isfinite(got["losses"]).all()
    # bf16 activations of other products' shapes differ by roundings of 2^-9 through four branches
    assert got["off"] < 0.03
