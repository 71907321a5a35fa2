"""A hyper-connection stack whose branches are mixtures of experts, trained and then served.

Everything between ``HyperConnection``'s branch input and its closure runs on ``mhc.branch``: the norm with
the residual's addition, the experts' products over rows sorted by expert, dropout without a stored mask,
and for serving the same products in 8 bits, captured in a HIP graph.  The router, the sort and the
combination are plain torch and wait for nothing on the host.

    python examples/expert_branch.py            # trains a few steps on synthetic data, then decodes
"""

from __future__ import annotations

import argparse
import os
import sys
import time

import torch
from torch import nn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (os.path.join(ROOT, "mhc-triton_amd"),):
    if p not in sys.path:
        sys.path.insert(0, p)

import mhc  # noqa: E402
from mhc.branch import dropout, grouped_matmul, grouped_matmul_mx, quantize_mx, rms_norm, rms_norm_mx  # noqa: E402
from mhc.streams import collapse_streams, expand_streams  # noqa: E402


class ExpertBranch(nn.Module):
    """h = x + shifted x;  x -> h + dropout(experts(norm(h))), each token through its top_k experts."""

    def __init__(self, dim: int, hidden: int, experts: int, top_k: int = 2, p: float = 0.1):
        super().__init__()
        self.experts, self.top_k, self.p = experts, top_k, p
        self.shift = nn.Parameter(torch.full((dim,), 0.1))
        self.norm = nn.Parameter(torch.ones(dim))
        self.router = nn.Parameter(torch.randn(dim, experts) * dim ** -0.5)
        self.up = nn.Parameter(torch.randn(experts, 2 * hidden, dim) * dim ** -0.5)  # gate and value
        self.down = nn.Parameter(torch.randn(experts, dim, hidden) * hidden ** -0.5)

    def mixed(self, x):
        """The previous token's features, a channel's share of them each."""
        return torch.cat((torch.zeros_like(x[:, :1]), x[:, :-1]), 1) * self.shift.to(x.dtype)

    def route(self, h):
        """(gates [T, k], order [T k], offsets [E]): the experts of each token, and the (token, choice) pairs
        sorted by expert."""
        gates, chosen = (h.float() @ self.router.float()).softmax(-1).topk(self.top_k, -1)
        chosen = chosen.flatten()
        order = chosen.argsort(stable=True)
        counts = torch.zeros(self.experts, dtype=torch.int64, device=h.device).scatter_add_(
            0, chosen, torch.ones_like(chosen))
        return gates / gates.sum(-1, keepdim=True), order, counts.cumsum(0).int()

    def combine(self, rows, order, gates):
        """Rows sorted by expert back to their tokens, weighted by the gates."""
        back = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device=order.device))
        return (rows[back].view(*gates.shape, -1) * gates.to(rows.dtype).unsqueeze(-1)).sum(1)

    def forward(self, x, rng):
        """x (batch, seq, dim); rng (seed, offset) or a tensor of two on the GPU."""
        tokens = x.flatten(0, 1)
        y, h = rms_norm(self.mixed(x).flatten(0, 1), self.norm, residual=tokens)
        gates, order, offsets = self.route(h)
        u = grouped_matmul(y[order // self.top_k], self.up, offsets)
        gate, value = u.chunk(2, -1)
        out = self.combine(grouped_matmul(nn.functional.silu(gate) * value, self.down, offsets), order, gates)
        return dropout(out, self.p, rng, residual=h, training=self.training).view_as(x)

    def quantized(self):
        """The experts' weights in 8 bits, made once for serving."""
        with torch.no_grad():
            return quantize_mx(self.up), quantize_mx(self.down)

    @torch.no_grad()
    def serve(self, x, weights):
        """The same without dropout, its products in 8 bits."""
        (up, up_scales), (down, down_scales) = weights
        tokens = x.flatten(0, 1)
        q, scales, h = rms_norm_mx(self.mixed(x).flatten(0, 1), self.norm, residual=tokens)
        gates, order, offsets = self.route(h)
        token = order // self.top_k
        q, scales = (t.view(torch.uint8)[token].view(t.dtype) for t in (q, scales))
        u = grouped_matmul_mx(q, scales, up, up_scales, offsets, out_dtype=x.dtype)
        gate, value = u.chunk(2, -1)
        rows = grouped_matmul_mx(*quantize_mx(nn.functional.silu(gate) * value), down, down_scales, offsets,
                                 out_dtype=x.dtype)
        return (h + self.combine(rows, order, gates)).view_as(x)


class Stack(nn.Module):
    def __init__(self, dim: int, hidden: int, experts: int, layers: int):
        super().__init__()
        self.hc = nn.ModuleList(mhc.HyperConnection(dim, layer_idx=i) for i in range(layers))
        self.branch = nn.ModuleList(ExpertBranch(dim, hidden, experts) for _ in range(layers))

    def forward(self, x, seed: int, step: int):
        H = expand_streams(x)
        for i, (hc, branch) in enumerate(zip(self.hc, self.branch)):
            bi, add_residual = hc(H)
            H = add_residual(branch(bi, (seed, step * len(self.hc) + i)))  # a mask of its own each layer and step
        return collapse_streams(H)

    @torch.no_grad()
    def serve(self, x, weights):
        H = expand_streams(x)
        for hc, branch, w in zip(self.hc, self.branch, weights):
            bi, add_residual = hc(H)
            H = add_residual(branch.serve(bi, w))
        return collapse_streams(H)


def train(model, steps: int, batch: int, seq: int, dim: int, dtype=torch.bfloat16, seed: int = 0):
    """Losses of learning a fixed random map of each token from its own and the previous one."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    target = torch.randn(dim, dim, generator=g, device="cuda") * dim ** -0.5
    opt = torch.optim.AdamW(model.parameters(), lr=2e-3)
    losses = []
    for step in range(steps):
        x = torch.randn(batch, seq, dim, generator=g, device="cuda").to(dtype)
        want = torch.tanh(x.float() @ target)
        loss = (model(x, seed, step).float() - want).square().mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main(argv=None) -> dict:
    a = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    a.add_argument("--dim", type=int, default=512)
    a.add_argument("--hidden", type=int, default=512)
    a.add_argument("--experts", type=int, default=8)
    a.add_argument("--layers", type=int, default=2)
    a.add_argument("--batch", type=int, default=8)
    a.add_argument("--seq", type=int, default=256)
    a.add_argument("--steps", type=int, default=60)
    o = a.parse_args(argv)
    torch.manual_seed(0)
    model = Stack(o.dim, o.hidden, o.experts, o.layers).cuda().to(torch.bfloat16)
    losses = train(model, o.steps, o.batch, o.seq, o.dim)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {o.steps} steps", flush=True)

    model.eval()
    weights = [b.quantized() for b in model.branch]
    x = torch.randn(o.batch, 1, o.dim, device="cuda").to(torch.bfloat16)  # one token of each sequence
    with torch.no_grad():
        plain = model(x, 0, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model.serve(x, weights)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.serve(x, weights)
    graph.replay()
    torch.cuda.synchronize()
    off = float((out.float() - plain.float()).norm() / plain.float().norm())
    began = time.perf_counter()
    for _ in range(50):
        graph.replay()
    torch.cuda.synchronize()
    us = (time.perf_counter() - began) / 50 * 1e6
    print(f"decode in 8 bits: {100 * off:.1f}% from bf16, {us:.0f} us a step of {o.batch} tokens", flush=True)
    return {"losses": losses, "off": off, "us": us}


if __name__ == "__main__":
    main()
