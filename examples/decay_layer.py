"""A hyper-connection stack that mixes tokens by decay attention, trained, given a prompt, and then decoded.

Each layer has two branches, each behind a ``HyperConnection`` of its own: one mixes tokens (norm, projections,
rotary positions, linear attention with a decay for each head), one is a gated feed-forward.  Training and
prompts run over whole sequences; decoding moves each sequence's state on by a token, in a captured HIP graph, over
a pool of states that requests share.

    python examples/decay_layer.py              # trains a few steps on synthetic data, then decodes
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
from mhc.branch import (decay_attention, decay_attention_step, gated_matmul, rms_norm, rotary,  # noqa: E402
                        rotary_frequencies)
from mhc.streams import collapse_streams, expand_streams  # noqa: E402


class DecayMixer(nn.Module):
    """x -> out(attention(norm(x))); heads keep between half and all but 2^-8 of their state at each token."""

    def __init__(self, dim: int, heads: int):
        super().__init__()
        self.heads, self.head_dim = heads, dim // heads
        self.norm = nn.Parameter(torch.ones(dim))
        self.qkv = nn.Parameter(torch.randn(3 * dim, dim) * dim ** -0.5)
        self.out = nn.Parameter(torch.randn(dim, dim) * dim ** -0.5)
        self.register_buffer("log_decay", -torch.exp2(-torch.linspace(0.0, 8.0, heads)), persistent=False)
        self.register_buffer("frequencies", rotary_frequencies(self.head_dim), persistent=False)

    def _apply(self, fn):  # a cast of the module to 16 bits leaves decays and frequencies as they are
        decay, freq = self.log_decay, self.frequencies
        super()._apply(fn)
        self.log_decay, self.frequencies = decay.to(self.log_decay.device), freq.to(self.frequencies.device)
        return self

    def heads_of(self, x, positions):
        """q, k, v (..., heads, head dim) of x (..., dim); they stay parts of one projection's rows."""
        qkv = nn.functional.linear(rms_norm(x, self.norm), self.qkv).unflatten(-1, (3 * self.heads, self.head_dim))
        q, k, v = qkv.split(self.heads, -2)
        return (*rotary(q, k, positions, self.frequencies), v)

    def forward(self, x, offsets=None, return_state=False):
        """x (batch, tokens, dim), or packed (tokens, dim) with the sequences' ends, each from its first position on."""
        if offsets is None:
            positions = torch.arange(x.shape[1], device=x.device, dtype=torch.int32)
        else:
            row = torch.arange(x.shape[0], device=x.device)
            start = torch.cat((offsets.new_zeros(1), offsets)).long()
            positions = (row - start[torch.searchsorted(offsets.long(), row, right=True)]).int()
        o = decay_attention(*self.heads_of(x, positions), self.log_decay, offsets=offsets, return_state=return_state)
        o, state = o if return_state else (o, None)
        y = nn.functional.linear(o.flatten(-2), self.out)
        return (y, state) if return_state else y

    def step(self, x, positions, state, slots):
        """One token of each request, x (requests, dim), whose states lie at `slots` of the pool `state`."""
        o = decay_attention_step(*self.heads_of(x, positions), self.log_decay, state, slots=slots)
        return nn.functional.linear(o.flatten(-2), self.out)


class GatedFeedForward(nn.Module):
    def __init__(self, dim: int, hidden: int):
        super().__init__()
        self.norm = nn.Parameter(torch.ones(dim))
        self.up = nn.Parameter(torch.randn(2 * hidden, dim) * dim ** -0.5)  # gate, then value
        self.down = nn.Parameter(torch.randn(dim, hidden) * hidden ** -0.5)

    def forward(self, x):
        rows = gated_matmul(rms_norm(x, self.norm).flatten(0, -2), self.up)
        return nn.functional.linear(rows, self.down).view(x.shape)


class Stack(nn.Module):
    def __init__(self, dim: int, heads: int, hidden: int, layers: int):
        super().__init__()
        # static weights: those of a dynamic layer come from a whole sequence's mean, which decoding does not have
        self.hc = nn.ModuleList(mhc.HyperConnection(dim, dynamic=False, layer_idx=i) for i in range(2 * layers))
        self.mixer = nn.ModuleList(DecayMixer(dim, heads) for _ in range(layers))
        self.ff = nn.ModuleList(GatedFeedForward(dim, hidden) for _ in range(layers))

    def forward(self, x, offsets=None):
        return self._run(x, lambda mixer, bi: mixer(bi, offsets), packed=offsets is not None)

    def _run(self, x, mix, packed=False):
        """x (batch, tokens, dim) through the layers; mix(mixer, branch input) mixes the tokens."""
        H = expand_streams(x[None] if packed else x)
        for i, (mixer, ff) in enumerate(zip(self.mixer, self.ff)):
            for hc, branch in ((self.hc[2 * i], lambda bi: mix(mixer, bi)), (self.hc[2 * i + 1], ff)):
                bi, add_residual = hc(H)
                H = add_residual(branch(bi[0])[None] if packed else branch(bi))
        y = collapse_streams(H)
        return y[0] if packed else y

    @torch.no_grad()
    def prompt(self, x, offsets, pool, slots):
        """Packed prompts x (tokens, dim): their outputs; the states go to `slots` of each layer's pool."""
        def mix(mixer, bi):
            y, state = mixer(bi, offsets, return_state=True)
            pool[states.pop(0)].index_copy_(0, slots.long(), state)
            return y

        states = list(range(len(self.mixer)))
        return self._run(x, mix, packed=True)

    @torch.no_grad()
    def step(self, x, positions, pool, slots):
        """One token of each request, x (requests, dim)."""
        states = list(pool)
        return self._run(x[:, None], lambda mixer, bi: mixer.step(bi[:, 0], positions, states.pop(0), slots)[:, None])[:, 0]

    def states(self, places: int, device):
        """A pool of states for each layer, zeros."""
        m = self.mixer[0]
        return [torch.zeros(places, m.heads, m.head_dim, m.head_dim, device=device) for _ in self.mixer]


def train(model, steps: int, batch: int, seq: int, dim: int, dtype=torch.bfloat16, seed: int = 0):
    """Losses of learning a fixed map of each token's running average over its past."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    target = torch.randn(dim, dim, generator=g, device="cuda") * dim ** -0.5
    opt = torch.optim.AdamW(model.parameters(), lr=1e-3)
    losses = []
    for _ in range(steps):
        x = torch.randn(batch, seq, dim, generator=g, device="cuda")
        past = x.cumsum(1) / torch.arange(1, seq + 1, device="cuda").sqrt()[:, None]
        loss = (model(x.to(dtype)).float() - torch.tanh(past @ target)).square().mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main(argv=None) -> dict:
    a = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    a.add_argument("--dim", type=int, default=512)
    a.add_argument("--heads", type=int, default=8)
    a.add_argument("--hidden", type=int, default=1024)
    a.add_argument("--layers", type=int, default=2)
    a.add_argument("--batch", type=int, default=8)
    a.add_argument("--seq", type=int, default=256)
    a.add_argument("--steps", type=int, default=40)
    o = a.parse_args(argv)
    torch.manual_seed(0)
    model = Stack(o.dim, o.heads, o.hidden, o.layers).cuda().to(torch.bfloat16)
    losses = train(model, o.steps, o.batch, o.seq, o.dim)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {o.steps} steps", flush=True)

    # prompts of several lengths, packed, then tokens one by one; the whole sequences at once are the yardstick
    model.eval()
    lengths, more = [o.seq - 7 * i for i in range(o.batch)], 4
    whole = [torch.randn(n + more, o.dim, device="cuda").to(torch.bfloat16) for n in lengths]
    with torch.no_grad():
        want = [model(x[None])[0] for x in whole]
    pool = model.states(o.batch + 3, "cuda")
    slots = torch.arange(o.batch, device="cuda", dtype=torch.int32) + 2
    offsets = torch.tensor(lengths, device="cuda").cumsum(0).int()
    out = model.prompt(torch.cat([x[:n] for x, n in zip(whole, lengths)]), offsets, pool, slots)
    x = torch.zeros(o.batch, o.dim, device="cuda", dtype=torch.bfloat16)
    positions = torch.zeros(o.batch, device="cuda", dtype=torch.int32)
    spare = [p.clone() for p in pool]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model.step(x, positions, spare, slots)
    torch.cuda.current_stream().wait_stream(side)
    kept = [p.clone() for p in pool]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = model.step(x, positions, pool, slots)
    for p, k in zip(pool, kept):
        p.copy_(k)
    off = [float((out[e - n:e].float() - w[:n].float()).norm() / w[:n].float().norm())
           for e, n, w in zip(offsets.tolist(), lengths, want)]
    for t in range(more):
        x.copy_(torch.stack([w[n + t] for w, n in zip(whole, lengths)]))
        positions.copy_(torch.tensor([n + t for n in lengths], dtype=torch.int32))
        graph.replay()
        off += [float((row.float() - w[n + t].float()).norm() / w[n + t].float().norm())
                for row, w, n in zip(y, want, lengths)]
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(50):
        graph.replay()
    torch.cuda.synchronize()
    us = (time.perf_counter() - began) / 50 * 1e6
    print(f"prompts and decoding: at most {100 * max(off):.2f}% from whole sequences, {us:.0f} us a step of {o.batch} tokens",
          flush=True)
    return {"losses": losses, "off": max(off), "us": us}


if __name__ == "__main__":
    main()
