"""The operators of a token-mixing layer (``mhc.branch``), as cases that can be timed and checked.

A layer's mixing branch gives its queries and keys rotary positions and runs them through linear attention with a
decay for each head: chunk by chunk over prompts and training sequences, a token at a time when decoding.  Its
feed-forward branch begins with a gated product.  ``op`` names the operator of a case:

* ``rotary``  ``rotary`` of queries and keys (fewer heads), forward alone ("infer") or with the backward ("train").
* ``decay``   ``decay_attention`` over sequences of one length or packed ones ("infer" returns the states, "train"
              the gradients), or ``decay_attention_step`` of one token a sequence ("step").
* ``gated``   ``gated_matmul``: act(x gate) * (x up), of all rows by one weight or of rows sorted by expert.

Sizes are the benchmark's, the tests' and the README example's, or plain round and odd numbers between
them.  ``run`` computes the plain form in 32-bit torch operations, or with ``own`` calls the package.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mhc-triton_amd")
_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_CHUNK = 64


def _rotary(name, R, heads, kv_heads, D, part, dtype, mode, interleaved=False, factor=1.0, far=4096):
    return {"name": name, "op": "rotary", "R": R, "heads": heads, "kv_heads": kv_heads, "D": D, "part": part,
            "dtype": dtype, "mode": mode, "interleaved": interleaved, "factor": factor, "far": far}


def _decay(name, seqs, tokens, heads, Dk, Dv, dtype, mode, packed=False, states=False, empty=0):
    return {"name": name, "op": "decay", "seqs": seqs, "tokens": tokens, "heads": heads, "Dk": Dk, "Dv": Dv,
            "dtype": dtype, "mode": mode, "packed": packed, "states": states, "empty": empty}


def _gated(name, R, K, N, E, dtype, mode, act="silu", empty=0):
    return {"name": name, "op": "gated", "R": R, "K": K, "N": N, "E": E, "empty": empty, "dtype": dtype, "mode": mode,
            "act": act}


def listed():
    return [
        # a batch of 16 decoded tokens far into a context that was stretched 8 times: latency
        _rotary("rotary decode", 16, 32, 8, 128, 128, "bf16", "infer", factor=8.0, far=131072),
        # the headline workload's tokens (batch 4, sequence 4096) in heads of 128, forward and backward
        _rotary("rotary train", 16384, 32, 8, 128, 128, "bf16", "train"),
        # an odd number of tokens, heads that are no whole vectors, part of each turned, neighbours paired
        _rotary("rotary ragged", 3069, 12, 12, 100, 36, "fp32", "train", interleaved=True),
        # one decoded token: a state of 2 MB
        _decay("decay step", 1, 1, 32, 128, 128, "bf16", "step"),
        # 128 decoded tokens of as many sequences, their states in places of a pool
        _decay("decay step batch", 128, 128, 32, 128, 128, "bf16", "step"),
        # a long prompt alone: few heads for many CUs; its state is what decoding starts from
        _decay("decay prompt", 1, 8192, 32, 128, 128, "bf16", "infer"),
        # the headline workload's tokens, forward and backward
        _decay("decay train", 4, 16384, 32, 128, 128, "bf16", "train"),
        # packed sequences of uneven lengths that go on from states, one of them without tokens, odd head sizes
        _decay("decay ragged", 7, 3069, 12, 100, 72, "fp32", "train", packed=True, states=True, empty=1),
        # a batch of 16 decoded tokens: bound by reading the weight
        _gated("gated decode", 16, 4096, 8192, 1, "bf16", "infer"),
        # the headline workload's tokens, forward and both gradients
        _gated("gated train", 16384, 4096, 8192, 1, "bf16", "train"),
        # 4096 tokens through two experts each of 16 narrow ones
        _gated("gated experts", 8192, 2048, 1024, 16, "bf16", "train"),
        # odd lengths, widths that are not whole vectors, experts without tokens
        _gated("gated ragged", 3069, 1500, 1001, 6, "fp16", "train", act="gelu", empty=2),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi, unit=8, any_share=0.25):
    """A width: mostly whole 16-byte vectors, now and then any number."""
    v = _log(rng, lo, hi)
    return v if rng.random() < any_share else max(unit, v // unit * unit)


def _draw_any(rng):
    op = rng.choice(["rotary", "decay", "decay", "decay", "gated", "gated"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "rotary":
        D = _width(rng, 16, 256)
        part = D // 2 * 2 if rng.random() < 0.6 else 2 * rng.randint(1, D // 2)
        kv = _log(rng, 1, 16)
        return {"op": op, "R": _log(rng, 1, 32768), "heads": kv * rng.randint(1, 8), "kv_heads": kv, "D": D,
                "part": part, "dtype": dtype, "mode": rng.choice(["infer", "train"]),
                "interleaved": rng.random() < 0.5, "factor": rng.choice([1.0, 4.0, 8.0]),
                "far": _log(rng, 1024, 1 << 20)}
    if op == "decay":
        mode = rng.choice(["step", "infer", "train", "train"])
        seqs = _log(rng, 1, 128 if mode == "step" else 24)
        packed = mode != "step" and rng.random() < 0.5
        if mode == "step":
            tokens = seqs
        elif packed:
            tokens = _log(rng, 1, 16384)
        else:
            tokens = seqs * _log(rng, 1, max(1, 16384 // seqs))
        return {"op": op, "seqs": seqs, "tokens": tokens, "heads": _log(rng, 1, 40), "Dk": _width(rng, 16, 128),
                "Dv": _width(rng, 16, 128), "dtype": dtype, "mode": mode, "packed": packed,
                "states": mode != "step" and rng.random() < 0.4, "empty": rng.randint(0, seqs // 4) if packed else 0}
    E = rng.choice([1, _log(rng, 2, 48)])
    return {"op": op, "R": _log(rng, 1, 16384), "K": _width(rng, 64, 8192), "N": _width(rng, 64, 8192), "E": E,
            "empty": rng.randint(0, E // 3), "dtype": dtype, "mode": rng.choice(["infer", "train"]),
            "act": rng.choice(["silu", "gelu", "gelu_tanh"])}


def draw(rng):
    top = [work(c) for c in listed()]
    while True:
        case = _draw_any(rng)
        w = work(case)
        # a matrix product in 32 bits costs about 16 times one in 16 bits
        flops = w["flops"] * (16 if case["op"] == "gated" and case["dtype"] == "fp32" else 1)
        weights = case["op"] == "gated" and case["E"] * case["K"] * case["N"]
        if (w["bytes"] <= max(t["bytes"] for t in top) and flops <= max(t["flops"] for t in top)
                and weights <= 1 << 27):
            return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _randn(shape, g, dtype, scale=1.0):
    t = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    return (t.mul_(scale) if scale != 1.0 else t).to(dtype)


def _sizes(R, E, empty, seed):
    """Rows of each expert, or tokens of each sequence: a few times more at one than at another, some without any."""
    r = np.random.RandomState(seed % (1 << 32))
    share = np.exp(0.5 * r.standard_normal(E))
    share[r.permutation(E)[:empty]] = 0.0
    return r.multinomial(R, share / share.sum())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _DT[case["dtype"]]
    mode = case["mode"]
    s = {"op": case["op"], "mode": mode}
    {"rotary": _prepare_rotary, "decay": _prepare_decay, "gated": _prepare_gated}[case["op"]](s, case, g, dtype, int(seed))
    return s


def _prepare_rotary(s, case, g, dtype, seed):
    R, D, train = case["R"], case["D"], case["mode"] == "train"
    # a projection's output holds a token's queries and keys side by side
    both = _randn((R, case["heads"] + case["kv_heads"], D), g, dtype)
    s["q"], s["k"] = (t.requires_grad_(train) for t in (both[:, :case["heads"]], both[:, case["heads"]:]))
    # sequences that begin anywhere up to the farthest position
    start = torch.randint(0, case["far"], ((R + 511) // 512,), generator=g, device="cuda")
    row = torch.arange(R, device="cuda")
    s["positions"] = (start[row // 512] + row % 512).int()
    i = torch.arange(case["part"] // 2, dtype=torch.float64, device="cuda")
    s["frequencies"] = 10000.0 ** (-2.0 * i / case["part"]) / case["factor"]
    s["interleaved"] = case["interleaved"]
    s["magnitude"] = 0.1 * math.log(case["factor"]) + 1.0
    if train:
        s["dq"], s["dk"] = _randn(s["q"].shape, g, dtype), _randn(s["k"].shape, g, dtype)


def _prepare_decay(s, case, g, dtype, seed):
    N, T, H, Dk, Dv = (case[n] for n in ("seqs", "tokens", "heads", "Dk", "Dv"))
    step, train = case["mode"] == "step", case["mode"] == "train"
    lead = (T,) if step or case["packed"] else (N, T // N)
    q, k, v = (_randn((*lead, H, d), g, dtype) for d in (Dk, Dk, Dv))
    # from heads that forget within a few tokens to heads that hardly do
    s["log_decay"] = -torch.exp2(-torch.linspace(1.0, 11.0, H, device="cuda"))
    s["scale"] = Dk ** -0.5
    if step:
        pool = N + (N + 3) // 4
        s["state"] = _randn((pool, H, Dk, Dv), g, torch.float32, 4.0)
        s["next"] = s["state"].clone()
        s["slots"] = torch.randperm(pool, generator=g, device="cuda")[:N].int()
        s["q"], s["k"], s["v"] = q, k, v
        return
    s["q"], s["k"], s["v"] = (t.requires_grad_(train) for t in (q, k, v))
    sizes = _sizes(T, N, case["empty"], seed) if case["packed"] else np.full(N, T // N)
    s["most"] = int(sizes.max())
    s["sizes"] = torch.tensor(sizes, device="cuda")
    s["offsets"] = torch.tensor(np.cumsum(sizes), dtype=torch.int32, device="cuda") if case["packed"] else None
    s["state"] = _randn((N, H, Dk, Dv), g, torch.float32, 2.0).requires_grad_(train) if case["states"] else None
    if train:
        s["do"] = _randn(v.shape, g, dtype)
        s["dstate"] = _randn((N, H, Dk, Dv), g, torch.float32, 0.2) if case["states"] else None


def _prepare_gated(s, case, g, dtype, seed):
    R, K, N, E, train = case["R"], case["K"], case["N"], case["E"], case["mode"] == "train"
    s["act"] = case["act"]
    s["x"] = _randn((R, K), g, dtype).requires_grad_(train)
    s["w"] = _randn((2 * N, K) if E == 1 else (E, 2 * N, K), g, dtype, K ** -0.5).requires_grad_(train)
    sizes = _sizes(R, E, case["empty"], seed)
    s["most"] = int(sizes.max())
    s["offsets"] = torch.tensor(np.cumsum(sizes), dtype=torch.int32, device="cuda") if E > 1 else None
    if train:
        s["dy"] = _randn((R, N), g, dtype)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"rotary": _plain_rotary, "decay": _plain_decay, "gated": _plain_gated}[s["op"]](s)


def _run_own(s):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from mhc import branch

    train = s["mode"] == "train"
    with torch.set_grad_enabled(train):
        if s["op"] == "rotary":
            q, k = branch.rotary(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=s["interleaved"],
                                 magnitude=s["magnitude"])
            if not train:
                return {"q": q, "k": k}
            dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
            return {"q": q, "k": k, "dq": dq, "dk": dk}
        if s["op"] == "gated":
            y = branch.gated_matmul(s["x"], s["w"], s["offsets"], activation=s["act"])
            if not train:
                return {"y": y}
            dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
            return {"y": y, "dx": dx, "dw": dw}
        if s["mode"] == "step":
            o = branch.decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], slots=s["slots"],
                                            scale=s["scale"], state_out=s["next"])
            return {"o": o, "state": s["next"]}
        states = s["state"] is not None
        out = branch.decay_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["state"],
                                     offsets=s["offsets"], scale=s["scale"], return_state=states or not train)
        if not train:
            return {"o": out[0], "state": out[1]}
        if not states:
            dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"])
            return {"o": out, "dq": dq, "dk": dk, "dv": dv}
        dq, dk, dv, ds = torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["state"]), (s["do"], s["dstate"]))
        return {"o": out[0], "state": out[1], "dq": dq, "dk": dk, "dv": dv, "dstate": ds}


def _turned(x, cos, sin, interleaved, magnitude):
    """Rows (R, heads, D) with the pairs of the first 2 * cos.shape[1] elements turned; fp32."""
    n = cos.shape[1]
    x = x.float()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    c, t = (magnitude * cos).unsqueeze(1), (magnitude * sin).unsqueeze(1)
    a, b = a * c - b * t, b * c + a * t
    front = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((front, x[..., 2 * n:]), -1)


def _plain_rotary(s):
    angle = s["positions"].double().unsqueeze(1) * s["frequencies"]
    cos, sin = angle.cos().float(), angle.sin().float()
    dt, more = s["q"].dtype, (s["interleaved"], s["magnitude"])
    out = {"q": _turned(s["q"], cos, sin, *more).to(dt), "k": _turned(s["k"], cos, sin, *more).to(dt)}
    if s["mode"] == "train":
        out["dq"] = _turned(s["dq"], cos, -sin, *more).to(dt)
        out["dk"] = _turned(s["dk"], cos, -sin, *more).to(dt)
    return out


def _weighted(q, k, v, ld):
    """o_t = sum over s <= t of exp(ld (t - s)) (q_t . k_s) v_s for q, k, v (N, H, T, D), T whole chunks: inside the
    chunks by their weight matrices, across them through the chunks' states."""
    N, H, T, _ = q.shape
    n = T // _CHUNK
    q, k, v = (t.reshape(N, H, n, _CHUNK, t.shape[-1]) for t in (q, k, v))
    i = torch.arange(_CHUNK, device=q.device)
    far = (i.unsqueeze(1) - i).clamp_min(0)
    inside = torch.exp(ld.view(-1, 1, 1) * far) * (i.unsqueeze(1) >= i)
    o = (torch.matmul(q, k.transpose(-1, -2)) * inside.unsqueeze(1)).matmul(v)
    last = torch.exp(ld.view(-1, 1) * (_CHUNK - 1 - i))
    states = torch.matmul((k * last.view(H, 1, _CHUNK, 1)).transpose(-1, -2), v)
    c = torch.arange(n, device=q.device)
    gap = (c.unsqueeze(1) - c - 1).clamp_min(0) * _CHUNK
    across = torch.exp(ld.view(-1, 1, 1) * gap) * (c.unsqueeze(1) > c)
    before = torch.matmul(across, states.flatten(-2)).view_as(states)
    first = torch.exp(ld.view(-1, 1) * (i + 1))
    return (o + (q * first.view(H, 1, _CHUNK, 1)).matmul(before)).reshape(N, H, T, -1)


def _plain_decay(s):
    ld, c = s["log_decay"], s["scale"]
    dt = s["q"].dtype
    if s["mode"] == "step":
        q, k, v = (s[n].float() for n in "qkv")
        rows = s["slots"].long()
        new = s["state"][rows] * torch.exp(ld).view(-1, 1, 1) + k.unsqueeze(-1) * v.unsqueeze(-2)
        s["next"].index_copy_(0, rows, new)
        return {"o": (c * torch.matmul(q.unsqueeze(-2), new).squeeze(-2)).to(dt), "state": s["next"]}
    # each sequence's tokens side by side, filled up with zeros to whole chunks
    N, H = s["sizes"].shape[0], ld.shape[0]
    T = max(1, -(-s["most"] // _CHUNK)) * _CHUNK
    tokens = s["q"].numel() // (H * s["q"].shape[-1])
    row = torch.arange(tokens, device=ld.device)
    ends = s["sizes"].cumsum(0)
    e = torch.searchsorted(ends, row, right=True)
    t = row - (ends - s["sizes"])[e]
    at = e * T + t

    def spread(x):
        x = x.float().reshape(tokens, H, -1)
        return x.new_zeros((N * T, H, x.shape[-1])).index_copy_(0, at, x).view(N, T, H, -1).transpose(1, 2).contiguous()

    def gather(x, like):
        return x.transpose(1, 2).reshape(N * T, H, -1)[at].reshape(like.shape).to(dt)

    q, k, v = (spread(s[n]) for n in "qkv")
    pos = torch.arange(T, device=ld.device)
    after = torch.exp(ld.view(-1, 1, 1) * (pos + 1).view(1, -1, 1))  # what is left of the first state at a token
    left = (s["sizes"].view(-1, 1) - 1 - pos).clamp_min(0)
    until = torch.exp(ld.view(1, -1, 1, 1) * left.view(N, 1, -1, 1))  # what is left of a token in the last state
    whole = torch.exp(ld.view(1, -1, 1, 1) * s["sizes"].view(-1, 1, 1, 1))
    o = _weighted(q, k, v, ld) * c
    state = torch.matmul((k * until).transpose(-1, -2), v)
    if s["state"] is not None:
        o += c * after * torch.matmul(q, s["state"])
        state += whole * s["state"]
    out = {"o": gather(o, s["v"])}
    if s["mode"] == "infer" or s["state"] is not None:
        out["state"] = state
    if s["mode"] == "train":
        do = spread(s["do"]) * c
        back = lambda a, b, d: _weighted(a.flip(2), b.flip(2), d.flip(2), ld).flip(2)  # noqa: E731
        dq, dk, dv = _weighted(do, v, k, ld), back(v, do, q), back(k, q, do)
        if s["state"] is not None:
            s0, ds = s["state"], s["dstate"]
            dq += after * torch.matmul(do, s0.transpose(-1, -2).contiguous())
            dk += until * torch.matmul(v, ds.transpose(-1, -2).contiguous())
            dv += until * torch.matmul(k, ds)
            out["dstate"] = torch.matmul((q * after).transpose(-1, -2), do) + whole * ds
        out["dq"], out["dk"], out["dv"] = gather(dq, s["q"]), gather(dk, s["k"]), gather(dv, s["v"])
    return out


def _activated(g, act):
    """(act(g), its derivative)."""
    if act == "silu":
        t = torch.sigmoid(g)
        return g * t, t * (1.0 + g * (1.0 - t))
    if act == "gelu":
        below = 0.5 * torch.erfc(-g * math.sqrt(0.5))
        return g * below, below + g * torch.exp(-0.5 * g * g) * math.sqrt(0.5 / math.pi)
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * g * g)


def _plain_gated(s):
    """The rows of each expert side by side, filled up to the most that one has, and batched products."""
    x, w = s["x"].float(), s["w"].float()
    R = x.shape[0]
    w = w.view(-1, *w.shape[-2:])
    E, N = w.shape[0], w.shape[1] // 2
    if E > 1:
        ends, most = s["offsets"].long(), s["most"]
        row = torch.arange(R, device=x.device)
        e = torch.searchsorted(ends, row, right=True)
        at = e * most + row - torch.nn.functional.pad(ends, (1, 0))[e]
    else:
        most, at = R, None

    def spread(t):
        return t.view(1, R, -1) if at is None else t.new_zeros((E * most, t.shape[1])).index_copy_(0, at, t).view(E, most, -1)

    def gather(t):
        return (t.view(R, -1) if at is None else t.reshape(E * most, -1)[at]).to(s["x"].dtype)

    xp = spread(x)
    u = torch.bmm(xp, w.transpose(1, 2).contiguous())
    gate, up = u[..., :N], u[..., N:]
    a, slope = _activated(gate, s["act"])
    out = {"y": gather(a * up)}
    if s["mode"] == "train":
        dy = spread(s["dy"].float())
        du = torch.cat((dy * up * slope, dy * a), -1)
        out["dx"] = gather(torch.bmm(du, w))
        out["dw"] = torch.bmm(du.transpose(1, 2).contiguous(), xp).view(s["w"].shape).to(s["w"].dtype)
    return out


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    e = _SIZE[case["dtype"]]
    train = case["mode"] == "train"
    if case["op"] == "rotary":
        rows = case["R"] * (case["heads"] + case["kv_heads"])
        b = rows * case["D"] * e * 2 + case["R"] * 4
        return {"bytes": b * (1 + train), "flops": rows * case["part"] * 3 * (1 + train)}
    if case["op"] == "gated":
        R, K, N, E = case["R"], case["K"], case["N"], case["E"]
        hit = min(R, E - case["empty"])  # at most so many experts' weights are read
        b = (R * K + hit * 2 * N * K + R * N) * e
        if train:  # dy read; dx and dw (of every expert) written
            b += (R * N + R * K + E * 2 * N * K) * e
        return {"bytes": b, "flops": 2 * R * K * 2 * N * (3 if train else 1)}
    T, H, Dk, Dv = case["tokens"], case["heads"], case["Dk"], case["Dv"]
    states = case["seqs"] * H * Dk * Dv * 4
    b = T * H * (2 * Dk + 2 * Dv) * e
    if case["mode"] == "step":
        return {"bytes": b + 2 * states, "flops": T * H * Dk * Dv * 5}
    # a token's own chunk so far, and the state that it reads and adds to
    flops = T * H * (_CHUNK * (Dk + Dv) + 4 * Dk * Dv)
    if train:  # do read, dq, dk, dv written; three sums like the forward's
        b += T * H * (2 * Dk + 2 * Dv) * e
        flops *= 4
    if case["states"] or not train:
        b += states
    if case["states"]:
        b += states * (3 if train else 1)
    return {"bytes": b, "flops": flops}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "decay": _exact_decay, "gated": _exact_gated}[case["op"]](s)


def _exact_rotary(s):
    """A pair as a complex number times magnitude * exp(i position frequency)."""
    n = s["frequencies"].shape[0]
    angle = torch.outer(s["positions"].double(), s["frequencies"].double())
    turn = torch.polar(torch.full_like(angle, s["magnitude"]), angle).unsqueeze(1)

    def turned(x, turn):
        y = x.double().clone()
        pairs = y[..., :2 * n].unflatten(-1, (n, 2) if s["interleaved"] else (2, n))
        z = torch.view_as_complex((pairs if s["interleaved"] else pairs.transpose(-1, -2)).contiguous()) * turn
        z = torch.view_as_real(z)
        y[..., :2 * n] = (z if s["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        return y

    out = {"q": turned(s["q"], turn), "k": turned(s["k"], turn)}
    if s["mode"] == "train":
        out["dq"], out["dk"] = turned(s["dq"], turn.conj()), turned(s["dk"], turn.conj())
    return out


def _exact_decay(s):
    """Every pair of tokens of a sequence and head by itself, and the states token by token's weight."""
    ld, c = s["log_decay"].double(), s["scale"]
    if s["mode"] == "step":
        state = s["state"].double()
        o = torch.zeros(s["v"].shape, dtype=torch.float64, device=ld.device)
        for r, slot in enumerate(s["slots"].tolist()):
            k, v, q = (s[n][r].double() for n in "kvq")
            state[slot] = torch.exp(ld)[:, None, None] * state[slot] + k[:, :, None] * v[:, None, :]
            o[r] = c * (q[:, :, None] * state[slot]).sum(1)
        return {"o": o, "state": state}
    H = ld.shape[0]
    flat = lambda t: t.reshape(-1, H, t.shape[-1])  # noqa: E731
    q, k, v = (flat(s[n]) for n in "qkv")
    N, Dk, Dv = s["sizes"].shape[0], q.shape[-1], v.shape[-1]
    train, states = s["mode"] == "train", s["state"] is not None
    new = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=ld.device)  # noqa: E731
    o, state = new(*v.shape), new(N, H, Dk, Dv)
    dq, dk, dv, ds0 = new(*q.shape), new(*k.shape), new(*v.shape), new(N, H, Dk, Dv)
    lo = 0
    for n, size in enumerate(s["sizes"].tolist()):
        here = slice(lo, lo + size)
        lo += size
        t = torch.arange(size, dtype=torch.float64, device=ld.device)
        for h in range(H):
            a, b, d = (x[here, h].double() for x in (q, k, v))
            w = torch.exp(ld[h] * (t[:, None] - t).clamp_min(0)).tril_() * c
            last = torch.exp(ld[h] * (size - 1 - t))[:, None]
            o[here, h] = (w * (a @ b.T)) @ d
            state[n, h] = (last * b).T @ d
            first = c * torch.exp(ld[h] * (t + 1))[:, None]
            if states:
                s0 = s["state"][n, h].double()
                o[here, h] += first * (a @ s0)
                state[n, h] += torch.exp(ld[h] * size) * s0
            if train:
                g = flat(s["do"])[here, h].double()
                dp = w * (g @ d.T)
                dq[here, h], dk[here, h], dv[here, h] = dp @ b, dp.T @ a, (w * (a @ b.T)).T @ g
                if states:
                    dsn = s["dstate"][n, h].double()
                    dq[here, h] += first * (g @ s0.T)
                    dk[here, h] += last * (d @ dsn.T)
                    dv[here, h] += last * (b @ dsn)
                    ds0[n, h] = (first * a).T @ g + torch.exp(ld[h] * size) * dsn
    out = {"o": o.view(s["v"].shape)}
    if states or not train:
        out["state"] = state
    if train:
        out.update(dq=dq.view(s["q"].shape), dk=dk.view(s["k"].shape), dv=dv.view(s["v"].shape))
        if states:
            out["dstate"] = ds0
    return out


def _exact_gated(s):
    x, w = s["x"].double(), s["w"]
    w = w.view(-1, *w.shape[-2:])
    E, N = w.shape[0], w.shape[1] // 2
    ends = [x.shape[0]] if E == 1 else s["offsets"].tolist()
    new = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=x.device)  # noqa: E731
    y, dx, dw = new(x.shape[0], N), new(*x.shape), new(*w.shape)
    for e, (lo, hi) in enumerate(zip([0] + ends[:-1], ends)):
        if lo == hi:
            continue
        we, xe = w[e].double(), x[lo:hi]
        g, u = (xe @ we.T).split(N, 1)
        if s["act"] == "silu":
            a = g / (1 + torch.exp(-g))
            slope = 1 / (1 + torch.exp(-g)) + g / (2 * torch.cosh(g / 2)) ** 2
        elif s["act"] == "gelu":
            below = (1 + torch.erf(g / 2 ** 0.5)) / 2
            a, slope = g * below, below + g * torch.exp(-g ** 2 / 2) / (2 * math.pi) ** 0.5
        else:  # 0.5 (1 + tanh z) = 1 / (1 + exp(-2 z))
            z = (2 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3)
            below = 1 / (1 + torch.exp(-2 * z))
            a = g * below
            slope = below + 2 * a * (1 - below) * (2 / math.pi) ** 0.5 * (1 + 0.134145 * g ** 2)
        y[lo:hi] = a * u
        if s["mode"] == "train":
            dy = s["dy"][lo:hi].double()
            du = torch.cat((dy * u * slope, dy * a), 1)
            dx[lo:hi], dw[e] = du @ we, du.T @ xe
    if s["mode"] != "train":
        return {"y": y}
    return {"y": y, "dx": dx, "dw": dw.view(s["w"].shape)}
