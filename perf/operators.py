"""The operators of a hyper-connection's branch (``mhc.branch``), as cases that can be timed and checked.

A branch between ``HyperConnection``'s branch input and its closure normalises its input, multiplies the
tokens that a router has sorted by expert with their experts' weights, and in training drops out parts of
its output.  ``op`` names the operator of a case:

* ``norm``     ``rms_norm`` with or without the residual's addition: forward alone ("infer"), forward and
               backward ("train"), or ``rms_norm_mx``, whose output is in 8 bits with a power-of-two
               scale for every 32 values ("mx").
* ``experts``  ``grouped_matmul`` over rows sorted by expert, some experts without any, or
               ``grouped_matmul_mx`` on 8-bit rows and weights ("mx").
* ``dropout``  ``dropout`` with or without the residual's addition, from a seed and an offset.

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
_EPS = 1e-6
_F8 = torch.float8_e4m3fn
_E8 = torch.float8_e8m0fnu


def _norm(name, R, D, dtype, mode, residual):
    return {"name": name, "op": "norm", "R": R, "D": D, "dtype": dtype, "mode": mode, "residual": residual}


def _experts(name, R, K, N, E, dtype, mode, empty=0):
    return {"name": name, "op": "experts", "R": R, "K": K, "N": N, "E": E, "empty": empty, "dtype": dtype,
            "mode": mode}


def _dropout(name, R, D, dtype, mode, residual, p=0.1):
    return {"name": name, "op": "dropout", "R": R, "D": D, "dtype": dtype, "mode": mode, "residual": residual, "p": p}


def listed():
    return [
        # one decoded token: latency is all there is
        _norm("norm decode", 1, 4096, "bf16", "infer", True),
        # the headline workload's tokens (batch 4, sequence 4096), forward and backward
        _norm("norm train", 16384, 4096, "bf16", "train", True),
        # a width that is not a whole number of 16-byte vectors, and an odd length (3 sequences of 1023)
        _norm("norm ragged", 3069, 1500, "fp16", "train", False),
        # a long prompt at the widest dim, into the 8-bit products of its experts
        _norm("norm 8 bits", 8192, 7168, "bf16", "mx", True),
        # the README's example size in fp32: a small experiment
        _dropout("dropout small", 256, 512, "fp32", "train", False),
        # the headline workload's tokens, with the residual's addition
        _dropout("dropout train", 16384, 4096, "bf16", "train", True),
        # a batch of 16 decoded tokens with 4 experts each: bound by reading the weights that are hit
        _experts("experts decode", 64, 2048, 4096, 32, "bf16", "infer", empty=4),
        # the headline workload's tokens over 8 experts, forward and both gradients
        _experts("experts train", 16384, 4096, 4096, 8, "bf16", "train"),
        # odd lengths, widths that are not whole vectors, experts without tokens
        _experts("experts ragged", 3069, 1500, 1001, 12, "fp16", "train", empty=3),
        # a small experiment in fp32
        _experts("experts small fp32", 256, 512, 2048, 4, "fp32", "train"),
        # 32 decoded tokens with 4 experts each, weights in 8 bits
        _experts("experts 8 bits decode", 128, 4096, 4096, 32, "bf16", "mx", empty=2),
        # a long prompt at the widest dim over 16 experts, in 8 bits
        _experts("experts 8 bits prefill", 8192, 7168, 2048, 16, "bf16", "mx"),
    ]


def _log(rng, lo, hi):
    v = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return v + 1 if v == 3072 else v


def _width(rng, lo, hi, unit=8, any_share=0.25):
    """A width: mostly whole 16-byte vectors, now and then any number."""
    v = _log(rng, lo, hi)
    if rng.random() >= any_share:
        v = max(unit, v // unit * unit)
    return v + unit if v == 3072 else v


def _draw_any(rng):
    op = rng.choice(["norm", "norm", "experts", "experts", "experts", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    residual = rng.random() < 0.5
    if op == "norm":
        mode = rng.choice(["infer", "train", "train", "mx"])
        if mode == "mx":
            D = _width(rng, 64, 8192, 32, 0.0)
        else:
            D = _width(rng, 64, 8192)
        return {"op": op, "R": _log(rng, 1, 32768), "D": D, "dtype": dtype, "mode": mode, "residual": residual}
    if op == "dropout":
        return {"op": op, "R": _log(rng, 1, 32768), "D": _width(rng, 64, 8192), "dtype": dtype,
                "mode": rng.choice(["infer", "train", "train"]), "residual": residual,
                "p": round(rng.uniform(0.02, 0.5), 3)}
    mode = rng.choice(["infer", "train", "mx"])
    E = _log(rng, 2, 64)
    if mode == "mx":
        K, N = _width(rng, 128, 8192, 32, 0.0), _width(rng, 64, 8192)
        dtype = rng.choice(["bf16", "bf16", "fp16"])
    else:
        K, N = _width(rng, 64, 8192), _width(rng, 64, 8192)
    return {"op": op, "R": _log(rng, 1, 16384), "K": K, "N": N, "E": E, "empty": rng.randint(0, E // 3),
            "dtype": dtype, "mode": mode}


def draw(rng):
    top = [work(c) for c in listed()]
    while True:
        case = _draw_any(rng)
        w = work(case)
        # a matrix product in 32 bits costs about 16 times one in 16 bits
        flops = w["flops"] * (16 if case["op"] == "experts" and case["dtype"] == "fp32" else 1)
        weights = case["op"] == "experts" and case["E"] * case["K"] * case["N"]
        if (w["bytes"] <= max(t["bytes"] for t in top) and flops <= max(t["flops"] for t in top)
                and weights <= 1 << 28):
            return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _randn(shape, g, dtype, scale=1.0):
    t = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    return (t.mul_(scale) if scale != 1.0 else t).to(dtype)


def _sizes(R, E, empty, seed):
    """Rows of each expert as a router leaves them: a few times more at one than at another, some without any."""
    r = np.random.RandomState(seed % (1 << 32))
    share = np.exp(0.5 * r.standard_normal(E))
    share[r.permutation(E)[:empty]] = 0.0
    return r.multinomial(R, share / share.sum())


def _quantised(t):
    """(values in 8 bits, scales) of rows whose width is a multiple of 32; scale rows are filled up to a
    multiple of 4 with the smallest scale."""
    b = t.float().reshape(*t.shape[:-1], -1, 32)
    top = b.abs().amax(-1)
    m, e = torch.frexp(top)  # top = m 2^e <= 448 2^k = 0.875 2^(k + 9)
    k = torch.where(top > 0, (e - 9 + (m > 0.875)).float(), -127.0).clamp(-127, 127)
    q = (b * torch.exp2(-k).unsqueeze(-1)).to(_F8).reshape(t.shape)
    k = torch.nn.functional.pad(k, (0, -k.shape[-1] % 4), value=-127.0)
    return q, (k + 127).to(torch.uint8).view(_E8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _DT[case["dtype"]]
    mode = case["mode"]
    train = mode == "train"
    s = {"op": case["op"], "mode": mode}
    if case["op"] == "experts":
        R, K, N, E = case["R"], case["K"], case["N"], case["E"]
        sizes = _sizes(R, E, case["empty"], int(seed))
        s["most"] = int(sizes.max())
        s["offsets"] = torch.tensor(np.cumsum(sizes), dtype=torch.int32, device="cuda")
        x = _randn((R, K), g, dtype)
        w = _randn((E, N, K), g, dtype, K ** -0.5)
        if mode == "mx":
            s["dtype"] = dtype
            s["x"], s["xs"] = _quantised(x)
            s["w"], s["ws"] = _quantised(w)
            return s
        s["x"], s["w"] = x.requires_grad_(train), w.requires_grad_(train)
        if train:
            s["dy"] = _randn((R, N), g, dtype)
        return s
    R, D = case["R"], case["D"]
    # a few channels are much larger than the rest, as in trained models' hidden states
    x = torch.randn((R, D), generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn((D,), generator=g, device="cuda"))
    s["x"] = x.to(dtype).requires_grad_(train)
    if case["residual"]:
        s["res"] = _randn((R, D), g, dtype, 2.0).requires_grad_(train)
    if train:
        s["dy"] = _randn((R, D), g, dtype)
    if case["op"] == "dropout":
        s["p"] = case["p"]
        s["rng"] = (int(seed) * 0x9E3779B97F4A7C15 % (1 << 63), int(seed) % 1000)
        return s
    s["w"] = (1.0 + 0.2 * torch.randn((D,), generator=g, device="cuda")).requires_grad_(train)
    if train and case["residual"]:
        s["dh"] = _randn((R, D), g, dtype)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"norm": _plain_norm, "experts": _plain_experts, "dropout": _plain_dropout}[s["op"]](s)


def _run_own(s):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from mhc import branch

    train = s["mode"] == "train"
    with torch.set_grad_enabled(train):
        if s["op"] == "norm":
            res = s.get("res")
            if s["mode"] == "mx":
                out = branch.rms_norm_mx(s["x"], s["w"], residual=res, eps=_EPS)
                return dict(zip(("q", "scales", "h"), out))
            out = branch.rms_norm(s["x"], s["w"], residual=res, eps=_EPS)
            if res is None:
                if not train:
                    return {"y": out}
                dx, dw = torch.autograd.grad(out, (s["x"], s["w"]), s["dy"])
                return {"y": out, "dx": dx, "dw": dw}
            y, h = out
            if not train:
                return {"y": y, "h": h}
            dx, dres, dw = torch.autograd.grad((y, h), (s["x"], res, s["w"]), (s["dy"], s["dh"]))
            return {"y": y, "h": h, "dx": dx, "dres": dres, "dw": dw}
        if s["op"] == "experts":
            if s["mode"] == "mx":
                return {"y": branch.grouped_matmul_mx(s["x"], s["xs"], s["w"], s["ws"], s["offsets"],
                                                      out_dtype=s["dtype"])}
            y = branch.grouped_matmul(s["x"], s["w"], s["offsets"])
            if not train:
                return {"y": y}
            dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
            return {"y": y, "dx": dx, "dw": dw}
        res = s.get("res")
        y = branch.dropout(s["x"], s["p"], s["rng"], residual=res)
        if not train:
            return {"y": y}
        if res is None:
            return {"y": y, "dx": torch.autograd.grad(y, (s["x"],), s["dy"])[0]}
        dx, dres = torch.autograd.grad(y, (s["x"], res), s["dy"])
        return {"y": y, "dx": dx, "dres": dres}


def _plain_norm(s):
    x, w = s["x"], s["w"]
    h = x if "res" not in s else (x.float() + s["res"].float()).to(x.dtype)
    hf = h.float()
    r = torch.rsqrt((hf * hf).mean(-1, keepdim=True) + _EPS)
    n = hf * r
    y = n * w
    if s["mode"] == "mx":
        q, scales = _quantised(y)
        out = {"q": q, "scales": scales}
        if "res" in s:
            out["h"] = h
        return out
    out = {"y": y.to(x.dtype)}
    if "res" in s:
        out["h"] = h
    if s["mode"] == "train":
        dy = s["dy"].float()
        gw = dy * w
        dx = r * (gw - n * (gw * n).mean(-1, keepdim=True))
        if "res" in s:
            dx += s["dh"].float()
        out["dx"] = dx.to(x.dtype)
        if "res" in s:
            out["dres"] = out["dx"]
        out["dw"] = (dy * n).sum(0)
    return out


def _values(q, scales):
    """The 32-bit values that 8-bit rows and their scales stand for."""
    n = q.shape[-1] // 32
    k = scales.view(torch.uint8)[..., :n].float() - 127.0
    return (q.float().reshape(*q.shape[:-1], n, 32) * torch.exp2(k).unsqueeze(-1)).reshape(q.shape)


def _plain_experts(s):
    """The rows of each expert side by side, filled up to the most that one has, and one batched product."""
    ends, most = s["offsets"].long(), s["most"]
    mx = s["mode"] == "mx"
    x = _values(s["x"], s["xs"]) if mx else s["x"].float()
    w = _values(s["w"], s["ws"]) if mx else s["w"].float()
    R, E = x.shape[0], w.shape[0]
    row = torch.arange(R, device=x.device)
    e = torch.searchsorted(ends, row, right=True)
    at = e * most + row - torch.nn.functional.pad(ends, (1, 0))[e]
    xp = x.new_zeros((E * most, x.shape[1])).index_copy_(0, at, x).view(E, most, -1)
    y = torch.bmm(xp, w.transpose(1, 2).contiguous()).view(E * most, -1)[at]
    out = {"y": y.to(s["dtype"] if mx else s["x"].dtype)}
    if s["mode"] == "train":
        dy = s["dy"].float()
        dyp = dy.new_zeros((E * most, dy.shape[1])).index_copy_(0, at, dy).view(E, most, -1)
        out["dx"] = torch.bmm(dyp, w).view(E * most, -1)[at].to(s["x"].dtype)
        out["dw"] = torch.bmm(dyp.transpose(1, 2).contiguous(), xp).to(s["w"].dtype)
    return out


def _words(count, rng, device):
    """Four 32-bit words for each counter 0 .. count - 1 (Philox4x32, ten rounds), in 64-bit integers."""
    low = 0xFFFFFFFF
    seed, offset = rng
    i = torch.arange(count, device=device)
    a, b = i & low, i >> 32
    c, d = torch.full_like(i, offset & low), torch.full_like(i, offset >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        p, q = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = ((q >> 32) & low) ^ b ^ k0, q & low, ((p >> 32) & low) ^ d ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((a, b, c, d), 1)


def _plain_dropout(s):
    x = s["x"]
    n = x.numel()
    words = _words((n + 7) // 8, s["rng"], x.device)
    u = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:n].view(x.shape)
    kept = round((1.0 - s["p"]) * 65536)
    factor = (u < kept).float() * (65536.0 / kept)
    y = x.float() * factor
    if "res" in s:
        y += s["res"].float()
    out = {"y": y.to(x.dtype)}
    if s["mode"] == "train":
        out["dx"] = (s["dy"].float() * factor).to(x.dtype)
        if "res" in s:
            out["dres"] = s["dy"]
    return out


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    e = _SIZE[case["dtype"]]
    train = case["mode"] == "train"
    mx = case["mode"] == "mx"
    if case["op"] == "experts":
        R, K, N, E = case["R"], case["K"], case["N"], case["E"]
        hit = min(R, E - case["empty"])  # at most so many experts' weights are read
        flops = 2 * R * K * N * (3 if train else 1)
        if mx:
            per = 1 + 1 / 32
            return {"bytes": (R * K + hit * K * N) * per + R * N * e, "flops": flops}
        b = (R * K + hit * K * N + R * N) * e
        if train:  # dy read; dx and dw (of every expert) written
            b += (R * N + R * K + E * K * N) * e
        return {"bytes": b, "flops": flops}
    n = case["R"] * case["D"]
    res = bool(case["residual"])
    if case["op"] == "dropout":
        b = n * e * (2 + res)
        if train:  # dy read, dx written
            b += n * e * 2
        return {"bytes": b, "flops": n * (1 + res + train)}
    if mx:
        b = n * (e * (1 + 2 * res) + 1 + 1 / 32)
    else:
        b = n * e * (2 + 2 * res)
        if train:  # dy and dh read, dx written
            b += n * e * (2 + res)
    return {"bytes": b + case["D"] * 4 * (1 + train), "flops": n * (4 + res + (8 if train else 0))}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            return _exact_norm(s)
        if case["op"] == "experts":
            return _exact_experts(s)
        return _exact_dropout(s)


def _exact_norm(s):
    """The definition's values before they are rounded to their types: y = w h / rms(h) of the stored sum h,
    its derivatives from the quotient rule, and for 8 bits y over its block's scale."""
    dt = s["x"].dtype
    x, w = s["x"].double(), s["w"].double()
    out = {}
    if "res" in s:
        out["h"] = x + s["res"].double()
        x = out["h"].to(dt).double()
    D = x.shape[1]
    ms = torch.linalg.vector_norm(x, dim=1).square() / D + _EPS
    rms = ms.sqrt().unsqueeze(1)
    y = w * (x / rms)
    if s["mode"] == "mx":
        blocks = y.unflatten(1, (-1, 32))
        top = blocks.abs().max(-1).values
        # smallest power of two that brings the block's largest magnitude to 448 or below
        m, k = torch.frexp(top / 448.0)
        k = torch.where(m == 0.5, k - 1, k).clamp_min(-127)
        q = torch.ldexp(blocks, -k.double().unsqueeze(-1)).flatten(1)
        scales = torch.exp2(k.double())
        fill = -scales.shape[1] % 4
        if fill:
            scales = torch.cat((scales, scales.new_full((scales.shape[0], fill), 2.0 ** -127)), 1)
        return {"q": q, "scales": scales, **out}
    out = {"y": y, **out}
    if s["mode"] == "train":
        dy = s["dy"].double()
        # d(1/rms)/dx_i = -x_i / (D rms^3)
        along = ((dy * w) * x).sum(1, keepdim=True)
        dx = dy * w / rms - x * along / (D * rms.pow(3))
        if "res" in s:
            dx = dx + s["dh"].double()
            out["dres"] = dx
        out["dx"] = dx
        out["dw"] = (dy * x / rms).sum(0)
    return out


def _exact_experts(s):
    mx = s["mode"] == "mx"
    x, w = s["x"], s["w"]
    if mx:  # each value times its block's scale
        def values(q, k):
            k = torch.exp2(k.view(torch.uint8).double() - 127).repeat_interleave(32, -1)
            return q.double() * k[..., :q.shape[-1]]
        x = values(x, s["xs"])
    ends = s["offsets"].tolist()
    y = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.float64, device=x.device)
    out = {"y": y}
    if s["mode"] == "train":
        out["dx"] = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
        out["dw"] = torch.zeros(w.shape, dtype=torch.float64, device=x.device)
    for e, (lo, hi) in enumerate(zip([0] + ends[:-1], ends)):
        if lo == hi:
            continue
        we = values(w[e], s["ws"][e]) if mx else w[e].double()
        xe = x[lo:hi].double()
        y[lo:hi] = xe @ we.T
        if s["mode"] == "train":
            de = s["dy"][lo:hi].double()
            out["dx"][lo:hi] = de @ we
            out["dw"][e] = de.T @ xe
    return out


def _exact_dropout(s):
    x = s["x"]
    n = x.numel()
    seed, offset = s["rng"]
    blocks = (n + 7) // 8
    index = np.arange(blocks, dtype=np.uint64)
    ctr = [index.astype(np.uint32), (index >> np.uint64(32)).astype(np.uint32),
           np.full(blocks, offset % 2 ** 32, np.uint32), np.full(blocks, offset // 2 ** 32, np.uint32)]
    key = np.array([seed % 2 ** 32, seed // 2 ** 32], np.uint64)
    for rnd in range(10):
        k = ((key + np.uint64(rnd) * np.array([0x9E3779B9, 0xBB67AE85], np.uint64)) % np.uint64(2 ** 32)).astype(np.uint32)
        p0 = ctr[0].astype(np.uint64) * np.uint64(0xD2511F53)
        p1 = ctr[2].astype(np.uint64) * np.uint64(0xCD9E8D57)
        ctr = [(p1 >> np.uint64(32)).astype(np.uint32) ^ ctr[1] ^ k[0], p1.astype(np.uint32),
               (p0 >> np.uint64(32)).astype(np.uint32) ^ ctr[3] ^ k[1], p0.astype(np.uint32)]
    u = np.ascontiguousarray(np.stack(ctr, 1)).view("<u2").reshape(-1)[:n]
    kept = round((1.0 - s["p"]) * 65536)
    keep = torch.from_numpy(u < kept).to(x.device).view(x.shape)
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    y = torch.where(keep, x.double() * 65536 / kept, zero)
    out = {"y": y + s["res"].double() if "res" in s else y}
    if s["mode"] == "train":
        out["dx"] = torch.where(keep, s["dy"].double() * 65536 / kept, zero)
        if "res" in s:
            out["dres"] = s["dy"].double()
    return out
