"""The operators that mix tokens (``mhc.branch``: rotary, decay attention, gated products) on the GPU against the
float64 oracle (oracle/mixer_oracle.py).

Tolerances are of the terms' magnitudes (the oracle's recurrence of absolute values) and one rounding to the result's type.

Decay attention.  fp32 sums: a result passes through a product over the key dim, one over at most 64 tokens and the state's chain (three
roundings a chunk), the weights through a few more; (2 * 128 + 64 + 4 chunks) * 2^-23 allows for every order.  Operands that are
computed, P and the state, are two bf16 parts for 16-bit types: each is off by 2^-18 at most, of fp16's products of second parts
2^-18 is left out three times: 2^-15 allows for their sum.  In fp32 three parts leave 2^-26.

Gated products are sums of K terms as in test_gpu_branch.py.  What an error in g and u does to y follows from the
slopes of the activations, below 1.2; expf and erfcf are within 2^-21 of their values.  [dg du] is rounded to the type before
its products.
"""

import itertools

import numpy as np
import pytest
import torch

from helpers import to_np
from test_gpu_branch import DT, HALF_ULP, close, rand
from mhc import _mixer, branch
from oracle import mixer_oracle as M

pytestmark = pytest.mark.gpu

DEV = "cuda"


# --------------------------------------------------------------------------
# Rotary positions
# --------------------------------------------------------------------------

def positions_of(R, far, dtype=torch.int32):
    return (torch.arange(R, device=DEV) * 7919 % max(far, 1)).to(dtype)


def check_rotary(q, k, pos, f, inter, mag, dq, dk):
    out = branch.rotary(q, k, pos, f, interleaved=inter, magnitude=mag)
    leaves, outs, grads = ((q,), (out,), (dq,)) if k is None else ((q, k), out, (dq, dk))
    got = torch.autograd.grad(outs, leaves, grads)
    p = np.resize(to_np(pos.reshape(-1)), q.shape[:-2]).reshape(-1) if pos.dim() else np.full(int(np.prod(q.shape[:-2])), int(pos))
    rows = lambda t: to_np(t).reshape(-1, *t.shape[-2:])  # noqa: E731
    for name, y, x, g, d in zip("qk", outs, leaves, got, grads):
        assert y.is_contiguous() and y.shape == x.shape and y.dtype == x.dtype
        ref, size = M.rotary(rows(x), p, to_np(f), inter, mag)
        close(y.flatten(0, -3) if y.dim() > 2 else y[None], ref, size, 2.0 ** -21, name)
        ref, size = M.rotary(rows(d), p, to_np(f), inter, mag, inverse=True)
        close(g.flatten(0, -3) if g.dim() > 2 else g[None], ref, size, 2.0 ** -21, "d" + name)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("R,H,Hk,D,part", [(1, 1, 1, 2, 2), (5, 4, 2, 64, 64), (33, 3, 1, 128, 128), (37, 2, 2, 100, 36),
                                           (9, 5, 1, 80, 40), (7, 2, 1, 33, 10), (3, 1, 1, 7, 6), (1100, 6, 2, 96, 96),
                                           (1030, 3, 3, 58, 50), (4, 2, 2, 256, 2), (6, 2, 2, 40, 0), (2, 1, 1, 4096, 4096)])
def test_rotary(R, H, Hk, D, part, inter, dtype):
    dt = DT[dtype]
    q, k = rand(R, H, D, seed=1, dtype=dt).requires_grad_(), rand(R, Hk, D, seed=2, dtype=dt).requires_grad_()
    f = branch.rotary_frequencies(part, device=DEV)
    check_rotary(q, k, positions_of(R, 5000), f, inter, 1.25, rand(R, H, D, seed=3, dtype=dt), rand(R, Hk, D, seed=4, dtype=dt))


# --------------------------------------------------------------------------
# Decay attention
# --------------------------------------------------------------------------

def decays(H):
    return -torch.exp2(-torch.linspace(0.0, 10.0, H, device=DEV)) if H > 1 else torch.tensor([-0.02], device=DEV)


def decay_tol(dtype, T):
    return (320 + 4 * (T // 64 + 1)) * 2.0 ** -23 + (0.0 if dtype == torch.float32 else 2.0 ** -15)


def check_decay(q, k, v, ld, offsets, first, do, d_last, scale, spans):
    """Output, state and every gradient; q, k, v (rows, H, D) or (B, T, H, D) leaves."""
    with_state = first is not None or d_last is not None
    out = branch.decay_attention(q, k, v, ld, initial_state=first, offsets=offsets, scale=scale, return_state=True)
    leaves = [q, k, v] + ([first] if first is not None else [])
    grads = torch.autograd.grad(out if with_state else out[:1], leaves, (do, d_last) if with_state else (do,))
    rows = lambda t: to_np(t).reshape(-1, *t.shape[-2:])  # noqa: E731
    s = None if first is None else to_np(first)
    g = None if d_last is None or not with_state else to_np(d_last)
    args = (rows(q), rows(k), rows(v))
    mag = lambda *ts: [None if t is None else np.abs(t) for t in ts]  # noqa: E731
    L = to_np(ld)
    o, st = M.decay_attention(*args, L, spans, s, scale)
    so, sst = M.decay_attention(*mag(*args), L, spans, *mag(s), abs(scale))
    ref = M.decay_attention_backward(*args, rows(do), L, spans, s, g, scale)
    size = M.decay_attention_backward(*mag(*args, rows(do)), L, spans, *mag(s, g), abs(scale))
    tol = decay_tol(q.dtype, max([hi - lo for lo, hi in spans] + [1]))
    flat = lambda t: t.reshape(-1, *t.shape[-2:])  # noqa: E731
    close(flat(out[0]), o, so, tol, "o")
    close(out[1], st, sst, decay_tol(torch.float32, max([hi - lo for lo, hi in spans] + [1])), "state")
    for name, got, r, z in zip(("dq", "dk", "dv"), grads, ref, size):
        assert got.dtype == q.dtype
        close(flat(got), r, z, tol, name)
    if first is not None:
        close(grads[3], ref[3], size[3], decay_tol(torch.float32, max([hi - lo for lo, hi in spans] + [1])), "d_first")
    return out


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("B,T,H,Dk,Dv", [(1, 1, 1, 1, 1), (2, 3, 2, 16, 16), (1, 63, 2, 64, 64), (1, 64, 1, 128, 128),
                                         (2, 65, 3, 128, 64), (1, 130, 2, 64, 128), (3, 200, 2, 72, 104), (1, 77, 2, 33, 95),
                                         (2, 129, 1, 7, 121)])
def test_decay_attention(B, T, H, Dk, Dv, dtype):
    dt = DT[dtype]
    q, k = (rand(B, T, H, Dk, seed=i, dtype=dt).requires_grad_() for i in (1, 2))
    v, do = rand(B, T, H, Dv, seed=3, dtype=dt).requires_grad_(), rand(B, T, H, Dv, seed=4, dtype=dt)
    first, d_last = rand(B, H, Dk, Dv, seed=5).requires_grad_(), rand(B, H, Dk, Dv, seed=6)
    spans = [(n * T, (n + 1) * T) for n in range(B)]
    check_decay(q, k, v, decays(H), None, first, do, d_last, Dk ** -0.5, spans)
    check_decay(q, k, v, decays(H), None, None, do, None, 0.3, spans)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("lens,extra", [([5, 0, 70, 1, 64], 9), ([0, 0, 3], 0), ([130], 70), ([1] * 70, 3), ([0, 0], 4)])
@pytest.mark.parametrize("Dk,Dv", [(64, 72), (128, 128), (20, 9)])
def test_decay_attention_packed(lens, extra, Dk, Dv, dtype):
    dt, H = DT[dtype], 2
    R, N = sum(lens) + extra, len(lens)
    off = torch.tensor(np.cumsum(lens), dtype=torch.int32, device=DEV)
    q, k = (rand(R, H, Dk, seed=i, dtype=dt).requires_grad_() for i in (1, 2))
    v, do = rand(R, H, Dv, seed=3, dtype=dt).requires_grad_(), rand(R, H, Dv, seed=4, dtype=dt)
    first, d_last = rand(N, H, Dk, Dv, seed=5).requires_grad_(), rand(N, H, Dk, Dv, seed=6)
    check_decay(q, k, v, decays(H), off, first, do, d_last, Dk ** -0.5, M.spans_of(off.tolist(), R))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("Dk,Dv", [(128, 128), (64, 40)])
def test_decay_attention_in_segments(Dk, Dv, dtype):
    """Long sequences of few heads: several segments each, dense and packed."""
    dt, H, T = DT[dtype], 1, 1500
    q, k = (rand(1, T, H, Dk, seed=i, dtype=dt).requires_grad_() for i in (1, 2))
    v, do = rand(1, T, H, Dv, seed=3, dtype=dt).requires_grad_(), rand(1, T, H, Dv, seed=4, dtype=dt)
    first, d_last = rand(1, H, Dk, Dv, seed=5).requires_grad_(), rand(1, H, Dk, Dv, seed=6)
    for ld in (-0.001, 0.0, -0.3):
        check_decay(q, k, v, torch.tensor([ld], device=DEV), None, first, do, d_last, Dk ** -0.5, [(0, T)])
    off = torch.tensor([20, 1300, 1300, 1490], device=DEV)
    first, d_last = rand(4, H, Dk, Dv, seed=5).requires_grad_(), rand(4, H, Dk, Dv, seed=6)
    check_decay(*(t.detach()[0].requires_grad_() for t in (q, k, v)), torch.tensor([-0.01], device=DEV), off, first, do[0], d_last,
                Dk ** -0.5, M.spans_of(off.tolist(), T))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("Dk,Dv,ends", [(128, 128, None), (64, 40, [8800, 8800, 9290]), (40, 100, [9301]), (100, 70, [30, 9000]),
                                        (72, 72, [7000] + list(range(7001, 7040, 3)))])
def test_decay_attention_in_many_segments(Dk, Dv, ends, dtype):
    """More segments than each adds up for itself."""
    dt, H, T = DT[dtype], 1, 9301
    q, k = (rand(T, H, Dk, seed=i, dtype=dt).requires_grad_() for i in (1, 2))
    v, do = rand(T, H, Dv, seed=3, dtype=dt).requires_grad_(), rand(T, H, Dv, seed=4, dtype=dt)
    spans = [(0, T)] if ends is None else M.spans_of(ends, T)
    N, off = len(spans), None if ends is None else torch.tensor(ends, device=DEV)
    first, d_last = rand(N, H, Dk, Dv, seed=5).requires_grad_(), rand(N, H, Dk, Dv, seed=6)
    ld = torch.tensor([-0.0005], device=DEV)
    if ends is None:
        q, k, v = (t.detach()[None].requires_grad_() for t in (q, k, v))
        do = do[None]
    check_decay(q, k, v, ld, off, first, do, d_last, Dk ** -0.5, spans)
    check_decay(q, k, v, ld, off, None, do, None, Dk ** -0.5, spans)


@pytest.mark.parametrize("Dk,Dv", [(128, 96), (40, 64), (100, 30)])
def test_decay_attention_some_gradients_of_many_segments(Dk, Dv):
    """Each gradient alone and with others, with the forward's states kept and not."""
    H, T = 1, 2700
    q, k, v, do = (rand(1, T, H, d, seed=i, dtype=torch.bfloat16) for i, d in enumerate((Dk, Dk, Dv, Dv)))
    first, d_last = rand(1, H, Dk, Dv, seed=5), rand(1, H, Dk, Dv, seed=6)
    ld = torch.tensor([-0.002], device=DEV)
    args = [to_np(t)[0] for t in (q, k, v, do)]
    states = to_np(first), to_np(d_last)
    ref = M.decay_attention_backward(*args, to_np(ld), [(0, T)], *states, 0.1)
    size = M.decay_attention_backward(*map(np.abs, args), to_np(ld), [(0, T)], *map(np.abs, states), 0.1)
    kept = _mixer.decay_attention_forward(q, k, v, ld, None, first, 0.1, True)[2]
    assert kept is not None
    for need in itertools.product((False, True), repeat=4):
        for states in (kept, None):
            got = _mixer.decay_attention_backward(q, k, v, do, ld, None, first, states, d_last, 0.1, need)
            for g, r, z, n in zip(got, ref, size, need):
                assert (g is not None) == n
                if n:
                    close(g if g.dim() == 4 and g.dtype == torch.float32 else g[0], r, z, decay_tol(g.dtype, T), str(need))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("R,pool,H,Dk,Dv", [(1, 1, 1, 1, 1), (3, 5, 2, 128, 128), (4, 4, 3, 64, 72), (5, 9, 2, 33, 95), (300, 310, 1, 16, 8)])
def test_decay_attention_step(R, pool, H, Dk, Dv, dtype):
    dt = DT[dtype]
    q, k, v = rand(R, H, Dk, seed=1, dtype=dt), rand(R, H, Dk, seed=2, dtype=dt), rand(R, H, Dv, seed=3, dtype=dt)
    state, ld = rand(pool, H, Dk, Dv, seed=4, scale=3.0), decays(H)
    g = torch.Generator().manual_seed(7)
    for slots in (None, torch.randperm(pool, generator=g)[:R].int().to(DEV), torch.randint(-2, pool + 2, (R,), generator=g).to(DEV)):
        at = list(range(R)) if slots is None else slots.tolist()
        o, st = M.decay_step(*(to_np(t) for t in (q, k, v, ld, state)), at, Dk ** -0.5)
        so, sst = M.decay_step(*(np.abs(to_np(t)) for t in (q, k, v)), to_np(ld), np.abs(to_np(state)), at, Dk ** -0.5)
        tol = (Dk + 8 + 2 * R) * 2.0 ** -23  # a sum over the key dim; a rounding or two a token of a slot
        mine, apart = state.clone(), state.clone()
        got = branch.decay_attention_step(q, k, v, ld, mine, slots=slots)
        close(got, o, so, tol, "o")
        close(mine, st, sst, tol, "state")
        again = branch.decay_attention_step(q, k, v, ld, state, slots=slots, state_out=apart)
        assert torch.equal(again, got) and torch.equal(apart, mine)
        untouched = [i for i in range(pool) if i not in at]
        assert torch.equal(mine[untouched], state[untouched])


# --------------------------------------------------------------------------
# Gated products
# --------------------------------------------------------------------------

def check_gated(x, w, off, act, dy):
    """y, dx and dw; off None or a list of ends."""
    t = None if off is None else torch.tensor(off, dtype=torch.int32, device=DEV)
    y = branch.gated_matmul(x, w, t, activation=act)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    with torch.no_grad():
        assert torch.equal(branch.gated_matmul(x, w, t, activation=act), y)
    (R, K), N = x.shape, w.shape[-2] // 2
    w3, ends = to_np(w).reshape(-1, 2 * N, K), [R] if off is None else off
    ref, g, u, sg, su = M.gated_matmul(to_np(x), w3, ends, act)
    a, slope = M.activation(g, act)
    e = (K + 8) * 2.0 ** -23  # of each product's terms
    size = np.abs(u) * 1.2 * sg + np.abs(a) * su
    close(y, ref, size * e + np.abs(ref) * 2.0 ** -20 + np.abs(u * g) * 2.0 ** -24 + e * e * sg * su, 1.0, "y")
    rx, rw, d = M.gated_matmul_backward(to_np(dy), to_np(x), w3, ends, act)
    # [dg du]: errors of g and u (the slopes' own slopes are below 1.2, too), the functions' and one rounding
    dyn = np.abs(to_np(dy))
    ed = np.concatenate((dyn * (np.abs(slope) * su + np.abs(u) * 1.2 * sg + e * sg * su), dyn * 1.2 * sg), 1) * e
    fn = np.concatenate((dyn * np.abs(u) * (1.0 + np.abs(g)), dyn * np.abs(g)), 1) * 2.0 ** -20
    half = 0.0 if x.dtype == torch.float32 else HALF_ULP[x.dtype]
    ed = ed + fn + half * np.abs(d) + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    sx, sw = np.zeros(rx.shape), np.zeros(rw.shape)
    for i, lo, hi in M.groups(ends, R):
        sx[lo:hi] = ed[lo:hi] @ np.abs(w3[i]) + (2 * N + 8) * 2.0 ** -23 * (np.abs(d[lo:hi]) @ np.abs(w3[i]))
        sw[i] = ed[lo:hi].T @ np.abs(to_np(x)[lo:hi]) + (R + 8) * 2.0 ** -23 * (np.abs(d[lo:hi]).T @ np.abs(to_np(x)[lo:hi]))
    close(dx, rx, sx, 1.01, "dx")
    close(dw.reshape(w3.shape), rw, sw, 1.01, "dw")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("R,K,N", [(1, 64, 16), (8, 96, 40), (7, 33, 21), (70, 128, 200), (65, 1, 1), (300, 200, 130), (129, 77, 65)])
def test_gated_matmul(R, K, N, act, dtype):
    dt = DT[dtype]
    x, w = rand(R, K, seed=1, dtype=dt).requires_grad_(), rand(2 * N, K, seed=2, dtype=dt, scale=2 * K ** -0.5).requires_grad_()
    check_gated(x, w, None, act, rand(R, N, seed=3, dtype=dt))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("R,K,N,E,off", [
    (60, 64, 40, 9, [5, 5, 20, 31, 30, 44, 44, 50, 57]),   # few rows an expert, some without, rows of none
    (60, 65, 41, 9, [0, 0, 20, 31, 33, 44, 44, 50, 60]),
    (700, 128, 96, 3, [300, 300, 690]), (700, 130, 97, 3, [1, 2, 700]),
])
def test_gated_matmul_of_experts(R, K, N, E, off, dtype):
    dt = DT[dtype]
    x = rand(R, K, seed=1, dtype=dt).requires_grad_()
    w = rand(E, 2 * N, K, seed=2, dtype=dt, scale=K ** -0.5).requires_grad_()
    check_gated(x, w, off, "silu", rand(R, N, seed=3, dtype=dt))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("R,K,N,off", [
    (1000, 64, 2100, None), (1100, 40, 2000, [400, 390, 1090]),      # 128-tiles
    (3000, 64, 2864, None), (2900, 72, 2800, [1500, 1500, 2890]),    # 256-tiles with quarters and half tiles
    (1500, 35, 2901, None),                                          # unaligned 128-tiles
])
def test_gated_matmul_large_tiles(R, K, N, off, dtype):
    dt = DT[dtype]
    x = rand(R, K, seed=1, dtype=dt).requires_grad_()
    w = rand(*(() if off is None else (len(off),)), 2 * N, K, seed=2, dtype=dt, scale=K ** -0.5).requires_grad_()
    check_gated(x, w, off, "silu", rand(R, N, seed=3, dtype=dt))
