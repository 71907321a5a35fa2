"""float64 restatement of the operators that mix tokens (``mhc.branch``), numpy only.

Each result comes with its size: the same expression of its terms' magnitudes, which bounds what rounding can do.
"""

import numpy as np

from .branch_oracle import groups


def rotary(x, positions, frequencies, interleaved=False, magnitude=1.0, inverse=False):
    """Rows (R, heads, D) with the first 2 * len(frequencies) elements turned, and the size."""
    x = np.asarray(x, np.float64)
    f = np.asarray(frequencies, np.float64)
    n = f.shape[0]
    t = np.outer(np.asarray(positions, np.float64), f)[:, None, :] * (-1.0 if inverse else 1.0)
    y, size = x.copy(), np.abs(x)
    ia = np.arange(0, 2 * n, 2) if interleaved else np.arange(n)
    ib = ia + 1 if interleaved else ia + n
    a, b, c, s = x[..., ia], x[..., ib], np.cos(t), np.sin(t)
    y[..., ia], y[..., ib] = magnitude * (a * c - b * s), magnitude * (a * s + b * c)
    size[..., ia] = size[..., ib] = abs(magnitude) * (np.abs(a) + np.abs(b))
    return y, size


def decay_attention(q, k, v, log_decay, spans, first=None, scale=1.0):
    """(o, states) of rows (R, H, D), token by token; spans: [(lo, hi)] of the sequences.  Rows of none are zeros."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    l = np.exp(np.minimum(np.asarray(log_decay, np.float64), 0.0))[:, None, None]
    N, H, Dk, Dv = len(spans), q.shape[1], q.shape[2], v.shape[2]
    o, states = np.zeros(v.shape), np.zeros((N, H, Dk, Dv))
    for n, (lo, hi) in enumerate(spans):
        s = np.zeros((H, Dk, Dv)) if first is None else np.array(first[n], np.float64)
        for t in range(lo, hi):
            s = l * s + k[t][:, :, None] * v[t][:, None, :]
            o[t] = scale * np.einsum("hd,hde->he", q[t], s)
        states[n] = s
    return o, states


def decay_attention_backward(q, k, v, do, log_decay, spans, first=None, d_last=None, scale=1.0):
    """(dq, dk, dv, d_first): the recurrence's derivative, from the last token to the first."""
    q, k, v, do = (np.asarray(t, np.float64) for t in (q, k, v, do))
    l = np.exp(np.minimum(np.asarray(log_decay, np.float64), 0.0))[:, None, None]
    N, H, Dk, Dv = len(spans), q.shape[1], q.shape[2], v.shape[2]
    dq, dk, dv, d_first = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape), np.zeros((N, H, Dk, Dv))
    for n, (lo, hi) in enumerate(spans):
        s = np.zeros((H, Dk, Dv)) if first is None else np.array(first[n], np.float64)
        for t in range(lo, hi):
            s = l * s + k[t][:, :, None] * v[t][:, None, :]
            dq[t] = scale * np.einsum("he,hde->hd", do[t], s)
        g = np.zeros((H, Dk, Dv)) if d_last is None else np.array(d_last[n], np.float64)
        for t in range(hi - 1, lo - 1, -1):
            g = g + scale * q[t][:, :, None] * do[t][:, None, :]
            dk[t] = np.einsum("hde,he->hd", g, v[t])
            dv[t] = np.einsum("hde,hd->he", g, k[t])
            g = l * g
        d_first[n] = g
    return dq, dk, dv, d_first


def spans_of(offsets, rows):
    return [(lo, hi) for _, lo, hi in groups(offsets, rows)]


def decay_step(q, k, v, log_decay, state, slots, scale=1.0):
    """(o, states): rows in order; a slot outside the pool gives zeros."""
    state = np.array(state, np.float64)
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    l = np.exp(np.minimum(np.asarray(log_decay, np.float64), 0.0))[:, None, None]
    o = np.zeros(v.shape)
    for r, slot in enumerate(slots):
        if 0 <= slot < state.shape[0]:
            state[slot] = l * state[slot] + k[r][:, :, None] * v[r][:, None, :]
            o[r] = scale * np.einsum("hd,hde->he", q[r], state[slot])
    return o, state


def _erf(x):
    from math import erf

    return np.vectorize(erf, otypes=[np.float64])(x)


def activation(g, name):
    """(act(g), act'(g))."""
    g = np.asarray(g, np.float64)
    with np.errstate(over="ignore"):
        if name == "silu":
            s = 1.0 / (1.0 + np.exp(-g))
            return g * s, s * (1.0 + g * (1.0 - s))
        if name == "gelu":
            s = 0.5 * (1.0 + _erf(g / np.sqrt(2.0)))
            return g * s, s + g * np.exp(-0.5 * g * g) / np.sqrt(2.0 * np.pi)
        c = np.sqrt(2.0 / np.pi)
        t = np.tanh(c * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g * g)


def gated_matmul(x, w, offsets, name):
    """y and, for the bounds: g, u and the sums of their terms' magnitudes; w (E, 2 N, K)."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    R, N = x.shape[0], w.shape[1] // 2
    g, u, sg, su = (np.zeros((R, N)) for _ in range(4))
    for e, lo, hi in groups(offsets, R):
        g[lo:hi], u[lo:hi] = x[lo:hi] @ w[e, :N].T, x[lo:hi] @ w[e, N:].T
        sg[lo:hi], su[lo:hi] = np.abs(x[lo:hi]) @ np.abs(w[e, :N].T), np.abs(x[lo:hi]) @ np.abs(w[e, N:].T)
    return activation(g, name)[0] * u, g, u, sg, su


def gated_matmul_backward(dy, x, w, offsets, name):
    """(dx, dw, [dg du])."""
    dy, x, w = (np.asarray(t, np.float64) for t in (dy, x, w))
    _, g, u, _, _ = gated_matmul(x, w, offsets, name)
    a, slope = activation(g, name)
    d = np.concatenate((dy * u * slope, dy * a), 1)
    dx, dw = np.zeros(x.shape), np.zeros(w.shape)
    for e, lo, hi in groups(offsets, x.shape[0]):
        dx[lo:hi], dw[e] = d[lo:hi] @ w[e], d[lo:hi].T @ x[lo:hi]
    return dx, dw, d
