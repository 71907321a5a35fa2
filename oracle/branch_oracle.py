"""float64 restatement of the operators inside a branch (``mhc.branch``), numpy only."""

import numpy as np

MX_MAX = 448.0  # largest e4m3 value
MX_BLOCK = 32


def rms_norm(h, w=None, eps=1e-6):
    """(y, rstd) of rows h (..., D)."""
    h = np.asarray(h, np.float64)
    r = 1.0 / np.sqrt((h * h).mean(-1) + eps)
    y = h * r[..., None]
    return (y if w is None else y * np.asarray(w, np.float64)), r


def rms_norm_backward(dy, h, dh=None, w=None, eps=1e-6):
    """(dx, dw) and bounds of the sums of their terms' magnitudes, for rows (R, D)."""
    dy, h = np.asarray(dy, np.float64), np.asarray(h, np.float64)
    n, r = rms_norm(h, None, eps)
    g = dy if w is None else dy * np.asarray(w, np.float64)
    r = r[:, None]
    dx = r * (g - n * (g * n).mean(-1, keepdims=True))
    size = r * (np.abs(g) + np.abs(n) * np.abs(g * n).mean(-1, keepdims=True))
    if dh is not None:
        dx = dx + np.asarray(dh, np.float64)
        size = size + np.abs(dh)
    return dx, (dy * n).sum(0), size, np.abs(dy * n).sum(0)


def mx_exponent(amax):
    """Exponent of the smallest power of two that brings amax to 448 or below, -127 at least."""
    amax = np.asarray(amax, np.float64)
    with np.errstate(divide="ignore"):
        m, e = np.frexp(amax)  # amax = m 2^e; 448 = 0.875 * 2^9
    k = e - 9 + (m > 0.875)
    return np.where(amax == 0, -127, np.maximum(k, -127))


def mx_exponents(x):
    """Exponents (..., D / 32) of rows (..., D)."""
    x = np.abs(np.asarray(x, np.float64))
    return mx_exponent(x.reshape(*x.shape[:-1], -1, MX_BLOCK).max(-1))


def e4m3_round(v):
    """Nearest e4m3 value (ties to even) of |v| <= 448."""
    v = np.asarray(v, np.float64)
    step = np.exp2(np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -6))) - 3)
    return np.round(v / step) * step


def philox(counter_lo, counter_hi, offset, seed, rounds=10):
    """Four uint32 arrays: Philox4x32 of the counters (lo, hi, offset lo, offset hi) under the key seed."""
    m32 = (1 << 32) - 1
    lo = np.asarray(counter_lo, np.uint64)
    c = [lo & np.uint64(m32), np.asarray(counter_hi, np.uint64) + lo * 0,
         lo * 0 + np.uint64(offset & m32), lo * 0 + np.uint64(offset >> 32)]
    k0, k1 = seed & m32, seed >> 32
    for _ in range(rounds):
        p = np.uint64(0xD2511F53) * c[0]
        q = np.uint64(0xCD9E8D57) * c[2]
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), q & np.uint64(m32),
             (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p & np.uint64(m32)]
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    return [x.astype(np.uint32) for x in c]


def dropout_factors(n, p, seed, offset, first=0):
    """What elements first .. first + n - 1 (first a multiple of 8) are multiplied by."""
    call = np.arange(first // 8, first // 8 + (n + 7) // 8, dtype=np.uint64)
    words = philox(call & np.uint64((1 << 32) - 1), call >> np.uint64(32), offset, seed)
    u = np.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], 1).reshape(-1)[:n]
    kept = int(np.rint((1.0 - p) * 65536))
    return np.where(u < kept, 65536.0 / kept if kept else 0.0, 0.0)


def groups(offsets, rows):
    """[(expert, lo, hi)]: offsets count clamped to [0, rows] and as their running maximum."""
    out, lo = [], 0
    for e, hi in enumerate(offsets):
        hi = max(lo, min(int(hi), rows))
        out.append((e, lo, hi))
        lo = hi
    return out


def grouped_matmul(x, w, offsets):
    """y (R, N) and the sums of its terms' magnitudes."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    y = np.zeros((x.shape[0], w.shape[1]))
    size = np.zeros_like(y)
    for e, lo, hi in groups(offsets, x.shape[0]):
        y[lo:hi] = x[lo:hi] @ w[e].T
        size[lo:hi] = np.abs(x[lo:hi]) @ np.abs(w[e].T)
    return y, size


def grouped_matmul_backward(dy, x, w, offsets):
    """(dx, dw) and the sums of their terms' magnitudes."""
    dy, x, w = (np.asarray(t, np.float64) for t in (dy, x, w))
    dx, dw = np.zeros(x.shape), np.zeros(w.shape)
    sx, sw = np.zeros(x.shape), np.zeros(w.shape)
    for e, lo, hi in groups(offsets, x.shape[0]):
        dx[lo:hi] = dy[lo:hi] @ w[e]
        sx[lo:hi] = np.abs(dy[lo:hi]) @ np.abs(w[e])
        dw[e] = dy[lo:hi].T @ x[lo:hi]
        sw[e] = np.abs(dy[lo:hi].T) @ np.abs(x[lo:hi])
    return dx, dw, sx, sw
