"""The operators that mix tokens (``mhc.branch``) without a GPU: the oracle's pins, frequencies, refusals, the C ABI's
host-side checks, and the torch.library fakes."""

import math

import numpy as np
import pytest
import torch

from mhc import _mixer, branch
from oracle import mixer_oracle as M

BF, F32 = torch.bfloat16, torch.float32


# --------------------------------------------------------------------------
# The oracle
# --------------------------------------------------------------------------

def test_oracle_rotary_is_a_complex_product():
    r = np.random.default_rng(0)
    x, pos, f = r.standard_normal((5, 2, 10)), np.array([0, 1, 7, 100, -3]), np.array([1.0, 0.3, 0.01])
    turn = 1.5 * np.exp(1j * np.outer(pos, f))[:, None]
    for inter in (False, True):
        y, _ = M.rotary(x, pos, f, inter, 1.5)
        pick = (lambda t: (t[..., 0:6:2], t[..., 1:6:2])) if inter else (lambda t: (t[..., :3], t[..., 3:6]))
        (a, b), (c, d) = pick(x), pick(y)
        assert np.allclose((a + 1j * b) * turn, c + 1j * d, rtol=1e-14, atol=1e-14) and np.array_equal(y[..., 6:], x[..., 6:])
        back, _ = M.rotary(y, pos, f, inter, 1 / 1.5, inverse=True)
        assert np.allclose(back, x, rtol=1e-13, atol=1e-13)


def test_oracle_decay_attention_is_the_weighted_sum_over_pairs():
    r = np.random.default_rng(1)
    q, k, v = r.standard_normal((9, 2, 3)), r.standard_normal((9, 2, 3)), r.standard_normal((9, 2, 4))
    first, ld = r.standard_normal((2, 2, 3, 4)), np.array([-0.3, 0.5])
    spans = [(0, 5), (5, 8)]
    o, s = M.decay_attention(q, k, v, ld, spans, first, 0.7)
    for n, (lo, hi) in enumerate(spans):
        for h, l in enumerate(np.exp(np.minimum(ld, 0))):
            for t in range(lo, hi):
                want = sum(l ** (t - u) * (q[t, h] @ k[u, h]) * v[u, h] for u in range(lo, t + 1))
                want = want + l ** (t - lo + 1) * q[t, h] @ first[n, h]
                assert np.allclose(o[t, h], 0.7 * want, rtol=1e-12, atol=1e-12)
            want = sum(l ** (hi - 1 - u) * np.outer(k[u, h], v[u, h]) for u in range(lo, hi)) + l ** (hi - lo) * first[n, h]
            assert np.allclose(s[n, h], want, rtol=1e-12, atol=1e-12)
    assert not o[8].any()
    # a step is one more token
    o2, s2 = M.decay_step(q[8:], k[8:], v[8:], ld, s, [1], 0.7)
    oo, ss = M.decay_attention(q, k, v, ld, [(0, 5), (5, 9)], first, 0.7)
    assert np.allclose(o2[0], oo[8]) and np.allclose(s2, ss)


def test_oracle_gradients_against_differences():
    r = np.random.default_rng(2)
    q, k = r.standard_normal((2, 9, 2, 3))
    v, do = r.standard_normal((2, 9, 2, 4))
    first, d_last = r.standard_normal((2, 3, 2, 3, 4))
    ld, spans = np.array([-0.3, -0.01]), [(0, 4), (4, 4), (4, 8)]

    def loss(*a):
        o, s = M.decay_attention(*a[:3], ld, spans, a[3], 0.7)
        return (o * do).sum() + (s * d_last).sum()

    args = [q, k, v, first]
    for i, g in enumerate(M.decay_attention_backward(q, k, v, do, ld, spans, first, d_last, 0.7)):
        e, t = r.standard_normal(args[i].shape), 1e-5
        up, down = ([a + s * t * e if j == i else a for j, a in enumerate(args)] for s in (1, -1))
        assert abs((loss(*up) - loss(*down)) / (2 * t) - (g * e).sum()) < 1e-8, i
    x, w, dy = r.standard_normal((6, 4)), r.standard_normal((2, 6, 4)), r.standard_normal((6, 3))
    for act in ("silu", "gelu", "gelu_tanh"):
        dx, dw, _ = M.gated_matmul_backward(dy, x, w, [2, 5], act)
        f = lambda x, w: (M.gated_matmul(x, w, [2, 5], act)[0] * dy).sum()  # noqa: E731
        ex, ew, t = r.standard_normal(x.shape), r.standard_normal(w.shape), 1e-5
        assert abs((f(x + t * ex, w) - f(x - t * ex, w)) / (2 * t) - (dx * ex).sum()) < 1e-8
        assert abs((f(x, w + t * ew) - f(x, w - t * ew)) / (2 * t) - (dw * ew).sum()) < 1e-8
        assert not dx[5].any()


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_oracle_activations_are_torchs(act):
    g = torch.linspace(-12, 12, 97, dtype=torch.float64, requires_grad=True)
    y = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g, approximate="tanh" if act == "gelu_tanh" else "none")
    slope, = torch.autograd.grad(y.sum(), g)
    a, s = M.activation(g.detach().numpy(), act)
    assert np.allclose(a, y.detach().numpy(), atol=1e-14) and np.allclose(s, slope.numpy(), atol=1e-14)


# --------------------------------------------------------------------------
# Frequencies
# --------------------------------------------------------------------------

def test_rotary_frequencies():
    f = branch.rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,)
    assert torch.allclose(f, torch.tensor([10000.0 ** (-i / 32) for i in range(32)], dtype=torch.float64), rtol=1e-14)
    assert torch.equal(branch.rotary_frequencies(64, factor=4.0), f / 4)
    assert branch.rotary_frequencies(0).shape == (0,) and branch.rotary_frequencies(2).tolist() == [1.0]
    # by parts: those that turn often over the trained length stay, those that hardly turn are divided, none rises
    g = branch.rotary_frequencies(64, factor=8.0, original_length=4096)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(g[turns > 40], f[turns > 40])
    assert torch.allclose(g[turns < 0.7], f[turns < 0.7] / 8, rtol=1e-12)
    assert bool((g <= f).all()) and bool((g >= f / 8 * (1 - 1e-12)).all()) and bool((g[1:] < g[:-1]).all())
    assert torch.equal(branch.rotary_frequencies(64, factor=1.0, original_length=4096), f)
    for bad in (dict(dim=7), dict(dim=8, base=0.0), dict(dim=8, factor=-1.0), dict(dim=8, factor=2.0, original_length=0),
                dict(dim=8, factor=2.0, original_length=64, fast=1.0, slow=2.0)):
        with pytest.raises(ValueError):
            branch.rotary_frequencies(**bad)


# --------------------------------------------------------------------------
# Refusals
# --------------------------------------------------------------------------

def _refusals():
    q, v = torch.zeros(2, 4, 3, 16), torch.zeros(2, 4, 3, 8)
    k, ld = q, torch.zeros(3)
    p, f = torch.zeros(4, dtype=torch.int32), torch.zeros(8, dtype=torch.float64)
    s = torch.zeros(2, 3, 16, 8)
    off = torch.zeros(2, dtype=torch.int32)
    x, w = torch.zeros(4, 6), torch.zeros(10, 6)
    rot = lambda **a: branch.rotary(**{**dict(q=q, k=k, positions=p, frequencies=f), **a})  # noqa: E731
    att = lambda **a: branch.decay_attention(**{**dict(q=q, k=k, v=v, log_decay=ld), **a})  # noqa: E731
    one = lambda **a: branch.decay_attention_step(  # noqa: E731
        **{**dict(q=q[0], k=k[0], v=v[0], log_decay=ld, state=torch.zeros(4, 3, 16, 8)), **a})
    gat = lambda *a, **b: branch.gated_matmul(*a, **b)  # noqa: E731
    wide = torch.zeros(1, 4, 3, 129)
    return [
        ("q dims", AssertionError, lambda: rot(q=torch.zeros(16))),
        ("k lead", AssertionError, lambda: rot(k=q[:1])),
        ("k dim", AssertionError, lambda: rot(k=q[..., :8])),
        ("k type", TypeError, lambda: rot(k=q.to(BF))),
        ("positions shape", AssertionError, lambda: rot(positions=p[:2])),
        ("positions lead", AssertionError, lambda: rot(positions=torch.zeros(2, dtype=torch.int32))),
        ("positions type", TypeError, lambda: rot(positions=p.float())),
        ("too many pairs", AssertionError, lambda: rot(frequencies=torch.zeros(9, dtype=torch.float64))),
        ("frequencies dims", AssertionError, lambda: rot(frequencies=f[None])),
        ("frequencies type", TypeError, lambda: rot(frequencies=f.long())),
        ("wide heads", AssertionError, lambda: rot(q=torch.zeros(2, 4, 1, 4098), k=None)),
        ("frequencies' gradient", RuntimeError, lambda: rot(frequencies=f.clone().requires_grad_())),
        ("q and k", AssertionError, lambda: att(k=q[:, :3])),
        ("v lead", AssertionError, lambda: att(v=v[:, :3])),
        ("v type", TypeError, lambda: att(v=v.to(BF))),
        ("wide key", AssertionError, lambda: att(q=wide, k=wide, v=v[:1])),
        ("wide value", AssertionError, lambda: att(q=q[:1], k=q[:1], v=wide)),
        ("decay count", AssertionError, lambda: att(log_decay=ld[:2])),
        ("decay type", TypeError, lambda: att(log_decay=ld.long())),
        ("decay's gradient", RuntimeError, lambda: att(log_decay=ld.clone().requires_grad_())),
        ("state shape", AssertionError, lambda: att(initial_state=s[:1])),
        ("state type", TypeError, lambda: att(initial_state=s.to(BF))),
        ("packed dims", AssertionError, lambda: att(offsets=off)),
        ("unpacked dims", AssertionError, lambda: att(q=q[0], k=k[0], v=v[0])),
        ("packed state", AssertionError, lambda: att(q=q[0], k=k[0], v=v[0], offsets=off, initial_state=s[:1])),
        ("step dims", AssertionError, lambda: one(q=q, k=k, v=v)),
        ("step state", AssertionError, lambda: one(state=torch.zeros(4, 3, 8, 16))),
        ("step state type", TypeError, lambda: one(state=torch.zeros(4, 3, 16, 8, dtype=BF))),
        ("step state strides", AssertionError, lambda: one(state=torch.zeros(4, 3, 8, 16).transpose(2, 3))),
        ("too few states", AssertionError, lambda: one(state=torch.zeros(3, 3, 16, 8))),
        ("slots count", AssertionError, lambda: one(slots=torch.zeros(3, dtype=torch.int32))),
        ("slots type", TypeError, lambda: one(slots=torch.zeros(4))),
        ("state_out", AssertionError, lambda: one(state_out=torch.zeros(5, 3, 16, 8))),
        ("step's gradient", RuntimeError, lambda: one(q=q[0].clone().requires_grad_())),
        ("activation", ValueError, lambda: gat(x, w, activation="relu")),
        ("odd weight", AssertionError, lambda: gat(x, w[:9])),
        ("weight dims", AssertionError, lambda: gat(x, w[None])),
        ("weight dims of experts", AssertionError, lambda: gat(x, w, off)),
        ("in width", AssertionError, lambda: gat(x[:, :5], w)),
        ("weight type", TypeError, lambda: gat(x, w.to(BF))),
        ("offsets count", AssertionError, lambda: _mixer._offsets(off, 3)),
    ]


@pytest.mark.parametrize("i", range(41))
def test_refusals(i):
    cases = _refusals()
    assert len(cases) == 41
    name, error, call = cases[i]
    with pytest.raises(error):
        call()


def test_cpu_tensors_are_refused():
    q, s = torch.zeros(2, 4, 3, 16), torch.zeros(4, 3, 16, 16)
    for call in (lambda: branch.rotary(q, q, torch.zeros(4, dtype=torch.int32), torch.zeros(8)),
                 lambda: branch.decay_attention(q, q, q, torch.zeros(3)),
                 lambda: branch.decay_attention_step(q[0], q[0], q[0], torch.zeros(3), s),
                 lambda: branch.gated_matmul(torch.zeros(2, 4), torch.zeros(6, 4))):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


def test_abi_refusals_before_any_device_work():
    from mhc import _lib

    lib = _lib.load()
    rot = lambda q=16, out=16, H=2, k=None, Hk=0, code=1, pos=16, count=4, f=16, pairs=4, R=4, D=8: lib.mhc_rotary(  # noqa: E731
        q, H * D, D, out, H, k, Hk * D, D, k, Hk, code, pos, 0, count, f, pairs, R, D, 1.0, 0, 0, None)
    assert rot(q=None) == rot(out=None) == rot(pos=None) == rot(f=None) == rot(Hk=1) == rot(count=0) == 1
    assert rot(pairs=5) == rot(R=-1) == rot(D=4098, pairs=4) == rot(H=65537) == 1
    assert b"rotary" in lib.mhc_last_error()
    assert rot(R=0, q=None) == rot(H=0, q=None) == 0 and rot(code=7) == 2

    def fwd(q=16, off=None, o=16, last=None, R=8, N=2, H=2, Dk=16, Dv=16, code=1, ws=None, nb=0, row=32, ld=16):
        return lib.mhc_decay_attention_forward(q, row, 16, 16, row, 16, 16, row, 16, code, ld, off, None, o, last, R, N, H, Dk, Dv,
                                               1.0, ws, nb, None)

    assert fwd(q=None) == fwd(o=None) == fwd(ld=None) == fwd(R=7) == fwd(Dk=129) == fwd(Dv=0) == fwd(R=-8) == 1
    assert fwd(row=(1 << 22) + 1) == fwd(row=-1) == fwd(R=1 << 31, N=1) == 1
    assert fwd(R=0, q=None, o=None) == fwd(H=0, q=None) == fwd(R=0, N=0) == 0 and fwd(code=3) == 2
    need = lib.mhc_decay_attention_workspace_bytes(8192, 1, 2, 64, 64, 0, 1)
    assert need > 0 and need % (2 * 64 * 64 * 4) == 0 and lib.mhc_decay_attention_workspace_bytes(64, 1, 2, 64, 64, 0, 1) == 0
    assert fwd(R=8192, N=1, Dk=64, Dv=64) == fwd(R=8192, N=1, Dk=64, Dv=64, ws=16, nb=need - 1) == 3

    def bwd(do=16, R=8, N=2, Dk=16, Dv=16, code=1, row=32):
        return lib.mhc_decay_attention_backward(16, row, 16, 16, row, 16, 16, row, 16, do, row, 16, code, 16, None, None, None, None, 16,
                                                16, 16, None, R, N, 2, Dk, Dv, 1.0, None, 0, None)

    assert bwd(do=None) == bwd(R=7) == bwd(Dk=200) == bwd(row=(1 << 22) + 1) == 1
    assert bwd(R=0, do=None) == 0 and bwd(code=9) == 2 and bwd(R=8192, N=1) == 3

    def step(q=16, slots=16, state=16, R=4, pool=4, Dk=16, Dv=16, code=1):
        return lib.mhc_decay_attention_step(q, 32, 16, 16, 32, 16, 16, 32, 16, code, 16, slots, state, state, 16, R, pool, 2, Dk, Dv,
                                            1.0, None)

    assert step(q=None) == step(state=None) == step(slots=None, pool=3) == step(Dk=129) == step(R=-1) == 1
    assert step(R=0, q=None) == 0 and step(code=5) == 2

    def gated(x=16, w=16, code=1, off=16, act=0, y=16, R=4, K=8, N=8, E=2):
        return lib.mhc_gated_matmul_forward(x, w, code, off, act, y, None, R, K, N, E, None)

    assert gated(x=None) == gated(w=None) == gated(y=None) == gated(off=None) == gated(act=3) == gated(N=-1) == 1
    assert gated(E=4097) == gated(N=(1 << 19) + 1) == gated(R=1 << 31) == 1
    assert gated(R=0, x=None) == gated(N=0, w=None) == 0 and gated(code=4) == 2

    def gated_bwd(dy=16, saved=16, x=16, w=16, dx=16, dw=16, ws=16, nb=1 << 20, R=4, N=8, off=16, E=2):
        return lib.mhc_gated_matmul_backward(dy, saved, x, w, 1, off, 0, dx, dw, R, 8, N, E, ws, nb, None)

    assert gated_bwd(dy=None) == gated_bwd(saved=None) == gated_bwd(x=None) == gated_bwd(w=None) == gated_bwd(off=None) == 1
    assert gated_bwd(ws=None) == gated_bwd(nb=4 * 16 * 2 - 1) == 3 and lib.mhc_gated_matmul_backward_workspace_bytes(4, 8, 1) == 128
    assert gated_bwd(dx=None, dw=None, dy=None) == 0


# --------------------------------------------------------------------------
# torch.library
# --------------------------------------------------------------------------

OPS = {"rotary", "decay_attention", "decay_attention_backward", "decay_attention_step", "decay_attention_step_out",
       "gated_matmul", "gated_matmul_backward"}


def test_every_launcher_is_registered():
    assert {n for n in dir(torch.ops.mhc_mixer) if not n.startswith("_") and n != "name"} == OPS
    for n in OPS:
        assert torch._C._dispatch_has_kernel_for_dispatch_key(f"mhc_mixer::{n}", "CUDA"), n
        assert not torch._C._dispatch_has_kernel_for_dispatch_key(f"mhc_mixer::{n}", "CPU"), n


def test_fakes_and_traced_gradients():
    """Meta tensors through the traced functions: every gradient has its input's shape and dtype."""
    from mhc import _mixer_library as L

    e = lambda *s, dt=BF: torch.empty(*s, device="meta", dtype=dt).requires_grad_(dt in (BF, F32))  # noqa: E731
    like = lambda ts: [(t.shape, t.dtype) for t in ts]  # noqa: E731
    q, k, v = e(2, 5, 3, 16), e(2, 5, 1, 16), e(2, 5, 3, 8)
    p, f, ld = e(5, dt=torch.int32), e(8, dt=torch.float64), e(3, dt=F32).detach()
    a, b = L.rotary(q, k, p, f, False, 1.0)
    assert like((a, b)) == like((q, k)) == like(torch.autograd.grad(a.sum() + b.sum(), (q, k)))
    assert L.rotary(q, None, p, f, True, 1.0).shape == q.shape
    s = e(2, 3, 16, 8, dt=F32)
    o, last = L.decay_attention(q, q, v, ld, None, s, 1.0)
    assert like((o, last)) == like((v, s))
    assert like(torch.autograd.grad(o.sum() + last.sum(), (q, v, s))) == like((q, v, s))
    o, last = L.decay_attention(q[0], q[0], v[0], ld, e(4, dt=torch.int32), None, 1.0)
    assert last.shape == (4, 3, 16, 8) and like(torch.autograd.grad(o.sum(), (q, v))) == like((q, v))
    with torch.no_grad():
        assert L.decay_attention_step(q[0], q[0], v[0], ld, e(9, 3, 16, 8, dt=F32), None, 1.0, None).shape == (5, 3, 8)
    x = e(6, 16)
    for w, off in ((e(24, 16), None), (e(3, 24, 16), e(3, dt=torch.int32))):
        y = L.gated_matmul(x, w, off, "gelu")
        assert y.shape == (6, 12) and like(torch.autograd.grad(y.sum(), (x, w))) == like((x, w))


def test_decay_workspace_holds_the_states_of_segments_alone():
    """Segments with a successor leave a state, at most one for every 256 tokens, however many sequences share them.  Many
    sequences have a table, 16 bytes for each segment and at most as many again."""
    from mhc import _lib

    lib = _lib.load()
    for R, H, Dk, Dv in ((16384, 32, 128, 128), (65536, 1, 40, 100), (3069, 12, 100, 72)):
        for of, times in ((lib.mhc_decay_attention_workspace_bytes, 1), (lib.mhc_decay_attention_backward_workspace_bytes, 2)):
            for N in (1, 64, 512, 2048, 100000):
                assert 0 < of(R, N, H, Dk, Dv, 1, 1) <= times * (R - 1) // 256 * H * Dk * Dv * 4 + 32 * (R // 256 + N + 1)


def test_decay_backward_workspace_with_the_forwards_states_kept():
    """Half the workspace of a backward that makes them again; it is checked before the dtype, and both before the device."""
    from mhc import _lib

    lib = _lib.load()

    def bwd(kept, ws, nb, Dk=64, Dv=64):
        return lib.mhc_decay_attention_backward(16, 128, 64, 16, 128, 64, 16, 128, 64, 16, 128, 64, 9, 16, None, None, kept, None, 16,
                                                16, 16, None, 8192, 1, 2, Dk, Dv, 1.0, ws, nb, None)

    for Dk, Dv in ((64, 64), (40, 100)):
        states = lib.mhc_decay_attention_workspace_bytes(8192, 1, 2, Dk, Dv, 0, 1)
        assert lib.mhc_decay_attention_backward_workspace_bytes(8192, 1, 2, Dk, Dv, 0, 1) == 2 * states > 0
        assert bwd(None, 16, 2 * states, Dk, Dv) == 2 and bwd(None, 16, 2 * states - 1, Dk, Dv) == 3
        assert bwd(16, 16, states, Dk, Dv) == 2 and bwd(16, 16, states - 1, Dk, Dv) == bwd(16, None, 0, Dk, Dv) == 3


@pytest.mark.parametrize("dim,length", [(64, 4096), (64, 65536), (128, 131072), (32, 131072), (16, 10 ** 6), (8, 10 ** 9),
                                        (64, 128), (64, 20), (64, 4), (2, 30)])
@pytest.mark.parametrize("fast,slow", [(32.0, 1.0), (9.0, 2.5)])
def test_rotary_frequencies_between_fast_and_slow(dim, length, fast, slow):
    """The share of a pair that turns between slow and fast times over the trained length is between none and all and linear in
    its index, whether or not there are pairs at the ramp's ends; beyond them frequencies are divided, or stay."""
    f = branch.rotary_frequencies(dim)
    share = (1 - branch.rotary_frequencies(dim, factor=8.0, original_length=length, fast=fast, slow=slow) / f) / (1 - 1 / 8)
    turns = length * f / (2 * math.pi)
    # a share is a quotient of fp64 roundings: 1 - 1/8 .. 1 of 2^-53 each
    assert bool((share[turns >= fast].abs() < 1e-14).all()) and bool(((share[turns <= slow] - 1).abs() < 1e-14).all())
    ramp = share[(turns > slow) & (turns < fast)]
    assert bool((ramp > 1e-6).all()) and bool((ramp < 1 - 1e-6).all())
    assert ramp.numel() < 3 or bool(((ramp.diff().diff()).abs() < 1e-14).all())
