"""The operators that mix tokens on the GPU, beside test_gpu_mixer.py: how they are called rather than what they compute."""

import numpy as np
import pytest
import torch

from helpers import to_np
from test_gpu_branch import DT, close, rand
from test_gpu_mixer import check_decay, check_gated, check_rotary, decay_tol, decays, positions_of
from test_gpu_native_nodes import both, same
from test_mixer_cpu import OPS
from mhc import _mixer, branch
from oracle import mixer_oracle as M

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF = torch.bfloat16


def leaf(*shape, seed, dtype=torch.float32, scale=1.0):
    return rand(*shape, seed=seed, dtype=dtype, scale=scale).requires_grad_()


# --------------------------------------------------------------------------
# C++ and Python nodes, torch.compile, registrations
# --------------------------------------------------------------------------

def _steps(dt):
    """name -> a step of each operator that returns everything it makes."""
    pos, f = positions_of(12, 900), branch.rotary_frequencies(16, device=DEV)
    q4, k4, v4 = leaf(3, 12, 2, 24, seed=1, dtype=dt), leaf(3, 12, 2, 24, seed=2, dtype=dt), leaf(3, 12, 2, 20, seed=3, dtype=dt)
    k1 = leaf(3, 12, 1, 24, seed=4, dtype=dt)
    ld, s3, s2 = decays(2), leaf(3, 2, 24, 20, seed=5), leaf(2, 2, 24, 20, seed=6)
    off = torch.tensor([5, 30], device=DEV)
    g = lambda t, seed: rand(*t.shape, seed=seed, dtype=t.dtype)  # noqa: E731
    x, w, we = leaf(30, 40, seed=7, dtype=dt), leaf(24, 40, seed=8, dtype=dt), leaf(2, 24, 40, seed=9, dtype=dt)

    def grads(outs, leaves):
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, [g(o, 20 + i) for i, o in enumerate(outs)])]

    def step():
        state = s3.detach().clone()
        with torch.no_grad():
            o = branch.decay_attention_step(q4[:, 0], k4[:, 0], v4[:, 0], ld, state, slots=torch.tensor([2, 0, 2], device=DEV))
        return [o, state]

    def packed(state):
        flat = [t.flatten(0, 1) for t in (q4, k4, v4)]
        o = branch.decay_attention(*flat, ld, initial_state=s2, offsets=off, return_state=state)
        return grads(o if state else (o,), [q4, k4, v4, s2])

    return {
        "rotary": lambda: grads(branch.rotary(q4, k1, pos, f, magnitude=1.3), [q4, k1]),
        "rotary alone": lambda: grads((branch.rotary(q4, None, pos, f, interleaved=True),), [q4]),
        "decay": lambda: grads((branch.decay_attention(q4, k4, v4, ld),), [q4, k4, v4]),
        "decay some": lambda: grads((branch.decay_attention(q4.detach(), k4, v4.detach(), ld, scale=0.5),), [k4]),
        "decay state": lambda: grads(branch.decay_attention(q4, k4, v4, ld, initial_state=s3, return_state=True), [q4, k4, v4, s3]),
        "decay packed": lambda: packed(False),
        "decay packed state": lambda: packed(True),
        "step": step,
        "gated": lambda: grads((branch.gated_matmul(x, w),), [x, w]),
        "gated experts": lambda: grads((branch.gated_matmul(x, we, off, activation="gelu"),), [x, we]),
        "gated weight": lambda: grads((branch.gated_matmul(x.detach(), w, activation="gelu_tanh"),), [w]),
    }


STEPS = ["rotary", "rotary alone", "decay", "decay some", "decay state", "decay packed",
         "decay packed state", "step", "gated", "gated experts", "gated weight"]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("name", STEPS)
def test_nodes_agree(monkeypatch, name, dtype):
    got, want = both(monkeypatch, _steps(DT[dtype])[name])
    same(got, want)


def test_forward_alone_gives_the_same_bits():
    for dt in DT.values():
        q, k, v = leaf(2, 70, 2, 64, seed=1, dtype=dt), leaf(2, 70, 2, 64, seed=2, dtype=dt), leaf(2, 70, 2, 72, seed=3, dtype=dt)
        ld, pos, f = decays(2), positions_of(70, 70), branch.rotary_frequencies(64, device=DEV)
        with torch.no_grad():
            a, (b, c) = branch.decay_attention(q, k, v, ld), branch.rotary(q, k, pos, f)
        assert torch.equal(branch.decay_attention(q, k, v, ld), a)
        assert all(torch.equal(x, y) for x, y in zip(branch.rotary(q, k, pos, f), (b, c)))


@pytest.mark.parametrize("name", ["rotary", "decay", "decay state", "decay packed state", "gated", "gated experts"])
@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_compiled(name, backend):
    """Traced calls give the eager bits, forward and backward."""
    dt = BF
    pos, f, ld = positions_of(12, 900), branch.rotary_frequencies(16, device=DEV), decays(2)
    q, k, v = leaf(3, 12, 2, 24, seed=1, dtype=dt), leaf(3, 12, 2, 24, seed=2, dtype=dt), leaf(3, 12, 2, 20, seed=3, dtype=dt)
    s, off = leaf(3, 2, 24, 20, seed=5), torch.tensor([5, 9, 30], dtype=torch.int32, device=DEV)
    x, w, we = leaf(30, 40, seed=7, dtype=dt), leaf(24, 40, seed=8, dtype=dt), leaf(3, 24, 40, seed=9, dtype=dt)
    call, leaves = {
        "rotary": (lambda q, k: branch.rotary(q, k, pos, f), (q, k)),
        "decay": (lambda q, k, v: (branch.decay_attention(q, k, v, ld),), (q, k, v)),
        "decay state": (lambda q, k, v, s: branch.decay_attention(q, k, v, ld, initial_state=s, return_state=True), (q, k, v, s)),
        "decay packed state": (lambda q, k, v, s: branch.decay_attention(
            q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), ld, initial_state=s, offsets=off, return_state=True), (q, k, v, s)),
        "gated": (lambda x, w: (branch.gated_matmul(x, w),), (x, w)),
        "gated experts": (lambda x, w: (branch.gated_matmul(x, w, off, activation="gelu"),), (x, we)),
    }[name]
    torch._dynamo.reset()
    want, got = call(*leaves), torch.compile(call, fullgraph=True, backend=backend)(*leaves)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    gs = [rand(*o.shape, seed=30, dtype=o.dtype) for o in want]
    for i, (a, b) in enumerate(zip(torch.autograd.grad(got, leaves, gs), torch.autograd.grad(want, leaves, gs))):
        # traced calls always make the state, with three parts of weighted V instead of two
        close(a, to_np(b), np.abs(to_np(b)).max(), 2.0 ** -7 if "decay" in name else 0.0, str(i))
    torch._dynamo.reset()


def test_compiled_step_moves_the_state():
    q, k, v = rand(3, 2, 24, seed=1), rand(3, 2, 24, seed=2), rand(3, 2, 20, seed=3)
    ld, slots = decays(2), torch.tensor([4, 0, 1], dtype=torch.int32, device=DEV)
    a, b = rand(5, 2, 24, 20, seed=4), rand(5, 2, 24, 20, seed=4)
    out = torch.empty_like(a)
    torch._dynamo.reset()
    with torch.no_grad():
        want = branch.decay_attention_step(q, k, v, ld, a, slots=slots)
        f = torch.compile(lambda s: branch.decay_attention_step(q, k, v, ld, s, slots=slots), fullgraph=True, backend="aot_eager")
        assert torch.equal(f(b), want) and torch.equal(a, b)
        out.copy_(b)
        g = torch.compile(lambda s, o: branch.decay_attention_step(q, k, v, ld, s, slots=slots, state_out=o), fullgraph=True,
                          backend="aot_eager")
        again = branch.decay_attention_step(q, k, v, ld, a, slots=slots)
        assert torch.equal(g(b, out), again) and torch.equal(out, a)
    torch._dynamo.reset()


def _registered():
    rg = lambda t: t.clone().requires_grad_()  # noqa: E731
    q, k, v = rand(2, 5, 2, 8, seed=1), rand(2, 5, 2, 8, seed=2), rand(2, 5, 2, 12, seed=3)
    pos, f, ld = positions_of(5, 50), branch.rotary_frequencies(8, device=DEV), decays(2)
    s, off = rand(2, 2, 8, 12, seed=4), torch.tensor([3, 9], dtype=torch.int32, device=DEV)
    x, w, we, dy = rand(6, 16, seed=5), rand(8, 16, seed=6), rand(2, 8, 16, seed=7), rand(6, 4, seed=8)
    eo = torch.tensor([2, 5], dtype=torch.int32, device=DEV)
    y, saved = _mixer.gated_matmul_forward(x, w, None, "silu")
    flat = lambda t: t.flatten(0, 1)  # noqa: E731
    return [
        ("rotary", (rg(q), rg(k), pos, f, False, 1.5, False)), ("rotary", (rg(q), None, pos, f, True, 1.0, True)),
        ("decay_attention", (rg(q), rg(k), rg(v), ld, None, rg(s), 0.5)),
        ("decay_attention", (rg(flat(q)), rg(flat(k)), rg(flat(v)), ld, off, None, 0.5)),
        ("decay_attention_backward", (q, k, v, v, ld, None, s, s, 0.5, [True, True, True, True])),
        ("decay_attention_backward", (flat(q), flat(k), flat(v), flat(v), ld, off, None, None, 0.5, [False, True, False, False])),
        ("decay_attention_step", (q[0], k[0], v[0], ld, rand(6, 2, 8, 12, seed=9), eo[[0, 1, 0, 0, 1]] - 1, 0.5)),
        ("decay_attention_step_out", (q[0], k[0], v[0], ld, rand(6, 2, 8, 12, seed=9), None, 0.5, rand(6, 2, 8, 12, seed=10))),
        ("gated_matmul", (rg(x), rg(w), None, "silu", True)), ("gated_matmul", (rg(x), rg(we), eo, "gelu", True)),
        ("gated_matmul_backward", (dy, saved, x, w, None, "silu", True, True)),
        ("gated_matmul_backward", (dy, saved, x, we, eo, "silu", False, True)),
    ]


@pytest.mark.parametrize("i", range(12))
def test_opcheck(i):
    cases = _registered()
    assert len(cases) == 12 and {n for n, _ in cases} == OPS
    name, args = cases[i]
    torch.library.opcheck(getattr(torch.ops.mhc_mixer, name).default, args,
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic"))


@pytest.mark.parametrize("name", ["rotary", "decay", "decay state", "gated"])
def test_second_derivatives_raise(monkeypatch, name):
    q, k, v = leaf(1, 5, 2, 8, seed=1), leaf(1, 5, 2, 8, seed=2), leaf(1, 5, 2, 8, seed=3)
    s, x, w = leaf(1, 2, 8, 8, seed=4), leaf(6, 16, seed=5), leaf(8, 16, seed=6)
    pos, f, ld = positions_of(5, 50), branch.rotary_frequencies(8, device=DEV), decays(2)

    def step():
        call, leaves = {
            "rotary": (lambda: branch.rotary(q, k, pos, f), (q, k)),
            "decay": (lambda: (branch.decay_attention(q, k, v, ld),), (q, k, v)),
            "decay state": (lambda: branch.decay_attention(q, k, v, ld, initial_state=s, return_state=True), (q, k, v, s)),
            "gated": (lambda: (branch.gated_matmul(x, w),), (x, w)),
        }[name]
        outs = call()
        gs = [rand(*o.shape, seed=9 + i).requires_grad_() for i, o in enumerate(outs)]
        plain = torch.autograd.grad(outs, leaves, gs, retain_graph=True)
        grads = torch.autograd.grad(outs, leaves, gs, create_graph=True)
        for a, b in zip(grads, plain):
            assert torch.equal(a, b) and a.requires_grad and not b.requires_grad
            with pytest.raises(RuntimeError, match="no second derivative"):
                a.square().sum().backward(retain_graph=True)
        return []

    both(monkeypatch, step)


def test_forward_mode_is_refused():
    from torch.autograd.forward_ad import dual_level, make_dual

    q, s, ld = rand(1, 5, 2, 8, seed=1), rand(5, 2, 8, 8, seed=4), decays(2)
    pos, f = positions_of(5, 50), branch.rotary_frequencies(8, device=DEV)
    x, w = rand(6, 16, seed=5), rand(8, 16, seed=6)
    calls = [lambda d: branch.rotary(d(q), q, pos, f), lambda d: branch.rotary(q, d(q), pos, f),
             lambda d: branch.decay_attention(d(q), q, q, ld), lambda d: branch.decay_attention(q, q, d(q), ld),
             lambda d: branch.decay_attention(q, q, q, ld, initial_state=d(s[:1])),
             lambda d: branch.decay_attention_step(q[0], d(q[0]), q[0], ld, s),
             lambda d: branch.decay_attention_step(q[0], q[0], q[0], ld, d(s)),
             lambda d: branch.gated_matmul(d(x), w), lambda d: branch.gated_matmul(x, d(w))]
    for call in calls:
        for mode in (torch.no_grad, torch.enable_grad):
            with mode(), dual_level():
                call(lambda t: t)
                with pytest.raises(NotImplementedError):
                    call(lambda t: make_dual(t, t.clone()))


# --------------------------------------------------------------------------
# Strides, broadcasts, positions
# --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shift", [0, 1])
def test_parts_of_a_fused_projection(dtype, shift):
    """q, k and v side by side in a token's row, and rows that begin off 16-byte boundaries; nothing is copied."""
    dt, B, T, H, D = DT[dtype], 2, 70, 2, 64
    rows = rand(B * T * 3 * H * D + 8, seed=1, dtype=dt)[shift:shift + B * T * 3 * H * D].view(B, T, 3 * H, D)
    q, k, v = (rows[:, :, i * H:(i + 1) * H] for i in range(3))
    for t in (q, k, v):
        assert _mixer._Heads(t).t.data_ptr() == t.data_ptr()
    f, pos = branch.rotary_frequencies(D, device=DEV), positions_of(T, 4000)
    check_rotary(q.detach().requires_grad_(), k.detach().requires_grad_(), pos, f, False, 1.0, rand(B, T, H, D, seed=2, dtype=dt),
                 rand(B, T, H, D, seed=3, dtype=dt))
    check_decay(*(t.detach().requires_grad_() for t in (q, k, v)), decays(H), None, None, rand(B, T, H, D, seed=4, dtype=dt), None,
                0.2, [(0, T), (T, 2 * T)])


def test_heads_that_are_one_and_rows_in_another_order():
    """k and v of one head expanded to all, whose gradients add up; heads before tokens (copied where rows do not merge)."""
    B, T, H, D = 2, 40, 3, 32
    q, k, v, do = (leaf(B, T, n, D, seed=i, dtype=BF) for i, n in ((1, H), (2, 1), (3, 1), (4, H)))
    ld = decays(H)
    o = branch.decay_attention(q, k.expand_as(q), v.expand_as(q), ld)
    got = torch.autograd.grad(o, (q, k, v), do.detach())
    full = [t.detach().expand_as(q).contiguous().requires_grad_() for t in (k, v)]
    o2 = branch.decay_attention(q, *full, ld)
    want = torch.autograd.grad(o2, (q, *full), do.detach())
    assert torch.equal(o, o2) and torch.equal(got[0], want[0])
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a, b.sum(2, keepdim=True))
    across = [t.detach().transpose(1, 2).contiguous().transpose(1, 2) for t in (q, *full)]
    assert torch.equal(branch.decay_attention(*across, ld), o)
    inner = [t.detach().transpose(2, 3).contiguous().transpose(2, 3) for t in (q, *full)]  # a head's elements apart
    assert torch.equal(branch.decay_attention(*inner, ld), o)
    pos, f = positions_of(T, 100), branch.rotary_frequencies(D, device=DEV)
    r = branch.rotary(q.detach(), None, pos, f)
    assert torch.equal(branch.rotary(across[0], None, pos, f), r) and torch.equal(branch.rotary(inner[0], None, pos, f), r)


def test_gradients_of_any_strides():
    """A gradient that is broadcast or transposed."""
    B, T, H, D = 2, 33, 2, 24
    q, k, v = (leaf(B, T, H, D, seed=i) for i in (1, 2, 3))
    pos, f, ld = positions_of(T, 100), branch.rotary_frequencies(D, device=DEV), decays(H)
    for do in (torch.ones((), device=DEV).expand(B, T, H, D), rand(B, H, T, D, seed=4).transpose(1, 2), rand(D, B, T, H, seed=5).permute(1, 2, 3, 0)):
        o, r = branch.decay_attention(q, k, v, ld), branch.rotary(q, None, pos, f)
        for a, b in zip(torch.autograd.grad(o, (q, k, v), do, retain_graph=True), torch.autograd.grad(o, (q, k, v), do.contiguous())):
            assert torch.equal(a, b)
        assert torch.equal(torch.autograd.grad(r, q, do, retain_graph=True)[0], torch.autograd.grad(r, q, do.contiguous())[0])


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_rotary_positions(dtype):
    """Of each row, of each token of every sequence, one for all; negative and far ones, whose angles stay exact."""
    D, f = 64, branch.rotary_frequencies(64, device=DEV)
    q = rand(3, 5, 2, D, seed=1)
    token = torch.tensor([0, 7, -3, 1 << 20, (1 << 31) - 1], device=DEV).to(dtype)
    rows = token.repeat(3).view(3, 5)
    want = branch.rotary(q, None, rows, f)
    assert torch.equal(branch.rotary(q, None, token, f), want)
    assert torch.equal(branch.rotary(q, None, rows.t().contiguous().t(), f), want)
    assert torch.equal(branch.rotary(q[0, 1], None, token[1], f), want[0, 1])
    ref, size = M.rotary(to_np(q).reshape(15, 2, D), to_np(rows).reshape(-1), to_np(f))
    # the oracle's own angle is off by 2^-53 of up to 2^31 radians
    close(want.view(15, 2, D), ref, size, 2.0 ** -21 + 2.0 ** -21, "far")
    if dtype == torch.int64:
        far = torch.tensor([1 << 40], device=DEV)
        a = branch.rotary(q[0, :1], None, far, torch.tensor([2 * np.pi * 2.0 ** -42], dtype=torch.float64, device=DEV))
        assert torch.allclose(a[0, :, 0], -q[0, 0, :, 1], atol=1e-6) and torch.allclose(a[0, :, 1], q[0, 0, :, 0], atol=1e-6)


def test_rotary_of_many_rows_and_scores_of_relative_positions():
    """More row tiles than a launch's workgroups walk once; q . k of turned heads depends on the distance alone."""
    R = 4 * 256 * 8 + 5
    q, f = rand(R, 2, 16, seed=1, dtype=BF), branch.rotary_frequencies(16, device=DEV)
    pos = positions_of(R, 1 << 20)
    y = branch.rotary(q, None, pos, f)
    for lo in (0, R // 2, R - 9):
        assert torch.equal(branch.rotary(q[lo:lo + 9], None, pos[lo:lo + 9], f), y[lo:lo + 9])
    a, b = rand(1, 1, 16, seed=2).expand(50, 1, 16), rand(1, 1, 16, seed=3).expand(50, 1, 16)
    p = torch.arange(50, device=DEV, dtype=torch.int32) * 1000
    x, z = branch.rotary(a, b, p, f)[0], branch.rotary(a, b, p + 77, f)[1]
    s = (x * z).sum(-1)
    assert float((s - s[0]).abs().max()) < 1e-5


# --------------------------------------------------------------------------
# Values that are not finite, decays at their ends
# --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("what", ["q", "k", "v"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_decay_attention_keeps_the_future_out(what, bad, dtype):
    """A value that is not finite at one token changes no earlier token, no other sequence and no other head; of q it
    stays in its row, of v in its column."""
    dt, B, T, H, D = DT[dtype], 2, 150, 2, 72
    t = {n: rand(B, T, H, D, seed=i, dtype=dt) for i, n in enumerate("qkv")}
    ld = torch.tensor([-0.1, 0.0], device=DEV)
    want = branch.decay_attention(t["q"], t["k"], t["v"], ld)
    for at in (0, 37, 64, 149):
        x = {n: v.clone() for n, v in t.items()}
        x[what][1, at, 0, 5] = bad
        o = branch.decay_attention(x["q"], x["k"], x["v"], ld)
        assert torch.equal(o[0], want[0]) and torch.equal(o[1, :, 1], want[1, :, 1])
        assert torch.allclose(o[1, :at, 0].float(), want[1, :at, 0].float(), rtol=2.0 ** -7, atol=1e-2)
        gone = ~torch.isfinite(o[1, :, 0])
        if what == "q":
            assert torch.equal(o[1, at + 1:, 0], want[1, at + 1:, 0]) and gone[at].all()
        elif what == "k":
            assert gone[at:].all()
        else:
            assert gone[at:, 5].all() and not gone[:, :5].any() and not gone[:, 6:].any()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_gradients_keep_the_future_out(dtype):
    """dq of tokens before a bad k or v, dk and dv of tokens behind a bad q or gradient."""
    dt, T, D = DT[dtype], 100, 64
    base = [rand(1, T, 1, D, seed=i, dtype=dt) for i in range(4)]
    ld = torch.tensor([-0.05], device=DEV)

    def grads(q, k, v, do):
        q, k, v = (t.clone().requires_grad_() for t in (q, k, v))
        return torch.autograd.grad(branch.decay_attention(q, k, v, ld), (q, k, v), do)

    want = grads(*base)
    for i in range(4):
        x = [t.clone() for t in base]
        x[i][0, 50, 0, 3] = float("nan")
        dq, dk, dv = grads(*x)
        near = lambda a, b: torch.allclose(a.float(), b.float(), rtol=2.0 ** -6, atol=2e-2)  # noqa: E731
        if i in (1, 2):
            assert near(dq[:, :50], want[0][:, :50])
        else:
            assert near(dk[:, 51:], want[1][:, 51:]) and near(dv[:, 51:], want[2][:, 51:])


def test_bad_rows_of_no_sequence_stay_there():
    """NaN behind the last sequence, in its rows and in the states of others."""
    R, H, D = 100, 2, 40
    off = torch.tensor([30, 30, 80], dtype=torch.int32, device=DEV)
    q, k, v, do = (rand(R, H, D, seed=i, dtype=BF) for i in range(4))
    s = rand(3, H, D, D, seed=5)

    def run():
        leaves = [t.clone().requires_grad_() for t in (q, k, v, s)]
        out = branch.decay_attention(*leaves[:3], decays(H), initial_state=leaves[3], offsets=off, return_state=True)
        return [*out, *torch.autograd.grad(out, leaves, (do, torch.ones_like(s)))]

    want = run()
    for t in (q, k, v, do):
        t[80:] = float("nan")
    s[1] = float("inf")
    got = run()
    for a, b in zip(got[:1] + got[2:5], want[:1] + want[2:5]):
        assert torch.equal(a[:80], b[:80]) and not a[80:].any()
    for a, b in ((got[1], want[1]), (got[5], want[5])):
        assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])


@pytest.mark.parametrize("dtype", list(DT))
def test_decays_at_their_ends(dtype):
    """Nothing kept, next to nothing, everything, and above 0, which counts as 0; NaN stays in its head."""
    dt, T, D = DT[dtype], 140, 64
    ld = torch.tensor([-float("inf"), -1e4, -30.0, -1e-7, 0.0, 3.0], device=DEV)
    H = ld.numel()
    q, k, v = (leaf(1, T, H, D, seed=i, dtype=dt) for i in range(3))
    do, first, d_last = rand(1, T, H, D, seed=4, dtype=dt), leaf(1, H, D, D, seed=5), rand(1, H, D, D, seed=6)
    check_decay(q, k, v, ld, None, first, do, d_last, 0.1, [(0, T)])
    with torch.no_grad():
        want = branch.decay_attention(q, k, v, ld)
        ld[1] = float("nan")
        got = branch.decay_attention(q, k, v, ld)
    assert torch.isnan(got[:, 1:, 1]).all() and all(torch.equal(got[:, :, h], want[:, :, h]) for h in (0, 2, 3, 4, 5))


def test_long_sequences_and_slow_decays():
    """Thousands of chunks' decays multiplied up: 2^-21 a chunk in between, mended every 16th."""
    T, D = 20000, 16
    for ld in (-1e-3, -1.0 / 8192, -1e-6, 0.0):
        q, k, v = (rand(1, T, 1, D, seed=i) for i in range(3))
        first = rand(1, 1, D, D, seed=4, scale=100.0)
        o, s = branch.decay_attention(q, k, v, torch.tensor([ld], device=DEV), initial_state=first, return_state=True, scale=1.0)
        rows = lambda t: to_np(t)[0]  # noqa: E731
        L = np.float64(np.float32(ld))[None]
        ro, rs = M.decay_attention(rows(q), rows(k), rows(v), L, [(0, T)], to_np(first), 1.0)
        assert np.linalg.norm(to_np(s) - rs) < 2e-6 * np.linalg.norm(rs)
        assert np.linalg.norm(rows(o) - ro) < 2e-6 * np.linalg.norm(ro)


# --------------------------------------------------------------------------
# Offsets, slots
# --------------------------------------------------------------------------

@pytest.mark.parametrize("ends", [[40, 20, 90], [-5, 300, 10], [0, 0, 0], [2 ** 40, 5, 7], [-2 ** 40, 50, 2 ** 31]])
def test_any_offsets(ends):
    """Clamped and as their running maximum, in int64, too."""
    R, H, D = 100, 2, 24
    q, k, v = (leaf(R, H, D, seed=i, dtype=BF) for i in range(3))
    do, first, d_last = rand(R, H, D, seed=4, dtype=BF), leaf(3, H, D, D, seed=5), rand(3, H, D, D, seed=6)
    check_decay(q, k, v, decays(H), torch.tensor(ends, device=DEV), first, do, d_last, 0.2, M.spans_of(ends, R))
    x, w, dy = leaf(R, 40, seed=7, dtype=BF), leaf(3, 48, 40, seed=8, dtype=BF), rand(R, 24, seed=9, dtype=BF)
    if all(abs(e) < 2 ** 31 for e in ends):
        check_gated(x, w, ends, "silu", dy)


def test_empty_calls():
    e = lambda *s: torch.empty(*s, device=DEV, dtype=BF).requires_grad_()  # noqa: E731
    f, ld = branch.rotary_frequencies(16, device=DEV), decays(2)
    q, k = branch.rotary(e(0, 2, 16), e(0, 1, 16), torch.empty(0, dtype=torch.int32, device=DEV), f)
    assert q.shape == (0, 2, 16) and k.shape == (0, 1, 16)
    s = rand(3, 2, 16, 16, seed=1).requires_grad_()
    x = e(3, 0, 2, 16)
    o, last = branch.decay_attention(x, x, x, ld, initial_state=s, return_state=True)
    assert o.shape == x.shape and torch.equal(last, s)
    g, = torch.autograd.grad(last, s, torch.ones_like(s))
    assert torch.equal(g, torch.ones_like(s))
    y = e(5, 2, 16)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    o, last = branch.decay_attention(y.detach().zero_().requires_grad_(), y, y, ld, offsets=none, return_state=True)
    assert not o.any() and last.shape == (0, 2, 16, 16)
    assert branch.decay_attention_step(e(0, 2, 16).detach(), e(0, 2, 16).detach(), e(0, 2, 16).detach(), ld, s.detach()).shape == (0, 2, 16)
    x, w = e(0, 8), e(12, 8)
    z = branch.gated_matmul(x, w)
    dx, dw = torch.autograd.grad(z, (x, w), torch.empty_like(z))
    assert z.shape == (0, 6) and dx.shape == (0, 8) and not dw.any()
    x, w = rand(4, 0, seed=1).requires_grad_(), torch.empty(12, 0, device=DEV).requires_grad_()
    z = branch.gated_matmul(x, w)
    assert z.shape == (4, 6) and not z.any()


def test_step_continues_a_prompt():
    """A prompt's state moved on token by token gives what the whole sequence gives, to rounding."""
    B, T, H, D = 3, 90, 2, 64
    q, k, v = (rand(B, T, H, D, seed=i) for i in range(3))
    ld = decays(H)
    whole, last = branch.decay_attention(q, k, v, ld, return_state=True)
    _, state = branch.decay_attention(q[:, :80], k[:, :80], v[:, :80], ld, return_state=True)
    for t in range(80, T):
        o = branch.decay_attention_step(q[:, t], k[:, t], v[:, t], ld, state)
        assert torch.allclose(o, whole[:, t], atol=2e-4, rtol=1e-4)
    assert torch.allclose(state, last, atol=1e-4, rtol=1e-4)


def test_step_updates_count_as_writes():
    s, q = rand(2, 1, 8, 8, seed=1), rand(2, 1, 8, seed=2)
    for native in (True, False):
        x = torch.ones(2, 1, 8, 8, device=DEV, requires_grad=True)
        y = x * s
        before = s._version
        branch.decay_attention_step(q, q, q, decays(1), s) if native else _mixer_step(q, s)
        assert s._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    with torch.inference_mode():
        t = rand(2, 1, 8, 8, seed=1).clone()
        branch.decay_attention_step(q, q, q, decays(1), t)


def _mixer_step(q, s):
    from mhc import _lib

    real = _lib._native
    _lib._native = _lib._NoBinding()
    try:
        branch.decay_attention_step(q, q, q, decays(1), s)
    finally:
        _lib._native = real


def test_step_refuses_states_that_overlap():
    pool = rand(6, 1, 8, 8, seed=1)
    q = rand(4, 1, 8, seed=2)
    with pytest.raises(ValueError, match="apart"):
        branch.decay_attention_step(q, q, q, decays(1), pool[:5], state_out=pool[1:])
    a, b = pool[:5].clone(), pool[:5].clone()
    branch.decay_attention_step(q, q, q, decays(1), a, state_out=a)
    branch.decay_attention_step(q, q, q, decays(1), b)
    assert torch.equal(a, b)


# --------------------------------------------------------------------------
# Streams, graphs, memory
# --------------------------------------------------------------------------

def test_another_stream():
    steps = _steps(BF)
    want = {n: f() for n, f in steps.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = {n: f() for n, f in steps.items()}
    torch.cuda.current_stream().wait_stream(side)
    for n in want:
        same(got[n], want[n])


def test_two_graphs_replayed_in_turn():
    """Prompts of changing lengths, and a decode step, in a graph each; the second may run between replays of the first."""
    R, N, H, D = 700, 3, 2, 64
    q, k, v = (rand(R, H, D, seed=i, dtype=BF) for i in range(3))
    pos, f, ld = torch.arange(R, device=DEV, dtype=torch.int32), branch.rotary_frequencies(D, device=DEV), decays(H)
    off = torch.tensor([100, 650, 690], dtype=torch.int32, device=DEV)
    state, slots = rand(8, H, D, D, seed=5), torch.tensor([1, 5, 2], dtype=torch.int32, device=DEV)
    x, w = rand(64, 96, seed=6, dtype=BF), rand(80, 96, seed=7, dtype=BF)

    def prompt():
        a, b = branch.rotary(q, k, pos, f)
        o, s = branch.decay_attention(a, b, v, ld, offsets=off, return_state=True)
        return o, s, branch.gated_matmul(x, w)

    def decode():
        return branch.decay_attention_step(q[:3], k[:3], v[:3], ld, state, slots=slots)

    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            prompt()
            kept = state.clone()
            decode()
            state.copy_(kept)
        torch.cuda.current_stream().wait_stream(side)
        one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(one):
            out = prompt()
        with torch.cuda.graph(two):
            step = decode()
        for i, (ends, at) in enumerate([([100, 650, 690], [1, 5, 2]), ([0, 1, 700], [7, 7, -1]), ([300, 300, 300], [0, 3, 0]), ([64, 128, 640], [2, 9, 4])]):
            off.copy_(torch.tensor(ends))
            slots.copy_(torch.tensor(at))
            q.add_(0.125 * i)
            before = state.clone()
            want = prompt()
            wstep = branch.decay_attention_step(q[:3], k[:3], v[:3], ld, before, slots=slots)
            one.replay()
            two.replay()
            torch.cuda.synchronize()
            same(list(out), list(want))
            assert torch.equal(step, wstep) and torch.equal(state, before)


def test_training_step_in_a_graph():
    q, k, v = (leaf(1, 600, 1, 64, seed=i, dtype=BF) for i in range(3))
    x, w = leaf(64, 96, seed=6, dtype=BF), leaf(80, 96, seed=7, dtype=BF)
    pos, f, ld = torch.arange(600, device=DEV, dtype=torch.int32), branch.rotary_frequencies(64, device=DEV), decays(1)
    do, dy = rand(1, 600, 1, 64, seed=8, dtype=BF), rand(64, 40, seed=9, dtype=BF)

    def step():
        a, b = branch.rotary(q, k, pos, f)
        o, y = branch.decay_attention(a, b, v, ld), branch.gated_matmul(x, w)
        return torch.autograd.grad((o, y), (q, k, v, x, w), (do, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        do.mul_(1.25)
        dy.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        kept = [g.clone() for g in got]
        same(kept, list(step()))


def test_outputs_and_workspaces_are_written_before_they_are_read(monkeypatch):
    """With every new tensor's bytes set to 0xFF (NaN in each type) the results are the same."""
    from mhc import _lib

    def run():
        out = []
        for dt in DT.values():
            for f in _steps(dt).values():
                out += f()
            H = 1  # several segments
            q, k, v = (leaf(1300, H, d, seed=i, dtype=dt) for i, d in enumerate((40, 40, 72)))
            off = torch.tensor([20, 1290], dtype=torch.int32, device=DEV)
            o = branch.decay_attention(q, k, v, decays(H), offsets=off, return_state=True)
            out += [*o, *torch.autograd.grad(o, (q, k, v), [torch.ones_like(t) for t in o])]
        return [t.detach().contiguous().view(torch.uint8) for t in out]

    class Off:
        def __getattr__(self, name):
            return lambda *a: None

    monkeypatch.setattr(_lib, "native", lambda: Off())
    want = run()
    for owner, name in ((torch, "empty"), (torch, "empty_like")):
        def poisoned(*a, _make=getattr(owner, name), **k):
            t = _make(*a, **k)
            if t.is_cuda and t.numel() and t.is_contiguous():
                t.view(torch.uint8).fill_(0xFF)
            return t
        monkeypatch.setattr(owner, name, poisoned)
    got = run()
    monkeypatch.undo()
    same(got, want)


def test_rows_past_32_bits():
    """Tensors past 2^32 bytes and 2^31 elements: the last rows come out as by themselves."""
    R, H, D = (1 << 21) + 70, 8, 128
    need = R * H * D * 2 * 5 + (4 << 30)
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < need:
        pytest.skip(f"needs {need >> 30} GiB of GPU memory")
    x = torch.empty(R, H, D, device=DEV, dtype=BF).fill_(0.01)
    x[-200:] = rand(200, H, D, seed=1, dtype=BF)
    pos, f, ld = torch.arange(R, device=DEV, dtype=torch.int32), branch.rotary_frequencies(D, device=DEV), torch.full((H,), -0.5, device=DEV)
    with torch.no_grad():
        y = branch.rotary(x, None, pos, f)
        assert torch.equal(y[-200:], branch.rotary(x[-200:].clone(), None, pos[-200:].clone(), f))
        del y
        off = torch.tensor([R - 133, R - 3], device=DEV)
        o = branch.decay_attention(x, x, x, ld, offsets=off)
        want = branch.decay_attention(*[x[-133:].clone()] * 3, ld, offsets=torch.tensor([130], device=DEV))
        assert torch.equal(o[-133:], want) and not o[-3:].any()
    del x, o
    torch.cuda.empty_cache()


def test_states_past_32_bits():
    """A pool of states past 2^32 bytes."""
    pool, H, D = 70000, 1, 128
    torch.cuda.empty_cache()
    need = pool * D * D * 4 + (2 << 30)
    if torch.cuda.mem_get_info()[0] < need:
        pytest.skip(f"needs {need >> 30} GiB of GPU memory")
    state = torch.zeros(pool, H, D, D, device=DEV)
    q, k, v = (rand(3, H, D, seed=i, dtype=BF) for i in range(3))
    slots = torch.tensor([pool - 1, 0, 65537], device=DEV)
    state[slots] = rand(3, H, D, D, seed=4)
    small = state[slots].clone()
    want = branch.decay_attention_step(q, k, v, decays(H), small)
    got = branch.decay_attention_step(q, k, v, decays(H), state, slots=slots)
    assert torch.equal(got, want) and torch.equal(state[slots], small) and not state[1:65537].any()
    del state
    torch.cuda.empty_cache()


def test_gradients_against_differences():
    """Central differences along a random direction, fp32.  Decay attention is linear in q and in v, and quadratic in
    nothing: differences of one operand are exact to rounding; gated products' third derivatives are of order one."""
    B, T, H, D = 1, 150, 2, 32
    q, k, v, do = (rand(B, T, H, D, seed=i) for i in range(4))
    first, d_last, ld = rand(B, H, D, D, seed=5), rand(B, H, D, D, seed=6), decays(H)
    pos, f = positions_of(T, 500), branch.rotary_frequencies(D, device=DEV)
    x, w, dy = rand(40, 24, seed=7), rand(32, 24, seed=8, scale=0.3), rand(40, 16, seed=9)

    def decay(q, k, v, s):
        o, last = branch.decay_attention(q, k, v, ld, initial_state=s, return_state=True)
        return float((o.double() * do.double()).sum() + (last.double() * d_last.double()).sum())

    def check(fn, args, grads, t, tol):
        for i, g in enumerate(grads):
            e = rand(*args[i].shape, seed=20 + i)
            up, down = [[a + s * t * e if j == i else a for j, a in enumerate(args)] for s in (1, -1)]
            diff, want = (fn(*up) - fn(*down)) / (2 * t), float((g.double() * e.double()).sum())
            scale = float((g.double() * e.double()).square().sum().sqrt()) + g.numel() ** 0.5
            assert abs(diff - want) < tol * scale, i

    leaves = [t.clone().requires_grad_() for t in (q, k, v, first)]
    o, last = branch.decay_attention(*leaves[:3], ld, initial_state=leaves[3], return_state=True)
    check(decay, (q, k, v, first), torch.autograd.grad((o, last), leaves, (do, d_last)), 1.0, 1e-3)
    leaf_q = q.clone().requires_grad_()
    g = torch.autograd.grad(branch.rotary(leaf_q, None, pos, f), leaf_q, do)
    check(lambda q: float((branch.rotary(q, None, pos, f).double() * do.double()).sum()), (q,), g, 1.0, 1e-3)
    for act in ("silu", "gelu", "gelu_tanh"):
        leaves = [t.clone().requires_grad_() for t in (x, w)]
        g = torch.autograd.grad(branch.gated_matmul(*leaves, activation=act), leaves, dy)
        check(lambda x, w: float((branch.gated_matmul(x, w, activation=act).double() * dy.double()).sum()), (x, w), g, 2.0 ** -6, 1e-2)


def test_gated_activations_at_their_ends():
    """Gates far from zero, infinite and NaN: values and slopes without overflow on the way."""
    g = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 30.0, -30.0, 90.0, -90.0, 1e4, -1e4, 1e20, -1e20, 3e38, -3e38], device=DEV)
    x, w = torch.ones(1, 1, device=DEV), torch.cat((g, torch.ones_like(g)))[:, None].contiguous()
    for act in ("silu", "gelu", "gelu_tanh"):
        wl, xl = w.clone().requires_grad_(), x.clone().requires_grad_()
        y = branch.gated_matmul(xl, wl, activation=act)
        _, dw = torch.autograd.grad(y, (xl, wl), torch.ones_like(y))
        a, slope = M.activation(to_np(g), act)
        assert np.allclose(to_np(y)[0], a, rtol=1e-5, atol=1e-12), act
        assert np.allclose(to_np(dw)[:14, 0], slope, rtol=1e-4, atol=1e-6) and np.allclose(to_np(dw)[14:, 0], a, rtol=1e-5, atol=1e-12)
