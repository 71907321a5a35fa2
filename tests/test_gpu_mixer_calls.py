"""The operators that mix tokens on the GPU: calls that their documentation allows and that test_gpu_mixer.py and
test_gpu_mixer_paths.py do not make."""

import numpy as np
import pytest
import torch

from helpers import to_np
from test_gpu_branch import DT, close, rand
from test_gpu_mixer import check_decay, check_gated, decays
from test_gpu_native_nodes import both
from mhc import _mixer, branch
from oracle import mixer_oracle as M

pytestmark = pytest.mark.gpu

DEV = "cuda"


# --------------------------------------------------------------------------
# Rows that share memory
# --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("which", ["kv", "qd", "qkvd"])
@pytest.mark.parametrize("B,T,D", [(1, 100, 64), (2, 1, 64), (2, 70, 128), (1, 300, 40)])
def test_tokens_that_are_one_expanded(B, T, D, which, dtype):
    """Operands and gradients of row stride 0, whole chunks and short ones."""
    dt, H = DT[dtype], 2
    t = {n: (rand(H, D, seed=i, dtype=dt).expand(B, T, H, D) if n in which else rand(B, T, H, D, seed=i, dtype=dt))
         for i, n in enumerate("qkvd")}
    q, k, v = (t[n].detach().requires_grad_() for n in "qkv")
    first, d_last = rand(B, H, D, D, seed=5).requires_grad_(), rand(B, H, D, D, seed=6)
    check_decay(q, k, v, decays(H), None, first, t["d"], d_last, 0.1, [(n * T, (n + 1) * T) for n in range(B)])


@pytest.mark.parametrize("dtype", list(DT))
def test_tokens_that_are_windows_of_one_row(dtype):
    """Rows 8 elements apart, which overlap."""
    dt, T, H, D = DT[dtype], 90, 2, 64
    q, k, v, do = (rand(8 * T + H * D, seed=i, dtype=dt).as_strided((T, H, D), (8, D, 1)) for i in range(4))
    off = torch.tensor([30, 85], device=DEV)
    first, d_last = rand(2, H, D, D, seed=5).requires_grad_(), rand(2, H, D, D, seed=6)
    check_decay(*(t.detach().requires_grad_() for t in (q, k, v)), decays(H), off, first, do, d_last, 0.1, [(0, 30), (30, 85)])


# --------------------------------------------------------------------------
# Segments of many sequences
# --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (40, 100)])
@pytest.mark.parametrize("lens", [None, [257, 256, 512, 513, 1, 0, 769, 255, 300, 300], [2500, 1, 1, 2500]])
def test_segments_of_many_sequences(lens, Dk, Dv, dtype):
    """Sequences a token shorter and longer than segments, whose states lie close together; several that are joined."""
    dt, H = DT[dtype], 1
    lead = (sum(lens),) if lens else (5, 600)
    spans = [(n * 600, (n + 1) * 600) for n in range(5)] if lens is None else [(sum(lens[:n]), sum(lens[:n + 1])) for n in range(len(lens))]
    off = None if lens is None else torch.tensor(lens, device=DEV).cumsum(0)
    q, k = (rand(*lead, H, Dk, seed=i, dtype=dt).requires_grad_() for i in (1, 2))
    v, do = rand(*lead, H, Dv, seed=3, dtype=dt).requires_grad_(), rand(*lead, H, Dv, seed=4, dtype=dt)
    first, d_last = rand(len(spans), H, Dk, Dv, seed=5).requires_grad_(), rand(len(spans), H, Dk, Dv, seed=6)
    ld = torch.tensor([-0.002], device=DEV)
    check_decay(q, k, v, ld, off, first, do, d_last, Dk ** -0.5, spans)
    check_decay(q, k, v, ld, off, None, do, None, Dk ** -0.5, spans)


def test_a_long_sequence_among_many_short_ones():
    """Its many segments' states are joined whatever it is packed with: the bits are those of the sequence alone.  Packed with
    another one, sequences of a few segments are summed beside it as among themselves."""
    H, D, T = 1, 64, 7000  # segments of 256
    ld = torch.tensor([-0.0005], device=DEV)

    def run(ends, R):
        q, k, v = (rand(9400, H, D, seed=i)[:R].contiguous().requires_grad_() for i in (1, 2, 3))
        off = torch.tensor(ends, dtype=torch.int32, device=DEV)
        o, state = branch.decay_attention(q, k, v, ld, offsets=off, return_state=True)
        do, d_state = rand(9400, H, D, seed=4)[:R], rand(200, H, D, D, seed=5)[:len(ends)]
        return [o, state, *torch.autograd.grad((o, state), (q, k, v), (do, d_state))]

    alone = run([T], T)
    for i, ends in enumerate(([T, T + 1500, T + 2000], [T, *range(T + 1, T + 200)])):
        got = run(ends, 9400)
        for a, b in zip(got, alone):
            assert torch.equal(a[:len(b)], b)
        if i == 0:  # two of 1500 and 500 tokens
            rows = slice(T, T + 2000)
            q, k, v = (rand(9400, H, D, seed=s)[rows] for s in (1, 2, 3))
            o = branch.decay_attention(q, k, v, ld, offsets=torch.tensor([1500, 2000], device=DEV))
            assert torch.equal(got[0][rows], o)


def _lengths(N, seed):
    """Mostly a few tokens or none, now and then some hundreds."""
    r = np.random.default_rng(seed)
    return np.where(r.random(N) < 0.005, r.integers(200, 700, N), r.integers(0, 4, N))


@pytest.mark.parametrize("N,long,extra", [(127, 0, 3), (128, 0, 0), (1023, 300, 5), (1024, 0, 300), (1025, 5000, 0), (2500, 4000, 700)])
def test_many_sequences(N, long, extra):
    """Around the sizes at which a table says where tiles begin and at which it takes another round; long sequences, whose
    segments are joined, among the first and the last; rows behind the last."""
    H, Dk, Dv = 1, 24, 40
    lens = _lengths(N, N)
    lens[3], lens[N - 2] = long or lens[3], long // 2 or lens[N - 2]
    ends = np.cumsum(lens)
    R = int(ends[-1]) + extra
    q, k = (rand(R, H, Dk, seed=i, dtype=torch.bfloat16).requires_grad_() for i in (1, 2))
    v, do = rand(R, H, Dv, seed=3, dtype=q.dtype).requires_grad_(), rand(R, H, Dv, seed=4, dtype=q.dtype)
    first, d_last = rand(N, H, Dk, Dv, seed=5).requires_grad_(), rand(N, H, Dk, Dv, seed=6)
    off, ld = torch.tensor(ends, device=DEV), torch.tensor([-0.002], device=DEV)
    check_decay(q, k, v, ld, off, first, do, d_last, Dk ** -0.5, M.spans_of(ends.tolist(), R))
    # each gradient by itself, which makes the table again
    o, state = branch.decay_attention(q, k, v, ld, initial_state=first, offsets=off, return_state=True)
    for a, b in zip((k, v, first), torch.autograd.grad((o, state), (k, v, first), (do, d_last), retain_graph=True)):
        got = _mixer.decay_attention_backward(q, k, v, do, ld, off, first, None, d_last, Dk ** -0.5,
                                              (False, a is k, a is v, a is first))
        close(next(g for g in got if g is not None), to_np(b), np.abs(to_np(b)).max(), 2.0 ** -7)


def test_many_sequences_of_any_offsets():
    """Offsets that fall, lie below 0 and past the rows; sequences without any token at all."""
    H, D, R, N = 2, 16, 500, 1500
    r = np.random.default_rng(1)
    ends = np.sort(r.integers(-50, R + 50, N)) + r.integers(-20, 20, N)
    q, k, v = (rand(R, H, D, seed=i).requires_grad_() for i in (1, 2, 3))
    first, d_last, do = rand(N, H, D, D, seed=5).requires_grad_(), rand(N, H, D, D, seed=6), rand(R, H, D, seed=4)
    check_decay(q, k, v, decays(H), torch.tensor(ends, device=DEV), first, do, d_last, 0.2, M.spans_of(ends.tolist(), R))
    e = torch.empty(0, H, D, device=DEV).requires_grad_()
    o, state = branch.decay_attention(e, e, e, decays(H), initial_state=first, offsets=torch.tensor(ends, device=DEV), return_state=True)
    g, = torch.autograd.grad(state, first, d_last)
    assert o.shape == e.shape and torch.equal(state, first) and torch.equal(g, d_last)


def test_many_sequences_whose_forward_left_nothing():
    """Without tokens and with no state wanted the forward does nothing; the gradient of the first states is there all the same.
    Whatever becomes of the states that a forward kept, gradients stay in their places."""
    H, D, N = 2, 16, 300
    off, ld = torch.zeros(N, dtype=torch.int32, device=DEV), decays(H)
    e, first = torch.empty(0, H, D, device=DEV).requires_grad_(), rand(N, H, D, D, seed=1).requires_grad_()
    o = branch.decay_attention(e, e, e, ld, initial_state=first, offsets=off)
    g, dq = torch.autograd.grad(o, (first, e), torch.empty_like(o))
    assert not g.any() and dq.shape == e.shape
    ends = torch.tensor(np.cumsum(_lengths(N, 7)) + 900, device=DEV)
    R = int(ends[-1]) + 9
    q, k, v, do = (rand(R, H, D, seed=i) for i in range(4))
    kept = _mixer.decay_attention_forward(q, k, v, ld, ends, None, 0.1, False)[2]
    want = _mixer.decay_attention_backward(q, k, v, do, ld, ends, None, kept, None, 0.1, (True,) * 4)
    got = _mixer.decay_attention_backward(q, k, v, do, ld, ends, None, torch.full_like(kept, 255), None, 0.1, (True,) * 4)
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a, b)
    assert torch.equal(got[0][:256], want[0][:256]) and torch.isnan(got[0][256:900]).all()


def test_many_sequences_in_a_graph():
    """A captured training step whose sequences change between replays."""
    H, D, R, N = 1, 32, 3500, 200
    q, k, v = (rand(R, H, D, seed=i, dtype=torch.bfloat16).requires_grad_() for i in (1, 2, 3))
    do, ld, off = rand(R, H, D, seed=4, dtype=q.dtype), decays(H), torch.zeros(N, dtype=torch.int32, device=DEV)
    splits = [np.cumsum(_lengths(N, s)) for s in range(3)] + [np.arange(N) // 150 * 3000 + 5]

    def step():
        o = branch.decay_attention(q, k, v, ld, offsets=off)
        return [o.detach(), *torch.autograd.grad(o, (q, k, v), do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for ends in splits:
        off.copy_(torch.tensor(ends))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_many_sequences_take_no_longer_than_their_tokens():
    """32768 packed sequences of 4 tokens against the same in a batch.  A search of the offsets by every workgroup took 50 times as
    long, a table 1.1 times."""
    N, T, H, D = 32768, 4, 8, 64
    q, k, v = (rand(N, T, H, D, seed=i, dtype=torch.bfloat16) for i in (1, 2, 3))
    ld, off = decays(H), torch.arange(T, N * T + 1, T, device=DEV, dtype=torch.int32)

    def time(f):
        out, best = f(), float("inf")
        for _ in range(3):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            f()
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return out, best

    want, dense = time(lambda: branch.decay_attention(q, k, v, ld))
    got, packed = time(lambda: branch.decay_attention(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), ld, offsets=off))
    print(f"packed {packed:.2f} ms, dense {dense:.2f} ms", flush=True)
    assert torch.equal(got.view_as(want), want) and packed < 8 * dense


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (100, 30), (30, 100)])
def test_the_forwards_states_serve_the_backward(Dk, Dv, dtype):
    """What the forward keeps is what q's gradient starts from in every segment but the first, and nothing else."""
    dt, H, T = DT[dtype], 1, 700  # segments of 256
    q, k, v, do = (rand(1, T, H, d, seed=i, dtype=dt) for i, d in enumerate((Dk, Dk, Dv, Dv)))
    ld = torch.tensor([-0.002], device=DEV)
    kept = _mixer.decay_attention_forward(q, k, v, ld, None, None, 0.1, False)[2]
    want = _mixer.decay_attention_backward(q, k, v, do, ld, None, None, kept, None, 0.1, (True,) * 4)
    got = _mixer.decay_attention_backward(q, k, v, do, ld, None, None, torch.full_like(kept, 255), None, 0.1, (True,) * 4)
    assert torch.equal(got[0][:, :256], want[0][:, :256]) and torch.isnan(got[0][:, 256:]).all()
    assert torch.isfinite(want[0]).all() and all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))


# --------------------------------------------------------------------------
# The most tokens
# --------------------------------------------------------------------------

def test_as_many_tokens_as_a_call_takes():
    """2^31 - 4096 tokens of one head, whose last segment ends within a segment of 2^31.  With nothing kept from token to
    token the output is v, and so is v's gradient where it is the output's."""
    R = (1 << 31) - 4096
    torch.cuda.empty_cache()
    need = R * 2 * 6 + (4 << 30)
    if torch.cuda.mem_get_info()[0] < need:
        pytest.skip(f"needs {need >> 30} GiB of GPU memory")
    v = torch.empty(1, R, 1, 1, device=DEV, dtype=torch.bfloat16).random_(1, 128, generator=torch.Generator(DEV).manual_seed(1))
    one = torch.ones((), device=DEV, dtype=v.dtype).expand(1, R, 1, 1)
    v.requires_grad_()
    o, state = branch.decay_attention(one, one, v, torch.tensor([-float("inf")], device=DEV), scale=1.0, return_state=True)
    assert torch.equal(o, v) and float(state) == float(v[0, -1])
    del state
    g, = torch.autograd.grad(o, v, v.detach())
    assert torch.equal(g, v)
    del o, g, v
    torch.cuda.empty_cache()


def test_rotary_of_more_row_tiles_than_a_launch_has_workgroups():
    """2^24 - 1 workgroups of four rows: those of the first rows take the last ones, too."""
    R, f = 4 * ((1 << 24) - 1 + 1000) + 3, torch.tensor([0.37], dtype=torch.float64, device=DEV)
    q = torch.empty(R, 1, 2, device=DEV, dtype=torch.bfloat16).normal_(generator=torch.Generator(DEV).manual_seed(1))
    pos = torch.arange(R, device=DEV, dtype=torch.int32) % 100003
    y = branch.rotary(q, None, pos, f)
    second = 4 * ((1 << 24) - 1)
    for lo, hi in ((0, 4096), (second - 100, second + 4003)):
        ref, size = M.rotary(to_np(q[lo:hi]), to_np(pos[lo:hi]), to_np(f))
        # an angle is off by its fp64 rounding, 2^-53 of up to 2^16 radians
        close(y[lo:hi], ref, size, 2.0 ** -21, "rows")
    # every row: turning keeps a pair's length, to the rounding of its two bf16 elements
    a, b = (t.float().square().sum((1, 2)).sqrt() for t in (q, y))
    assert bool(((a - b).abs() <= 2.0 ** -8 * a * 1.01 + 1e-30).all())


# --------------------------------------------------------------------------
# Gated products: fp32 in the largest tiles
# --------------------------------------------------------------------------

@pytest.mark.parametrize("R,K,N,off", [(6000, 64, 2864, None), (6000, 72, 2800, [2900, 2900, 5950])])
def test_gated_matmul_in_256_tiles_of_fp32(R, K, N, off):
    """Two likely tiles a CU and more: the last round in quarters, experts' last rows in half tiles, rows of no expert."""
    x = rand(R, K, seed=1).requires_grad_()
    w = rand(*(() if off is None else (len(off),)), 2 * N, K, seed=2, scale=K ** -0.5).requires_grad_()
    check_gated(x, w, off, "gelu", rand(R, N, seed=3))


# --------------------------------------------------------------------------
# No experts
# --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("K", [64, 65])
def test_gated_matmul_of_no_experts(monkeypatch, K, dtype):
    """As grouped_matmul: all rows are of no expert."""
    x, w = rand(70, K, seed=1, dtype=DT[dtype]).requires_grad_(), torch.empty(0, 24, K, dtype=DT[dtype], device=DEV).requires_grad_()
    off = torch.empty(0, dtype=torch.int32, device=DEV)

    def step():
        y = branch.gated_matmul(x, w, off)
        dx, dw = torch.autograd.grad(y, (x, w), rand(70, 12, seed=2, dtype=x.dtype))
        assert y.shape == (70, 12) and not y.any() and dx.shape == x.shape and not dx.any() and dw.shape == w.shape
        return [y.detach(), dx, dw]

    both(monkeypatch, step)
