"""The feed-forward operators run together, as a decoder runs them, and their
calls at the edges: captured and replayed, on other streams, prepared
elsewhere, between guard words, over rows past 32-bit offsets."""
import numpy as np
import pytest
import torch

import feedforward_reference as ref
import oracle_lib as ol
from gpu_util import say
from suf_amd import feedforward as ff
from suf_amd import native, tables, tasks
from test_gpu_feedforward import _empty, _open, _share, _values, _weights

pytestmark = pytest.mark.gpu

STATE = ol.mt64_bytes(4, ol.PRG_STATE_BYTES).tobytes()
F = 12


@pytest.fixture(scope="module", autouse=True)
def _init():
    native.call("sufhip_init", 0)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _act(name):
    return tables.gelu_table(F) if name == "gelu" else name


def _bias(rng, *shape):
    return (_values(rng, *shape, sigma=0.2) << np.uint64(F)).view(np.int64)


def _block(rng, rows, cols, hidden, act, weight):
    """A FeedForward, and what it computes of opened (x, residual)."""
    W = _weights(rng, 10, cols, hidden), _weights(rng, 10, hidden, cols)
    b = _bias(rng, hidden), _bias(rng, cols)
    w = np.rint((1 + 0.3 * rng.standard_normal(cols)) * 2 ** F).astype(np.int64) if weight else None
    block = ff.FeedForward(rows, ff.PublicWeights(W[0], b[0]), ff.PublicWeights(W[1], b[1]),
                           STATE, act=_act(act), weight=w, seed=100 * rows + cols)

    def want(x, residual):
        n = block.norm
        s, h = ref.rmsnorm(x, residual, n.inv_len, n.eps_q, n.table, F, w)
        u, _ = ref.linear(h, W[0], b[0], F, _act(act))
        return ref.linear(u, W[1], b[1], F, residual=s)[0]
    return block, want


BLOCKS = [(1, 64, 256, "relu", False), (1, 768, 100, "gelu", True), (3, 33, 70, None, True),
          (16, 96, 200, "gelu", False), (40, 130, 96, "relu", True), (200, 64, 160, "gelu", True),
          (300, 100, 64, "relu", False)]


@pytest.mark.parametrize("rows,cols,hidden,act,weight", BLOCKS)
def test_feed_forward(rows, cols, hidden, act, weight):
    say("feed forward %d x %d -> %d %s" % (rows, cols, hidden, act))
    rng = np.random.default_rng(rows + cols)
    block, want = _block(rng, rows, cols, hidden, act, weight)
    x, r = _values(rng, rows, cols), _values(rng, rows, cols)
    xs, rs = _share(rng, x, pad=4), _share(rng, r)
    out = _empty(rows, cols)
    assert block.eval2(xs, out, residual=rs) is out
    assert np.array_equal(_open(out), want(x, r))
    # Over the residual stream itself; prepared on another stream.
    side = torch.cuda.Stream()
    block.eval2(xs, rs, residual=rs, prep=(tasks.Prepared(side, [[], block.truncs()]), 1))
    assert all(torch.equal(a, b) for a, b in zip(rs, out))
    block.eval2(xs, xs)
    assert np.array_equal(_open(xs), want(x, None))


def _experts(rng, tokens, each, experts, cols, hidden, act):
    W = _weights(rng, 10, experts, cols, hidden), _weights(rng, 10, experts, hidden, cols)
    b = _bias(rng, experts, hidden), _bias(rng, experts, cols)
    block = ff.ExpertFeedForward(tokens, each, ff.PublicWeights(W[0], b[0]),
                                 ff.PublicWeights(W[1], b[1]), STATE, act=_act(act),
                                 seed=tokens + 1000)

    def want(x, residual, chosen, g):
        n = block.norm
        s, h = ref.rmsnorm(x, residual, n.inv_len, n.eps_q, n.table, F)
        out = np.zeros_like(s)
        with np.errstate(over="ignore"):
            for t in range(tokens):  # a token at a time, without any tables
                for e, w in zip(chosen[t], g[t]):
                    if 0 <= e < experts:
                        u, _ = ref.linear(h[t:t + 1], W[0][e], b[0][e], F, _act(act))
                        z, _ = ref.linear(u, W[1][e], b[1][e], F)
                        out[t] += z[0] * np.uint64(int(w) & ref.M64)
            return ref.floor_shift(out, F) + s
    return block, want


MIXED = [(1, 1, 1, 33, 40, "relu"), (1, 2, 8, 64, 128, "gelu"), (5, 3, 4, 96, 64, None),
         (60, 2, 7, 40, 72, "relu"), (400, 1, 2, 64, 64, "gelu")]


@pytest.mark.parametrize("tokens,each,experts,cols,hidden,act", MIXED)
def test_expert_feed_forward(tokens, each, experts, cols, hidden, act):
    say("expert feed forward %d tokens, %d of %d" % (tokens, each, experts))
    rng = np.random.default_rng(tokens + experts)
    block, want = _experts(rng, tokens, each, experts, cols, hidden, act)
    for k in range(2):  # another choice, with some in no expert, over the same buffers
        x, r = _values(rng, tokens, cols), _values(rng, tokens, cols)
        chosen = rng.integers(0 if k == 0 else -1, experts, (tokens, each))
        g = rng.integers(0, 2 ** F + 1, (tokens, each))
        tabs = ff.route(torch.from_numpy(chosen).cuda(), experts)
        out = block.eval2(_share(rng, x), _empty(tokens, cols), *tabs,
                          torch.from_numpy(g).cuda(), residual=_share(rng, r))
        assert np.array_equal(_open(out), want(x, r, chosen, g))


# ---- captured, and on other streams ----

def _replays(graph, load, out, eager, rounds=4):
    """Every replay against the eager result on the same inputs, with other work
    and synchronizations between."""
    for k in range(rounds):
        load(k)
        want = [t.clone() for t in eager()]
        for o in out:
            o.fill_(k)
        torch.cuda.synchronize()
        graph.replay()
        junk = torch.randn(1 << 16, device="cuda").sum()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), (k, float(junk))


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_captured_feed_forward(rows):
    say("captured feed forward, %d rows" % rows)
    rng = np.random.default_rng(rows)
    block, _ = _block(rng, rows, 96, 128, "gelu", True)
    xs, rs, out = _empty(rows, 96), _empty(rows, 96), _empty(rows, 96)
    inputs = [(_share(rng, _values(rng, rows, 96)), _share(rng, _values(rng, rows, 96)))
              for _ in range(4)]

    def load(k):
        for dst, src in zip(xs + rs, inputs[k][0] + inputs[k][1]):
            dst.copy_(src)
    load(0)
    graph = tasks.capture(lambda: block.eval2(xs, out, residual=rs))
    two = _empty(rows, 96)
    _replays(graph, load, out, lambda: block.eval2(xs, two, residual=rs))


def test_captured_experts():
    """The choice of experts may change between replays."""
    say("captured experts")
    rng = np.random.default_rng(5)
    tokens, each, experts, cols = 24, 2, 5, 64
    block, _ = _experts(rng, tokens, each, experts, cols, 96, "relu")
    xs, out, two = _share(rng, _values(rng, tokens, cols)), _empty(tokens, cols), \
        _empty(tokens, cols)
    tabs = ff.route(torch.zeros(tokens, each, dtype=torch.int64, device="cuda"), experts)
    g = torch.zeros(tokens, each, dtype=torch.int64, device="cuda")

    def load(k):
        chosen = torch.from_numpy(rng.integers(-1, experts, (tokens, each))).cuda()
        for dst, src in zip(tabs, ff.route(chosen, experts)):
            dst.copy_(src)
        g.copy_(torch.from_numpy(rng.integers(0, 4097, (tokens, each))))
    load(0)
    graph = tasks.capture(lambda: block.eval2(xs, out, *tabs, g))
    _replays(graph, load, out, lambda: block.eval2(xs, two, *tabs, g))


def test_captured_large_norm():
    say("captured large norm")
    rng = np.random.default_rng(6)
    rows, cols = 2100, 1000
    norm = ff.RMSNorm(rows, cols, STATE, seed=6)
    xs, out, two = _empty(rows, cols), _empty(rows, cols), _empty(rows, cols)
    inputs = [_share(rng, _values(rng, rows, cols)) for _ in range(3)]

    def load(k):
        for dst, src in zip(xs, inputs[k]):
            dst.copy_(src)
    load(0)
    graph = tasks.capture(lambda: norm.eval2(xs, out))
    _replays(graph, load, out, lambda: norm.eval2(xs, two), rounds=3)


def test_two_objects_on_two_streams():
    """Objects share nothing: their calls may run side by side."""
    say("two streams")
    rng = np.random.default_rng(7)
    made = [_block(rng, rows, 96, 160, act, True) for rows, act in ((30, "gelu"), (18, "relu"))]
    x = [_values(rng, b.rows, 96) for b, _ in made]
    xs = [_share(rng, v) for v in x]
    outs = [_empty(b.rows, 96) for b, _ in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(3):
        for (block, _), s, i, o in zip(made, streams, xs, outs):
            with torch.cuda.stream(s):
                block.eval2(i, o)
    torch.cuda.synchronize()
    for (_, want), v, o in zip(made, x, outs):
        assert np.array_equal(_open(o), want(v, None))


def test_objects_of_a_busy_stream():
    """Made on a stream with work before them, used on another at once."""
    say("objects of a busy stream")
    rng = np.random.default_rng(23)
    x = _values(rng, 50, 70)
    xs = _share(rng, x)
    weights = _weights(rng, 10, 70, 40)
    torch.cuda.synchronize()
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(20000000)
        digits = ff.Digits(50, 70)
        torch.cuda._sleep(20000000)
        lin = ff.Linear(ff.PublicWeights(weights), 50, STATE, seed=23)
        outs = ff.Digits(50, 40)
    with torch.cuda.stream(other):
        lin.eval2(digits.split(xs), None, digits=outs)
    torch.cuda.synchronize()
    assert np.array_equal(_open(outs.values()), ref.linear(x, weights, None, F)[0])


# ---- each operator at its edges ----

@pytest.mark.parametrize("rows,cols,weight", [(5, 40, True), (600, 1501, True), (2100, 1000, False),
                                              (1000, 2100, True)])
def test_norm_prepared_elsewhere_and_outputs_alone(rows, cols, weight):
    say("norm %d x %d, prepared" % (rows, cols))
    rng = np.random.default_rng(cols)
    x, r = _values(rng, rows, cols), _values(rng, rows, cols)
    w = np.rint(rng.standard_normal(cols) * 2 ** F).astype(np.int64) if weight else None
    norm = ff.RMSNorm(rows, cols, STATE, weight=w, seed=9)
    xs, rs, out = _share(rng, x), _share(rng, r), _empty(rows, cols)
    norm.eval2(xs, out, residual=rs)
    assert np.array_equal(_open(out), ref.rmsnorm(x, r, norm.inv_len, norm.eps_q, norm.table, F,
                                                  w)[1])
    want = [o.clone() for o in out]
    prep = (tasks.Prepared(torch.cuda.Stream(), [norm.truncs()]), 0)
    norm.eval2(xs, out, residual=rs, prep=prep)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    digits = ff.Digits(rows, cols)
    norm.eval2(xs, None, residual=rs, digits=digits)
    assert all(torch.equal(a, b) for a, b in zip(digits.values(), want))
    total = _empty(rows, cols)
    norm.eval2(xs, None, residual=rs, total=total)
    assert all(torch.equal(t, a + b) for t, a, b in zip(total, xs, rs))


@pytest.mark.parametrize("rows,cols", [(2100, 1000), (300, 7001)])
def test_large_norm_in_place(rows, cols):
    say("large norm in place, %d x %d" % (rows, cols))
    rng = np.random.default_rng(rows)
    x, r = _values(rng, rows, cols), _values(rng, rows, cols)
    norm = ff.RMSNorm(rows, cols, STATE, seed=20)
    xs, rs = _share(rng, x), _share(rng, r)
    norm.eval2(xs, xs, residual=rs, total=rs)
    s, want = ref.rmsnorm(x, r, norm.inv_len, norm.eps_q, norm.table, F)
    assert np.array_equal(_open(rs), s) and np.array_equal(_open(xs), want)
    xs = _share(rng, x)
    norm.eval2(xs, xs)
    assert np.array_equal(_open(xs), ref.rmsnorm(x, None, norm.inv_len, norm.eps_q, norm.table,
                                                 F)[1])


@pytest.mark.parametrize("f", [9, 13])
@pytest.mark.parametrize("weight", [False, True])
def test_large_norm_other_fraction(f, weight):
    """Gates whose tables are small, and those that LDS does not take."""
    say("large norm f=%d weight=%s" % (f, weight))
    rng = np.random.default_rng(f)
    rows, cols = 2100, 1000
    x = _values(rng, rows, cols, f=f)
    w = np.rint(rng.standard_normal(cols) * 2 ** f).astype(np.int64) if weight else None
    norm = ff.RMSNorm(rows, cols, STATE, frac_bits=f, weight=w, seed=10)
    out = norm.eval2(_share(rng, x), _empty(rows, cols))
    assert np.array_equal(_open(out), ref.rmsnorm(x, None, norm.inv_len, norm.eps_q, norm.table,
                                                  f, w)[1])


@pytest.mark.parametrize("rows,cols", [(9, 70), (2100, 1001)])
def test_columns_of_one_matrix(rows, cols):
    """Inputs and outputs as columns of one wider matrix, nothing else of which
    is written."""
    say("columns of one matrix, %d x %d" % (rows, cols))
    rng = np.random.default_rng(rows)
    x, r = _values(rng, rows, cols), _values(rng, rows, cols)
    wide = torch.full((rows, 8 * cols + 9), -7, dtype=torch.int64, device="cuda")
    part = [wide[:, k * (cols + 1) + 1:k * (cols + 1) + 1 + cols] for k in range(8)]
    for k, t in enumerate(_share(rng, x) + _share(rng, r)):
        part[k].copy_(t)
    before = wide.clone()
    norm = ff.RMSNorm(rows, cols, STATE, seed=11)
    norm.eval2(part[0:2], part[4:6], residual=part[2:4], total=part[6:8])
    s, want = ref.rmsnorm(x, r, norm.inv_len, norm.eps_q, norm.table, F)
    assert np.array_equal(_open(part[4:6]), want) and np.array_equal(_open(part[6:8]), s)
    W = _weights(rng, 10, cols, cols)
    lin = ff.Linear(ff.PublicWeights(W), rows, STATE, seed=12)
    lin.eval2(part[0:2], part[4:6], residual=part[2:4])
    assert np.array_equal(_open(part[4:6]), ref.linear(x, W, None, F, residual=r)[0])
    mix = ff.ExpertMix(rows, cols, STATE, seed=13)
    slots = rng.integers(0, rows, (rows, 2))
    g = rng.integers(0, 4096, (rows, 2))
    mix.eval2(part[0:2], _i32(slots), torch.from_numpy(g).cuda(), part[6:8], residual=part[2:4])
    assert np.array_equal(_open(part[6:8]), ref.mix(x, slots, g, F, r))
    for p in part[4:8]:
        p.fill_(-7)
    assert torch.equal(wide, before)


def test_rows_past_32_bit_offsets():
    """Rows 2^29 words apart: the last ones begin past 2^31 words.  (One buffer
    of 24 GiB, of which the rows' columns alone are touched.)"""
    say("far rows")
    rng = np.random.default_rng(14)
    rows, cols, stride = 6, 64, (1 << 29) + 16
    wide = torch.empty((rows - 1) * stride + 8 * cols, dtype=torch.int64, device="cuda")
    part = [wide.as_strided((rows, cols), (stride, 1), k * cols) for k in range(8)]
    x, r = _values(rng, rows, cols), _values(rng, rows, cols)
    for k, t in enumerate(_share(rng, x) + _share(rng, r)):
        part[k].copy_(t)
    norm = ff.RMSNorm(rows, cols, STATE, seed=14)
    norm.eval2(part[0:2], part[4:6], residual=part[2:4], total=part[6:8])
    s, want = ref.rmsnorm(x, r, norm.inv_len, norm.eps_q, norm.table, F)
    assert np.array_equal(_open(part[4:6]), want) and np.array_equal(_open(part[6:8]), s)
    W = _weights(rng, 10, cols, cols)
    lin = ff.Linear(ff.PublicWeights(W), rows, STATE, seed=15)
    lin.eval2(part[0:2], part[4:6], residual=part[2:4])
    assert np.array_equal(_open(part[4:6]), ref.linear(x, W, None, F, residual=r)[0])
    digits = ff.Digits(rows, cols).split(part[0:2])
    assert all(torch.equal(a, b) for a, b in zip(digits.values(), part[0:2]))
    mix = ff.ExpertMix(rows, cols, STATE, seed=16)
    slots, g = np.arange(rows)[::-1, None].copy(), rng.integers(0, 4096, (rows, 1))
    mix.eval2(part[0:2], _i32(slots), torch.from_numpy(g).cuda(), part[6:8], residual=part[2:4])
    assert np.array_equal(_open(part[6:8]), ref.mix(x, slots, g, F, r))


@pytest.mark.parametrize("rows,N", [(1, 768), (4, 4000), (40, 256), (250, 300)])
def test_linear_prepared_elsewhere(rows, N):
    """The walks beside the product, before it and on another stream give the
    same shares."""
    say("linear prepared, %d x %d" % (rows, N))
    rng = np.random.default_rng(N)
    x, W = _values(rng, rows, 256), _weights(rng, 12, 256, N)
    xs = _share(rng, x)
    for act in (None, "relu", _act("gelu")):
        lin = ff.Linear(ff.PublicWeights(W), rows, STATE, act=act, seed=17)
        out = lin.eval2(xs, _empty(rows, N))
        assert np.array_equal(_open(out), ref.linear(x, W, None, F, act)[0])
        prep = (tasks.Prepared(torch.cuda.Stream(), [lin.truncs()]), 0)
        again = lin.eval2(xs, _empty(rows, N), prep=prep)
        assert all(torch.equal(a, b) for a, b in zip(again, out))


def test_linear_of_broadcast_and_repeated_rows():
    """One row for all, a bias-like residual, the same x row many times."""
    say("broadcast rows")
    rng = np.random.default_rng(18)
    x, r, W = _values(rng, 1, 100), _values(rng, 1, 70), _weights(rng, 12, 100, 70)
    xs, rs = _share(rng, x), _share(rng, r)
    lin = ff.Linear(ff.PublicWeights(torch.from_numpy(W).cuda()), 21, STATE, seed=18)
    want = np.repeat(ref.linear(x, W, None, F, residual=r)[0], 21, 0)
    out = lin.eval2(tuple(t.expand(21, 100) for t in xs), _empty(21, 70),
                    residual=tuple(t.expand(21, 70) for t in rs))
    assert np.array_equal(_open(out), want)
    out = lin.eval2(xs, _empty(21, 70), residual=tuple(t.expand(21, 70) for t in rs),
                    rows=torch.zeros(21, dtype=torch.int32, device="cuda"))
    assert np.array_equal(_open(out), want)


def test_eval2_refuses():
    """On the host, before any launch."""
    say("refusals")
    rng = np.random.default_rng(19)
    norm = ff.RMSNorm(3, 40, STATE, seed=1)
    weights = ff.PublicWeights(_weights(rng, 10, 40, 24))
    lin = ff.Linear(weights, 3, STATE, x_rows=5, seed=2)
    grouped = ff.Linear(ff.PublicWeights(_weights(rng, 10, 2, 40, 24)), 3, STATE, seed=3)
    mix = ff.ExpertMix(3, 24, STATE, seed=4)
    x, y = _empty(3, 40), _empty(3, 24)
    slots = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    g = torch.zeros(3, 2, dtype=torch.int64, device="cuda")
    off = _i32([0, 1, 3])
    cpu = tuple(t.cpu() for t in x)
    for call in (
            lambda: norm.eval2(y, x), lambda: norm.eval2(x, None), lambda: norm.eval2(cpu, x),
            lambda: norm.eval2(x, tuple(t.int() for t in x)),
            lambda: norm.eval2(x, _empty(3, 40), residual=x[0]),
            lambda: norm.eval2(x, _empty(3, 40), digits=ff.Digits(3, 41)),
            lambda: norm.eval2(x, tuple(t[:1].expand(3, 40) for t in x)),
            lambda: norm.eval2(x, _empty(3, 40), total=(x[1], x[0])),
            lambda: lin.eval2(y, y), lambda: lin.eval2(None, y), lambda: lin.eval2(x, x),
            lambda: lin.eval2(x, None), lambda: lin.eval2(x, y, offsets=off),
            lambda: lin.eval2(_empty(2, 40), y), lambda: lin.eval2(_empty(6, 40), y),
            lambda: lin.eval2(x, y, rows=slots[:, 0]),
            lambda: lin.eval2(x, y, rows=torch.zeros(3, dtype=torch.int64, device="cuda")),
            lambda: lin.eval2(ff.Digits(3, 41), y), lambda: lin.eval2(x, y, digits=y),
            lambda: lin.eval2(x, y, residual=(y[1], y[0])),
            lambda: grouped.eval2(x, y), lambda: grouped.eval2(x, y, offsets=off.cpu()),
            lambda: grouped.eval2(x, y, offsets=off.long()),
            lambda: mix.eval2(y, slots, g, y), lambda: mix.eval2(None, slots, g, y),
            lambda: mix.eval2(y, slots.long(), g, _empty(3, 24)),
            lambda: mix.eval2(y, slots, g[:, :1], _empty(3, 24)),
            lambda: mix.eval2(x, slots, g, y)):
        with pytest.raises((ValueError, RuntimeError)):
            call()
    torch.cuda.synchronize()
    assert all(bool((t == -7).all()) for t in x + y)


# ---- many rows: 256 columns a workgroup ----

MANY = [
    # rows, K, N, bits, act, residual, digits in; one to five chunks of 64 k
    (400, 40, 2100, 12, None, True, True),
    (1603, 96, 500, 6, "relu", False, False),
    (393, 200, 2050, 13, "gelu", True, False),
    (410, 130, 1999, 7, None, False, True),
    (3100, 300, 256, 12, "relu", True, True),
    (395, 64, 2049, 22, None, True, False),  # three digits: 128 columns
]


@pytest.mark.parametrize("rows,K,N,bits,act,residual,split", MANY)
def test_linear_many_rows(rows, K, N, bits, act, residual, split):
    say("linear %dx%dx%d bits=%d act=%s digits=%s" % (rows, K, N, bits, act, split))
    rng = np.random.default_rng(rows + K)
    x, W = _values(rng, rows, K), _weights(rng, bits, K, N)
    W.flat[0], W.flat[-1] = -2 ** bits, 2 ** bits - 1
    bias = _bias(rng, N)
    res = _values(rng, rows, N) if residual else None
    lin = ff.Linear(ff.PublicWeights(W, bias), rows, STATE, act=_act(act), seed=21)
    xs = _share(rng, x, pad=6)
    out, digits = _empty(rows, N), ff.Digits(rows, N)
    lin.eval2(ff.Digits(rows, K).split(xs) if split else xs, out, digits=digits,
              residual=None if res is None else _share(rng, res))
    assert np.array_equal(_open(out), ref.linear(x, W, bias, F, _act(act), res)[0])
    assert all(torch.equal(a, b) for a, b in zip(digits.values(), out))


@pytest.mark.parametrize("bits", [7, 12])
@pytest.mark.parametrize("split", [False, True])
def test_experts_many_rows(bits, split):
    """Ragged experts, one without rows; rows in no expert between guard rows."""
    say("experts, many rows, bits=%d digits=%s" % (bits, split))
    rng = np.random.default_rng(bits)
    n_rows, T, K, N, E = 2500, 700, 70, 1000, 6
    off = np.array([3, 900, 900, 1001, 1003, 2200, 2491])
    src = rng.integers(-1, T + 1, n_rows)
    x, W, bias = _values(rng, T, K), _weights(rng, bits, E, K, N), _bias(rng, E, N)
    lin = ff.Linear(ff.PublicWeights(W, bias), n_rows, STATE, x_rows=T, seed=22)
    xs = _share(rng, x)
    out = _empty(n_rows, N)
    lin.eval2(ff.Digits(T, K).split(xs) if split else xs, out, offsets=_i32(off), rows=_i32(src))
    want, written = ref.linear(x, W, bias, F, offsets=off, rows=src)
    assert np.array_equal(_open(out)[written], want[written])
    assert all(bool((o[~torch.from_numpy(written)] == -7).all()) for o in out)
