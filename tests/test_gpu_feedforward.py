"""RMSNorm, Linear (dense and by expert) and ExpertMix on the GPU.

Reconstruction: equal, bit for bit, to the definitions in whole numbers
(tests/feedforward_reference.py).  Shares: equal to the same material run
through the framework's other entry points one step at a time."""
import numpy as np
import pytest
import torch

import feedforward_reference as ref
import oracle_lib as ol
from gpu_util import dev, say, u64
from suf_amd import feedforward as ff
from suf_amd import native, tables, tasks

pytestmark = pytest.mark.gpu

STATE = ol.mt64_bytes(3, ol.PRG_STATE_BYTES).tobytes()
F = 12


@pytest.fixture(scope="module", autouse=True)
def _init():
    native.call("sufhip_init", 0)


def _values(rng, *shape, sigma=1.0, f=F):
    return np.rint(rng.standard_normal(shape) * sigma * 2 ** f).astype(np.int64).view(np.uint64)


def _words(rng, *shape):
    return rng.integers(0, 1 << 64, shape, dtype=np.uint64)


def _share(rng, v, pad=0):
    """Shares of v on the GPU; pad: as columns of wider rows."""
    s = _words(rng, *v.shape)
    out = []
    for h in (s, v - s):
        wide = _words(rng, v.shape[0], v.shape[1] + pad)
        wide[:, pad // 2:pad // 2 + v.shape[1]] = h
        out.append(dev(wide)[:, pad // 2:pad // 2 + v.shape[1]])
    return tuple(out)


def _open(pair):
    with np.errstate(over="ignore"):
        return u64(pair[0].contiguous()) + u64(pair[1].contiguous())


def _empty(*shape):
    return tuple(torch.full(shape, -7, dtype=torch.int64, device="cuda") for _ in range(2))


# ---- the norm ----

NORM_SHAPES = [(1, 1), (1, 768), (3, 33), (5, 64), (2, 255), (7, 1000), (4, 1024), (3, 1025),
               (300, 96), (2, 2048), (2, 2049), (3, 4096), (2, 4097), (1, 9001),
              # in three launches (2^21 values and more): waves and workgroups a row
              (2100, 1000), (70000, 30), (1000, 2100), (30, 70001)]


@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("weight", [False, True])
def test_norm(rows, cols, weight):
    say("norm %d x %d weight=%s" % (rows, cols, weight))
    rng = np.random.default_rng(rows * 10007 + cols)
    # Rows of different sizes, one of zeros.
    x = _values(rng, rows, cols) * np.uint64(3)
    r = _values(rng, rows, cols)
    with np.errstate(over="ignore"):
        if rows > 1:
            x[1] = np.uint64(0) - r[1]
    if rows > 2:
        x[2] = _values(rng, cols, sigma=20.0)
    w = np.rint((1 + 0.3 * rng.standard_normal(cols)) * 2 ** F).astype(np.int64) if weight else None
    pad = 6 if cols % 2 else 0
    xs, rs = _share(rng, x, pad), _share(rng, r)
    norm = ff.RMSNorm(rows, cols, STATE, weight=None if w is None else torch.from_numpy(w), seed=5)
    total, out = _empty(rows, cols), _empty(rows, cols)
    digits = ff.Digits(rows, cols)
    norm.eval2(xs, out, residual=rs, total=total, digits=digits)
    torch.cuda.synchronize()
    s, want = ref.rmsnorm(x, r, norm.inv_len, norm.eps_q, norm.table, F, w)
    assert np.array_equal(_open(total), s)
    for p in range(2):
        assert torch.equal(total[p], xs[p] + rs[p])
    assert np.array_equal(_open(out), want)
    got = digits.values()
    assert torch.equal(got[0], out[0]) and torch.equal(got[1], out[1])


@pytest.mark.parametrize("cols", [40, 1500, 5000])
def test_norm_without_residual_and_in_place(cols):
    say("norm in place, %d" % cols)
    rng = np.random.default_rng(cols)
    x, r = _values(rng, 3, cols), _values(rng, 3, cols)
    norm = ff.RMSNorm(3, cols, STATE, seed=6)
    xs = _share(rng, x)
    norm.eval2(xs, xs)
    assert np.array_equal(_open(xs), ref.rmsnorm(x, None, norm.inv_len, norm.eps_q, norm.table,
                                                 F)[1])
    # The stream's sum over the residual, the output over x.
    xs, rs = _share(rng, x), _share(rng, r)
    norm.eval2(xs, xs, residual=rs, total=rs)
    s, want = ref.rmsnorm(x, r, norm.inv_len, norm.eps_q, norm.table, F)
    assert np.array_equal(_open(rs), s) and np.array_equal(_open(xs), want)


@pytest.mark.parametrize("f", [8, 13])
def test_norm_other_fraction(f):
    say("norm f=%d" % f)
    rng = np.random.default_rng(f)
    x = _values(rng, 4, 100, f=f)
    norm = ff.RMSNorm(4, 100, STATE, frac_bits=f, seed=7)
    out = _empty(4, 100)
    norm.eval2(_share(rng, x), out)
    assert np.array_equal(_open(out), ref.rmsnorm(x, None, norm.inv_len, norm.eps_q, norm.table,
                                                  f)[1])


def test_norm_is_a_norm():
    """Against real numbers: the mean square of the output is 1.  Off by the
    Newton step's 1.5 e^2 (e: the table's 0.06 on an octave's chord), y's
    steps of 2^-12 (1.5 of them at y = 1/8, the largest rows here), and the
    floors of two gates: 2^-12 each on values of size 1."""
    say("norm against real numbers")
    rng = np.random.default_rng(8)
    rows, cols = 12, 768
    x = np.stack([_values(rng, cols, sigma=2.0 ** (k / 2 - 2)) for k in range(rows)])
    norm = ff.RMSNorm(rows, cols, STATE, seed=8)
    out = _empty(rows, cols)
    norm.eval2(_share(rng, x), out)
    real = x.view(np.int64) / 2.0 ** F
    want = real / np.sqrt((real ** 2).mean(1, keepdims=True) + norm.eps_q / 2.0 ** F)
    got = _open(out).view(np.int64) / 2.0 ** F
    rel = 1.5 * 0.0625 ** 2 + 4 * 8 * 2.0 ** -F
    assert np.all(np.abs(got - want) <= rel * np.abs(want) + 3 * 2.0 ** -F)


def test_norm_shares_step_by_step():
    """The same material through row sums, products and gates of their own."""
    say("norm shares")
    rng = np.random.default_rng(9)
    rows, cols = 5, 70
    x = _values(rng, rows, cols)
    xs = _share(rng, x)
    norm = ff.RMSNorm(rows, cols, STATE, weight=torch.full((cols,), 5000), seed=9)
    out = _empty(rows, cols)
    norm.eval2(xs, out)
    torch.cuda.synchronize()

    def gate(tr, z0, z1, n):
        y = tasks.pair(n)
        with np.errstate(over="ignore"):
            tr.finish(dev((z0 + z1 + np.uint64(tr.mask)).ravel()), y)
        return u64(y[0]), u64(y[1])

    with np.errstate(over="ignore"):
        x0, x1 = u64(xs[0]), u64(xs[1])
        a0, a1, b0, b1 = (u64(t) for t in norm.a + norm.b)
        D = (x0 - a0) + (x1 - a1)
        two = np.uint64(2)
        s0 = (two * D * a0 + D * D).sum(1, dtype=np.uint64) + u64(norm.a2[0])
        s1 = (two * D * a1).sum(1, dtype=np.uint64) + u64(norm.a2[1])
        m = gate(norm.tr_ms[0], s0, s1, rows)
        inv = np.uint64(norm.inv_len)
        m = gate(norm.tr_ms[1], m[0] * inv, m[1] * inv, rows)
        m = gate(norm.tr_ms[2], m[0], m[1], rows)
        v = (dev(m[0] + np.uint64(norm.eps_q)), dev(m[1]))
        y = tasks.pair(rows)
        tasks.chain2(native.CHAIN_RSQRT, F, tasks.operand(tasks.term(v)), rows, norm.lut.keys,
                     norm.lut.key_bytes, norm.lut.intervals, norm.lut.mask, norm.tri,
                     norm.tr_rsqrt, y)
        E = ((u64(y[0]) - b0) + (u64(y[1]) - b1))[:, None]
        z0 = u64(norm.ab[0]) + D * b0[:, None] + a0 * E + D * E
        z1 = u64(norm.ab[1]) + D * b1[:, None] + a1 * E
        o = gate(norm.tr_norm, z0, z1, rows * cols)
        w = np.uint64(5000)
        o = gate(norm.tr_weight, o[0] * w, o[1] * w, rows * cols)
    for p in range(2):
        assert np.array_equal(u64(out[p]).ravel(), o[p])


# ---- products ----

def _weights(rng, bits, *shape):
    w = np.rint(rng.standard_normal(shape) * 2.0 ** (bits - 2))
    return np.clip(w, -2 ** bits, 2 ** bits - 1).astype(np.int64)


def _table():
    return tables.gelu_table(F)


LINEAR = [
    # rows, K, N, bits, act, residual, digits in
    (1, 1, 1, 6, None, False, False),
    (1, 768, 130, 12, None, True, False),
    (2, 100, 64, 7, None, False, True),
    (3, 64, 65, 12, "relu", True, False),
    (8, 130, 96, 15, None, True, False),
    (9, 95, 200, 12, None, False, False),
    (16, 256, 64, 22, "gelu", True, False),
    (17, 64, 33, 12, None, True, True),
    (31, 33, 40, 30, None, False, False),
    (32, 500, 128, 12, "relu", False, True),
    (33, 64, 128, 12, None, True, False),
    (64, 31, 129, 7, None, False, False),
    (65, 200, 300, 15, "gelu", True, False),
    (100, 1000, 70, 22, None, True, True),
    (130, 96, 256, 30, "relu", True, False),
    (257, 320, 64, 12, None, False, False),
]


@pytest.mark.parametrize("rows,K,N,bits,act,residual,split", LINEAR)
def test_linear(rows, K, N, bits, act, residual, split):
    say("linear %dx%dx%d bits=%d act=%s residual=%s digits=%s" % (rows, K, N, bits, act, residual,
                                                                 split))
    rng = np.random.default_rng(rows * 1000003 + K * 101 + N)
    act = _table() if act == "gelu" else act
    x = _values(rng, rows, K)
    W = _weights(rng, bits, K, N)
    W.flat[0], W.flat[-1] = -2 ** bits, 2 ** bits - 1
    # Values of moderate size whatever the weights': their scale is taken off.
    bias = (_values(rng, N) << np.uint64(F)).view(np.int64)
    res = _values(rng, rows, N) if residual else None
    weights = ff.PublicWeights(W, bias)
    lin = ff.Linear(weights, rows, STATE, act=act, seed=11)
    xs = _share(rng, x, pad=10)
    src = ff.Digits(rows, K).split(xs) if split else xs
    out = _empty(rows, N + 3)
    view = tuple(o[:, 1:1 + N] for o in out)
    digits = ff.Digits(rows, N)
    rs = None if res is None else _share(rng, res)
    want, _ = ref.linear(x, W, bias, F, act, res)
    lin.eval2(src, view, residual=rs)
    torch.cuda.synchronize()
    assert np.array_equal(_open(view), want)
    for o in out:  # nothing beside the columns
        assert bool((o[:, 0] == -7).all()) and bool((o[:, 1 + N:] == -7).all())
    shares = [o.clone() for o in view]
    lin.eval2(src, view, residual=rs, digits=digits)
    for o, s, d in zip(view, shares, digits.values()):
        assert torch.equal(o, s) and torch.equal(d, s)


@pytest.mark.parametrize("rows,K,N,digits", [(1, 70, 100, 2), (12, 300, 64, 1), (40, 64, 130, 4),
                                             (96, 1024, 256, 3)])
def test_product_is_exact_on_any_words(rows, K, N, digits):
    """Uniform words and weights of every digit, the extremes among them."""
    say("exact product %dx%dx%d digits=%d" % (rows, K, N, digits))
    rng = np.random.default_rng(K)
    x = _words(rng, rows, K)
    x.flat[0], x.flat[-1] = np.uint64(1 << 63), np.uint64(0x8080808080808080)
    lo, hi = -(128 * (256 ** digits - 1) // 255), 127 * (256 ** digits - 1) // 255
    W = rng.integers(lo, hi + 1, (K, N))
    W.flat[0], W.flat[-1] = lo, hi
    weights = ff.PublicWeights(torch.from_numpy(W).cuda())
    assert weights.digits == digits
    lin = ff.Linear(weights, rows, STATE, trunc=False, seed=12)
    xs = _share(rng, x)
    out = lin.eval2(xs, _empty(rows, N))
    for p in range(2):
        assert np.array_equal(u64(out[p]), ref.matmul(u64(xs[p]), W))


def test_product_of_the_largest_digits():
    """Every digit product at its largest, over as many rows of W as 4 digits
    allow: the sums in int32 stay exact."""
    say("largest digits")
    K, N = 32767, 64
    x = np.full((1, K), 0x7f7f7f7f7f7f7f80, np.uint64)  # eight digits of -128
    W = np.full((K, N), -(128 * (256 ** 4 - 1) // 255), np.int64)
    zero = tuple(torch.zeros(1, K, dtype=torch.int64, device="cuda") for _ in range(2))
    for v in (x, np.full((1, K), 0x8080808080808080, np.uint64)):
        xs = (dev(v), zero[1])
        out = ff.Linear(ff.PublicWeights(W), 1, STATE, trunc=False, seed=13).eval2(
            xs, _empty(1, N))
        assert np.array_equal(u64(out[0]), ref.matmul(v, W))


@pytest.mark.parametrize("rows", [1, 20, 70])
@pytest.mark.parametrize("act", ["relu", "gelu"])
def test_linear_shares_step_by_step(rows, act):
    say("linear shares rows=%d act=%s" % (rows, act))
    rng = np.random.default_rng(rows)
    K, N = 96, 50
    n = rows * N
    W = _weights(rng, 12, K, N)
    xs = _share(rng, _values(rng, rows, K))
    lin = ff.Linear(ff.PublicWeights(W), rows, STATE, act=_table() if act == "gelu" else act,
                    seed=14)
    out = lin.eval2(xs, _empty(rows, N))
    with np.errstate(over="ignore"):
        z = ref.matmul(u64(xs[0]), W) + ref.matmul(u64(xs[1]), W) + np.uint64(lin.tr.mask)
    y = tasks.pair(n)
    lin.tr.finish(dev(z.ravel()), y)
    if act == "gelu":
        o = tasks.pair(n)
        tasks.chain2(native.CHAIN_CUBIC, F, tasks.operand(tasks.term(y)), n, lin.lut.keys,
                     lin.lut.key_bytes, lin.lut.intervals, lin.lut.mask, lin.tri, lin.tr_act, o)
    else:
        c = tasks.pair(n, width=2)
        lin.lut.eval2(None, n, c, x=tasks.operand(tasks.term(y)))
        xh = y[0] + y[1] + torch.tensor(lin.lut.mask, dtype=torch.uint64).view(torch.int64).cuda()
        o = [t.view(n, 2)[:, 0] + t.view(n, 2)[:, 1] * xh for t in c]
    for p in range(2):
        assert torch.equal(out[p].reshape(-1), o[p])


# ---- by expert ----

EXPERTS = [
    # tokens, each, experts, K, N, act
    (1, 1, 4, 64, 64, None),
    (1, 2, 3, 100, 70, "relu"),
    (5, 2, 8, 64, 130, None),
    (8, 2, 70, 33, 40, None),
    (40, 4, 4, 96, 64, "gelu"),
    (200, 2, 5, 64, 100, None),
    (150, 3, 9, 130, 200, "relu"),
    (64, 1, 1, 64, 64, None),
]


@pytest.mark.parametrize("tokens,each,experts,K,N,act", EXPERTS)
def test_experts(tokens, each, experts, K, N, act):
    say("experts tokens=%d each=%d experts=%d %dx%d %s" % (tokens, each, experts, K, N, act))
    rng = np.random.default_rng(tokens * 31 + experts)
    off, rows, slots = ref.routing(rng, tokens, each, experts)
    x = _values(rng, tokens, K)
    W = _weights(rng, 12, experts, K, N)
    bias = (_values(rng, experts, N) << np.uint64(F)).view(np.int64)
    table = _table() if act == "gelu" else act
    lin = ff.Linear(ff.PublicWeights(W, bias), tokens * each, STATE, act=table, x_rows=tokens,
                    seed=15)
    out = lin.eval2(_share(rng, x), _empty(tokens * each, N),
                    offsets=torch.from_numpy(off.astype(np.int32)).cuda(),
                    rows=torch.from_numpy(rows.astype(np.int32)).cuda())
    want, _ = ref.linear(x, W, bias, F, table, offsets=off, rows=rows)
    assert np.array_equal(_open(out), want)
    # ... and the sum of each token's, with a residual.
    mix = ff.ExpertMix(tokens, N, STATE, seed=16)
    g = rng.integers(-4096, 4096, (tokens, each))
    res = _values(rng, tokens, N)
    y = mix.eval2(out, torch.from_numpy(slots.astype(np.int32)).cuda(), torch.from_numpy(g).cuda(),
                  _empty(tokens, N), residual=_share(rng, res))
    assert np.array_equal(_open(y), ref.mix(want, slots, g, F, res))


@pytest.mark.parametrize("n_rows", [6, 50, 400])
@pytest.mark.parametrize("act", [None, "relu"])
def test_rows_in_no_expert_are_left(n_rows, act):
    """Experts without rows, rows before the first and after the last expert,
    x rows that are not there."""
    say("rows in no expert, %d, %s" % (n_rows, act))
    rng = np.random.default_rng(n_rows)
    K, N = 64, 72
    off = np.array([1, 1, n_rows // 2, n_rows // 2, n_rows // 2, n_rows - 2])
    src = rng.integers(-2, 9, n_rows)
    src[1], src[2] = -2 ** 31, 2 ** 31 - 1
    x = _values(rng, 7, K)
    W = _weights(rng, 12, 5, K, N)
    lin = ff.Linear(ff.PublicWeights(W), n_rows, STATE, act=act, x_rows=7, seed=17)
    xs = _share(rng, x)
    digits = ff.Digits(7, K).split(xs)
    want, written = ref.linear(x, W, None, F, act, offsets=off, rows=src)
    assert written.sum() == n_rows - 3
    for source in (xs, digits):
        out, od = _empty(n_rows, N), ff.Digits(n_rows, N)
        for kw in ({}, {"digits": od}):
            lin.eval2(source, out, offsets=torch.from_numpy(off.astype(np.int32)).cuda(),
                      rows=torch.from_numpy(src.astype(np.int32)).cuda(), **kw)
            assert np.array_equal(_open(out)[written], want[written])
            assert bool((out[0][~torch.from_numpy(written)] == -7).all())
        got = od.values()
        assert torch.equal(got[0][written], out[0][written])
        assert not bool(got[0][~torch.from_numpy(written)].any())


@pytest.mark.parametrize("off", [[0, 0, 0, 0], [5, 3, 9, 1], [-7, 2, 2 ** 31 - 1, 40],
                                 [2 ** 31 - 1, -2 ** 31, 4, 4], [0, 40, 0, 40]])
@pytest.mark.parametrize("rows", [7, 40, 200])
def test_wrong_offsets_stay_inside(off, rows):
    """Offsets that are not what they should be give some values, in bounds:
    the rows around the output are untouched."""
    say("offsets %s rows %d" % (off, rows))
    rng = np.random.default_rng(rows)
    lin = ff.Linear(ff.PublicWeights(_weights(rng, 12, 3, 64, 64)), rows, STATE, seed=18)
    wide = _empty(rows + 64, 64)
    lin.eval2(_share(rng, _values(rng, rows, 64)), tuple(w[32:32 + rows] for w in wide),
              offsets=torch.tensor(off, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    for w in wide:
        assert bool((w[:32] == -7).all()) and bool((w[32 + rows:] == -7).all())


@pytest.mark.parametrize("tokens,each,cols", [(1, 1, 1), (1, 2, 1024), (7, 3, 33), (40, 8, 130),
                                              (3, 0, 20), (300, 2, 65), (1050, 3, 1001)])
def test_mix(tokens, each, cols):
    say("mix %d %d %d" % (tokens, each, cols))
    rng = np.random.default_rng(tokens + cols)
    z = _values(rng, tokens * each + 2, cols)
    slots = rng.integers(-1, tokens * each + 3, (tokens, each))
    if each > 1:
        slots[0, 1] = slots[0, 0]  # the same row twice
    w = rng.integers(-2 ** 13, 2 ** 13, (tokens, each))
    mix = ff.ExpertMix(tokens, cols, STATE, seed=19)
    zs = _share(rng, z, pad=4)
    s32, w64 = torch.from_numpy(slots.astype(np.int32)).cuda(), torch.from_numpy(w).cuda()
    out = mix.eval2(zs, s32, w64, _empty(tokens, cols))
    assert np.array_equal(_open(out), ref.mix(z, slots, w, F))
    res = _values(rng, tokens, cols)
    rs = _share(rng, res)
    mix.eval2(zs, s32, w64, rs, residual=rs)  # in place
    assert np.array_equal(_open(rs), ref.mix(z, slots, w, F, res))


def test_per_party_keystreams():
    """The same shares when each party computes its own keystream."""
    say("per-party keystreams")
    rng = np.random.default_rng(20)
    x = _values(rng, 9, 64)
    W = _weights(rng, 12, 64, 48)
    xs = _share(rng, x)
    for act in ("relu", _table()):
        lin = ff.Linear(ff.PublicWeights(W), 9, STATE, act=act, seed=20)
        norm = ff.RMSNorm(9, 64, STATE, seed=21)
        got = []
        for own in (0, 1):
            native.call("sufhip_set_keystream_per_party", own)
            try:
                got.append([t.clone() for t in
                            lin.eval2(xs, _empty(9, 48)) + norm.eval2(xs, _empty(9, 64))])
                torch.cuda.synchronize()
            finally:
                native.call("sufhip_set_keystream_per_party", 0)
        assert all(torch.equal(a, b) for a, b in zip(*got))
