"""The feed-forward operators on the CPU: what they refuse before any device
work, the layouts' sizes, the norm's table, the tables of a choice of experts.

Every call here is refused or has nothing to do: no address is read."""
import ctypes

import numpy as np
import pytest
import torch

import feedforward_reference as ref
from suf_amd import feedforward as ff
from suf_amd import native, tables

AT = 1 << 32  # addresses that nothing here reads, 2^32 bytes apart


def at(k):
    return AT * (k + 1)


def refused(name, args, *words):
    lib = native.load()
    rc = getattr(lib, name)(ctypes.byref(args) if args is not None else None, None)
    msg = lib.sufhip_last_error().decode()
    assert rc == -1, (name, rc, msg)
    assert msg.startswith(name) and all(w in msg for w in words), msg


def does_nothing(name, args):
    assert getattr(native.load(), name)(ctypes.byref(args), None) == 0


def put(a, **kw):
    """Sets fields; "x.p0" is entry 0 of the array p of a.x."""
    for k, v in kw.items():
        o, parts = a, k.split("__")
        for q in parts[:-1]:
            o = getattr(o, q)
        last = parts[-1]
        if isinstance(getattr(o, last.rstrip("01"), None), ctypes.Array):
            getattr(o, last[:-1])[int(last[-1])] = v
        else:
            setattr(o, last, v)
    return a


def gate(e, **kw):
    e.key[0], e.key[1], e.table[0], e.table[1] = at(40), at(41), at(42), at(43)
    e.frac_bits, e.work_bytes = 12, 1 << 30
    return put(e, **kw)


# ---- the products ----

def linear_args(**kw):
    a = native.Linear2Args()
    a.w.d_planes, a.w.experts, a.w.K, a.w.N, a.w.digits = at(0), 1, 64, 32, 2
    a.x.p[0], a.x.p[1], a.x.row_stride = at(1), at(2), 64
    a.x_rows = a.rows = 4
    e = native.TruncEpilogue()
    a.trunc = ctypes.pointer(gate(e))
    a.out[0], a.out[1], a.out_stride = at(3), at(4), 32
    a.d_work, a.work_bytes = at(5), 1 << 30
    return put(a, **kw)


LINEAR = [
    (dict(w__experts=0), "experts"), (dict(w__experts=4097), "experts"), (dict(w__K=0), "K"),
    (dict(w__K=65537), "K"), (dict(w__N=0), "N"), (dict(w__N=(1 << 24) + 1), "N"),
    (dict(w__digits=0), "digits"), (dict(w__digits=5), "digits"),
    (dict(w__digits=2, w__K=65536), "digits K"), (dict(rows=-1), "rows"),
    (dict(rows=(1 << 24) + 1), "rows"), (dict(x_rows=-1), "x_rows"),
    (dict(rows=1 << 24, x_rows=1 << 24, w__N=128), "2^31"), (dict(x_rows=0), "no rows"),
    (dict(w__d_planes=None), "planes"), (dict(w__d_planes=at(0) + 8), "planes"),
    (dict(w__experts=2), "d_offsets"), (dict(rows=5), "d_rows"), (dict(x__p0=None), "x is null"),
    (dict(x__row_stride=-1), "stride"), (dict(x__row_stride=(1 << 35) + 1), "stride"),
    (dict(x_digits__d_digits=at(6) + 8, x_digits__rows=4, x_digits__cols=64), "aligned"),
    (dict(x_digits__d_digits=at(6), x_digits__rows=5, x_digits__cols=64), "other rows"),
    (dict(x_digits__d_digits=at(6), x_digits__rows=4, x_digits__cols=63), "other rows"),
    (dict(act=1), "relu"), (dict(act=2), "cubic"), (dict(act=3), "unknown"),
    (dict(residual__p0=at(7), residual__row_stride=32), "residual"),
    (dict(residual__p0=at(7), residual__p1=at(8), residual__row_stride=-32), "stride"),
    (dict(out0=None), "both"), (dict(out0=None, out1=None), "no output"),
    (dict(out_stride=31), "overlap"), (dict(out_stride=-32), "overlap"),
    (dict(out_stride=(1 << 35) + 1), "2^35"),
    (dict(out_digits__d_digits=at(9), out_digits__rows=4, out_digits__cols=33), "other rows"),
    (dict(out_digits__d_digits=at(9) + 1, out_digits__rows=4, out_digits__cols=32), "aligned"),
    (dict(walk_count=-1), "walk_jobs"), (dict(walk_count=1), "walk_jobs"),
    # what the call writes, and what it reads
    (dict(out1=at(3)), "two shares"), (dict(out1=at(3) + 8 * 31), "two shares"),
    (dict(out0=at(1)), "meets x"), (dict(out1=at(1) + 8 * (3 * 64 + 63)), "meets x"),
    (dict(out0=at(0) + 8), "meets an input"),
    (dict(w__d_bias=at(3) + 8), "meets an input"),
    (dict(d_rows=at(4) + 128), "meets an input"),
    (dict(d_offsets=at(4) + 128), "meets an input"),
    (dict(residual__p0=at(3), residual__p1=at(4), residual__row_stride=33), "without being it"),
    (dict(residual__p0=at(4), residual__p1=at(3), residual__row_stride=32), "without being it"),
    (dict(residual__p0=at(3) + 8, residual__p1=at(4), residual__row_stride=32),
     "without being it"),
    (dict(x_digits__d_digits=at(3), x_digits__rows=4, x_digits__cols=64), "meets an input"),
    (dict(out_digits__d_digits=at(3), out_digits__rows=4, out_digits__cols=32), "out_digits"),
    (dict(out_digits__d_digits=at(1), out_digits__rows=4, out_digits__cols=32), "out_digits"),
    (dict(out_digits__d_digits=at(0), out_digits__rows=4, out_digits__cols=32), "out_digits"),
]


@pytest.mark.parametrize("kw,word", LINEAR)
def test_linear2_refuses(kw, word):
    refused("sufhip_linear2", linear_args(**kw), word)


def test_linear2_refuses_gates_and_workspaces():
    refused("sufhip_linear2", None, "null args")
    for kw, word in ((dict(frac_bits=15), "frac_bits"), (dict(work_bytes=8), "work bytes"),
                     (dict(key0=None), "keys"), (dict(add0=at(60), add1=at(61)), "addend")):
        a = linear_args()
        gate(a.trunc.contents, **kw)
        refused("sufhip_linear2", a, word)
    a = linear_args(act=1)
    a.trunc = None
    lib = native.load()
    put(a, relu__key0=at(20), relu__key1=at(21), relu__intervals=3,
        relu__key_bytes=lib.sufhip_interval_lut_key_bytes(3, 2))
    refused("sufhip_linear2", a, "needs trunc")
    for kw in (dict(relu__intervals=0), dict(relu__intervals=65), dict(relu__key_bytes=8),
               dict(relu__key0=at(20) + 4)):
        b = linear_args(act=1, relu__key0=at(20), relu__key1=at(21), relu__intervals=3,
                        relu__key_bytes=lib.sufhip_interval_lut_key_bytes(3, 2))
        refused("sufhip_linear2", put(b, **kw), "relu needs")
    # An epilogue of its own needs the opens.
    d = dict(out_digits__d_digits=at(9), out_digits__rows=4, out_digits__cols=32)
    need = lib.sufhip_linear2_work_bytes(ctypes.byref(linear_args(**d)))
    assert need >= 4 * 32 * 8
    for kw in (dict(work_bytes=need - 1), dict(d_work=None), dict(d_work=at(5) + 8)):
        refused("sufhip_linear2", linear_args(**d, **kw), "workspace")
    for meets in (at(0), at(1), at(3), at(9)):
        refused("sufhip_linear2", linear_args(**d, d_work=meets), "workspace")
    does_nothing("sufhip_linear2", linear_args(rows=0))
    # 2^17 column tiles of 128 (three digits) for each row tile of 127 experts:
    # past a launch's lanes.
    refused("sufhip_linear2", linear_args(rows=127, x_rows=127, w__N=1 << 24, w__experts=127,
                                          w__digits=3, d_offsets=at(22), out_stride=1 << 24),
            "tiles")


def test_sizes():
    lib = native.load()
    assert lib.sufhip_digits2_bytes(3, 33) == 2 * 2 * 3 * 256
    for rows, cols in ((0, 1), (1, 0), (-1, 5), ((1 << 24) + 1, 1), (1, (1 << 24) + 1)):
        assert lib.sufhip_digits2_bytes(rows, cols) == 0
    # K up to a multiple of 64, N too, a byte a digit.
    assert lib.sufhip_linear_planes_bytes(3, 65, 65, 2) == 3 * 128 * 128 * 2
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0), (1, 1, 1, 5),
                (4097, 1, 1, 1), (1, 65537, 1, 1), (1, 65536, 1, 2)):
        assert lib.sufhip_linear_planes_bytes(*bad) == 0
    assert lib.sufhip_linear2_work_bytes(None) == 0
    assert lib.sufhip_linear2_work_bytes(ctypes.byref(linear_args(rows=0))) == 0
    # The workspace is the same whether the walks come with the call or not,
    # where it has an epilogue of its own anyway.
    for rows in (1, 9, 300):
        a = linear_args(rows=rows, x_rows=rows, out_digits__d_digits=at(9))
        b = linear_args(rows=rows, x_rows=rows, out_digits__d_digits=at(9), walk_count=2)
        assert lib.sufhip_linear2_work_bytes(ctypes.byref(a)) == \
            lib.sufhip_linear2_work_bytes(ctypes.byref(b))
    assert lib.sufhip_rmsnorm2_work_bytes(1, 4096) == 0
    assert lib.sufhip_rmsnorm2_work_bytes(1 << 12, 1 << 9) == (1 << 12) * 24
    for rows, cols in ((0, 4), (4, 0), ((1 << 24) + 1, 4), (4, (1 << 20) + 1)):
        assert lib.sufhip_rmsnorm2_work_bytes(rows, cols) == 0


def test_prepare_and_split_refuse():
    lib = native.load()

    def bad(rc, word):
        assert rc == -1 and word in lib.sufhip_last_error().decode()
    for extents in ((0, 1, 1, 1), (1, 1, 1, 5), (1, 65536, 1, 2)):
        bad(lib.sufhip_linear_prepare(at(0), *extents, at(1), None), "needs 1 <=")
    bad(lib.sufhip_linear_prepare(None, 1, 1, 1, 1, at(1), None), "null")
    bad(lib.sufhip_linear_prepare(at(0), 1, 1, 1, 1, at(1) + 8, None), "aligned")
    x, d = native.Matrix2(), native.Digits2()
    x.p[0], x.p[1], x.row_stride = at(0), at(1), 40
    d.d_digits, d.rows, d.cols = at(2), 3, 40

    def split(word, **kw):
        y, e = native.Matrix2.from_buffer_copy(x), native.Digits2.from_buffer_copy(d)
        for k, v in kw.items():
            put(e if k in ("d_digits", "rows", "cols") else y, **{k: v})
        bad(lib.sufhip_digits2_split(ctypes.byref(y), ctypes.byref(e), None), word)
    split("2^24", rows=-1)
    split("2^24", d_digits=None)
    split("aligned", d_digits=at(2) + 8)
    split("null", p0=None)
    split("stride", row_stride=-1)
    split("meets", d_digits=at(1) + 8 * 112)
    bad(lib.sufhip_digits2_split(None, ctypes.byref(d), None), "null")


# ---- the norm ----

def norm_args(**kw):
    a = native.RmsNorm2Args()
    a.x.p[0], a.x.p[1], a.x.row_stride = at(0), at(1), 40
    a.rows, a.cols = 3, 40
    for k, name in enumerate(("a", "a2", "b", "ab")):
        for p in (0, 1):
            getattr(a, name)[p] = at(2 + 2 * k + p)
    for e in list(a.tr_ms) + [a.tr_norm, a.tr_weight]:
        gate(e)
    c = a.rsqrt
    c.kind, c.frac_bits, c.n = native.CHAIN_RSQRT, 12, 3
    c.lut[0], c.lut[1], c.intervals = at(50), at(51), 4
    c.lut_key_bytes = native.load().sufhip_interval_lut_key_bytes(4, 2)
    for t in list(c.a) + list(c.b) + list(c.c):
        t.p[0], t.p[1], t.len, t.stride, t.mul = at(52), at(53), 1 << 30, 1, 1
    for q, e in enumerate(c.trunc[:4]):
        gate(e, frac_bits=13 if q == 2 else 12)
    a.out[0], a.out[1], a.out_stride = at(10), at(11), 40
    return put(a, **kw)


NORM = [
    (dict(rows=-1), "rows"), (dict(rows=(1 << 24) + 1), "rows"), (dict(cols=-1), "cols"),
    (dict(cols=(1 << 20) + 1), "cols"), (dict(x__p1=None), "x is null"),
    (dict(x__row_stride=-40), "stride"), (dict(residual__p1=at(12)), "residual"),
    (dict(a0=None), "a, a2, b and ab"), (dict(ab1=None), "a, a2, b and ab"),
    (dict(tr_norm__frac_bits=15), "frac_bits"), (dict(tr_norm__work_bytes=8), "work bytes"),
    (dict(tr_norm__add0=at(13), tr_norm__add1=at(14)), "addend"),
    (dict(d_weight=at(13), tr_weight__key0=None), "keys"),
    (dict(rsqrt__kind=native.CHAIN_CUBIC), "RSQRT"), (dict(rsqrt__n=4), "n = rows"),
]
NORM_OUT = [
    (dict(out1=None), "both"), (dict(total0=at(13)), "both"),
    (dict(out0=None, out1=None), "no output"), (dict(out_stride=39), "overlap"),
    (dict(out_stride=-40), "overlap"), (dict(out_stride=(1 << 35) + 1), "2^35"),
    (dict(out_digits__d_digits=at(13), out_digits__rows=3, out_digits__cols=41), "other rows"),
    (dict(out_digits__d_digits=at(13) + 8, out_digits__rows=3, out_digits__cols=40), "aligned"),
    (dict(out1=at(10)), "meet"), (dict(out0=at(1)), "without being it"),
    (dict(out0=at(0) + 8), "without being it"),
    (dict(out0=at(0), out_stride=41), "without being it"),
    (dict(out0=at(2) + 8 * 119), "material"), (dict(out1=at(8)), "material"),
    (dict(out0=at(4)), "material"), (dict(out0=at(6)), "material"),
    (dict(d_weight=at(11)), "material"),
    (dict(total0=at(10) + 8 * 119, total1=at(13), total_stride=40), "two outputs"),
    (dict(out_digits__d_digits=at(10), out_digits__rows=3, out_digits__cols=40), "out_digits"),
    (dict(out_digits__d_digits=at(1), out_digits__rows=3, out_digits__cols=40), "out_digits"),
    (dict(out_digits__d_digits=at(9), out_digits__rows=3, out_digits__cols=40), "material"),
    (dict(walk_count=-1), "walk_jobs"), (dict(walk_count=2), "walk_jobs"),
    (dict(rows=1 << 12, cols=1 << 9, x__row_stride=1 << 9, out_stride=1 << 9, rsqrt__n=1 << 12),
     "workspace"),
    (dict(rows=1 << 12, cols=1 << 9, x__row_stride=1 << 9, out_stride=1 << 9, rsqrt__n=1 << 12,
          d_work=at(13), work_bytes=24 * (1 << 12) - 1), "workspace"),
    (dict(rows=1 << 12, cols=1 << 9, x__row_stride=1 << 9, out_stride=1 << 9, rsqrt__n=1 << 12,
          d_work=at(13) + 8, work_bytes=1 << 20), "workspace"),
    (dict(rows=1 << 12, cols=1 << 9, x__row_stride=1 << 9, out_stride=1 << 9, rsqrt__n=1 << 12,
          d_work=at(0), work_bytes=1 << 20), "workspace"),
    (dict(rows=1 << 12, cols=1 << 9, x__row_stride=1 << 9, out_stride=1 << 9, rsqrt__n=1 << 12,
          d_work=at(7), work_bytes=1 << 20), "workspace"),
]


@pytest.mark.parametrize("kw,word", NORM + NORM_OUT)
def test_rmsnorm2_refuses(kw, word):
    refused("sufhip_rmsnorm2", norm_args(**kw), word)


def test_rmsnorm2_of_nothing():
    refused("sufhip_rmsnorm2", None, "null args")
    does_nothing("sufhip_rmsnorm2", norm_args(rows=0))
    does_nothing("sufhip_rmsnorm2", norm_args(cols=0))


# ---- the weighted sum ----

def mix_args(**kw):
    a = native.ExpertMix2Args()
    a.z.p[0], a.z.p[1], a.z.row_stride = at(0), at(1), 40
    a.z_rows, a.tokens, a.each, a.cols = 6, 3, 2, 40
    a.d_slots, a.d_weights = at(2), at(3)
    e = native.TruncEpilogue()
    a.trunc = ctypes.pointer(gate(e))
    a.out[0], a.out[1], a.out_stride = at(4), at(5), 40
    return put(a, **kw)


MIX = [
    (dict(tokens=-1), "tokens"), (dict(tokens=(1 << 24) + 1), "tokens"), (dict(cols=-1), "cols"),
    (dict(each=1025), "each"), (dict(each=-1), "each"), (dict(z_rows=-1), "z_rows"),
    (dict(tokens=1 << 24, cols=128), "2^31"), (dict(d_slots=None), "d_slots"),
    (dict(d_weights=None), "d_weights"), (dict(z__p0=None), "z is null"),
    (dict(z__row_stride=-1), "stride"), (dict(residual__p0=at(6)), "residual"),
    (dict(residual__p0=at(6), residual__p1=at(7), residual__row_stride=-1), "stride"),
    (dict(out0=None), "out is null"), (dict(out_stride=39), "overlap"),
    (dict(out_stride=(1 << 35) + 1), "2^35"), (dict(out1=at(4) + 8), "two shares"),
    (dict(out0=at(1) + 8 * 239), "meets z"), (dict(out0=at(2)), "slots"),
    (dict(out1=at(3) + 40), "weights"),
    (dict(residual__p0=at(5), residual__p1=at(4), residual__row_stride=40), "without being it"),
]


@pytest.mark.parametrize("kw,word", MIX)
def test_expert_mix2_refuses(kw, word):
    refused("sufhip_expert_mix2", mix_args(**kw), word)


def test_expert_mix2_of_nothing():
    refused("sufhip_expert_mix2", None, "null args")
    does_nothing("sufhip_expert_mix2", mix_args(tokens=0))
    does_nothing("sufhip_expert_mix2", mix_args(cols=0))
    a = mix_args()
    gate(a.trunc.contents, frac_bits=15)
    refused("sufhip_expert_mix2", a, "frac_bits")


# ---- Python ----

STATE = bytes(240)


@pytest.mark.parametrize("make", [
    lambda: ff.RMSNorm(0, 8, STATE), lambda: ff.RMSNorm(1.5, 8, STATE),
    lambda: ff.RMSNorm((1 << 24) + 1, 8, STATE), lambda: ff.RMSNorm(1, 0, STATE),
    lambda: ff.RMSNorm(1, (1 << 20) + 1, STATE), lambda: ff.RMSNorm(1, 8, STATE, frac_bits=14),
    lambda: ff.RMSNorm(1, 8, STATE, frac_bits=12.0), lambda: ff.RMSNorm(1, 8, STATE, device="cpu"),
    lambda: ff.Digits(0, 8), lambda: ff.Digits(8, 1 << 25), lambda: ff.Digits(8, 8, "cpu"),
    lambda: ff.ExpertMix(0, 8, STATE), lambda: ff.ExpertMix(8, -1, STATE),
    lambda: ff.ExpertMix(1 << 20, 1 << 12, STATE), lambda: ff.ExpertMix(1, 8, STATE, frac_bits=15),
    lambda: ff.ExpertMix(1, 8, STATE, device="cpu"),
    lambda: ff.PublicWeights(torch.zeros(4, dtype=torch.int64)),
    lambda: ff.PublicWeights(torch.zeros(4, 4)), lambda: ff.PublicWeights(np.zeros((0, 4), int)),
    lambda: ff.PublicWeights(np.zeros((4, 5), int), np.zeros(4, int)),
    lambda: ff.PublicWeights(np.zeros((2, 4, 5), int), np.zeros(5, int)),
    lambda: ff.PublicWeights(np.zeros((4, 5), int), device="cpu"),
    lambda: ff.FeedForward(1, None, None, STATE),
    lambda: ff.ExpertFeedForward(1, 0, None, None, STATE),
    lambda: ff.ExpertFeedForward(0, 1, None, None, STATE),
])
def test_constructors_refuse(make):
    with pytest.raises(ValueError):
        make()


class Weights:
    """The extents of a PublicWeights."""

    def __init__(self, K=8, N=4, experts=1):
        self.K, self.N, self.experts, self.d = K, N, experts, 0


@pytest.mark.parametrize("kw", [dict(act="gelu"), dict(act="relu", trunc=False),
                                dict(frac_bits=15), dict(act=([0], [0]), frac_bits=14),
                                dict(x_rows=0), dict(rows=0), dict(rows=1 << 24)])
def test_linear_refuses(kw):
    rows = kw.pop("rows", 3)
    with pytest.raises(ValueError):
        ff.Linear(Weights(N=128), rows, STATE, **kw)


def test_rows_of_a_pair():
    """The tensors that a matrix may be, on the CPU's device number."""
    t = torch.zeros(4, 10, dtype=torch.int64)

    def take(pair, shape, written=False):
        m = native.Matrix2()
        ff._matrix(m, pair, shape, -1, "x", "x", written)
        return m.row_stride
    assert take((t, t), (4, 10)) == 10
    assert take((t[:, 2:7], t[:, 5:]), (4, 5)) == 10
    assert take((t[::2], t[::2]), (2, 10)) == 20
    assert take((t[:1].expand(3, 10),) * 2, (3, 10)) == 0
    assert take((t[:, :1], t[:, 3:4]), (4, 1)) == 10
    assert take((t.t()[:1].t(), t[:, :1]), (4, 1)) == 10
    for pair, shape, written in (
            (t, (4, 10), False), ((t,), (4, 10), False), ((t, t, t), (4, 10), False),
            ((t, None), (4, 10), False), ((t, t.int()), (4, 10), False),
            ((t, t), (4, 9), False), ((t, t[:, :9]), (4, 10), False),
            ((t[:, ::2], t[:, ::2]), (4, 5), False), ((t.t(), t.t()), (10, 4), False),
            ((t[:, :5], torch.zeros(4, 5, dtype=torch.int64)), (4, 5), False),
            ((t[:1].expand(3, 10),) * 2, (3, 10), True)):
        with pytest.raises(ValueError):
            take(pair, shape, written)


def test_digits_of():
    of = ff.PublicWeights._digits_of
    for n, (lo, hi) in enumerate([(-128, 127), (-32896, 32639), (-8421504, 8355711),
                                  (-2155905152, 2139062143)], 1):
        # The range's own numbers by their digits' definition.
        assert lo == sum(-128 * 256 ** i for i in range(n))
        assert hi == sum(127 * 256 ** i for i in range(n))
        assert of(lo, hi) == n and of(lo - 1, 0) == n + 1 and of(0, hi + 1) == n + 1
    assert of(0, 0) == 1 and of(-1 << 63, (1 << 63) - 1) == 8


def test_own_dealers_differ():
    seeds = [next(ff._seeds) for _ in range(3)]
    assert len(set(seeds)) == 3


@pytest.mark.parametrize("f", [8, 10, 12, 13])
def test_wide_rsqrt_table(f):
    """The chain's definition over the table's whole range.  A first guess off by
    e <= 6.25 % (a chord and its rounded slope; a quarter octave's constant: 4.5 %)
    leaves 1.5 e^2.  The floor of y y to 2^-f leaves a share of up to v 2^-f of
    it out: what a constant cannot make up for is the slope, off by 0.75 v 2^-f
    of an octave's 1/8 on each side (a factor of 1.09): 0.1 v 2^-f.  The floors
    and the constant's own rounding are less than four steps of 2^-f on y."""
    eps = 1.0 / 1024.0
    alpha, words = tables.rsqrt_wide_table(f, eps)
    assert alpha[0] == 0 and np.all(alpha[1:] > alpha[:-1]) and len(alpha) + 2 <= 64
    v = np.unique(np.rint(np.exp(np.linspace(0, np.log(4096), 4001)) * 2.0 ** f)).astype(np.uint64)
    y = ref.rsqrt(v, (alpha, words), f).view(np.int64) / 2.0 ** f
    want = 1 / np.sqrt(v / 2.0 ** f)
    real = v / 2.0 ** f
    assert np.all(np.abs(y - want) <= want * (1.5 * 0.0625 ** 2 + 0.1 * real * 2.0 ** -f)
                  + 4 * 2.0 ** -f)
    if f == 12:  # what the table says of itself
        for most, share in ((256, 0.005), (1024, 0.009), (4096, 0.025)):
            at_most = (real >= 1) & (real < most)
            assert np.abs(y / want - 1)[at_most].max() <= share


@pytest.mark.parametrize("tokens,each,experts", [(1, 1, 1), (5, 2, 4), (40, 3, 8), (7, 1, 300),
                                                 (3, 0, 2), (0, 2, 2)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_route(tokens, each, experts, dtype):
    rng = np.random.default_rng(tokens + experts)
    chosen = rng.integers(-1, experts + 1, (tokens, each))  # some in no expert
    offsets, rows, slots = ff.route(torch.from_numpy(chosen).to(dtype), experts)
    assert offsets.dtype == rows.dtype == slots.dtype == torch.int32
    offsets, rows, slots = offsets.numpy(), rows.numpy(), slots.numpy()
    assert offsets.shape == (experts + 1,) and rows.shape == (tokens * each,)
    there = (chosen >= 0) & (chosen < experts)
    assert offsets[0] == 0 and offsets[-1] == there.sum()
    assert np.array_equal(np.diff(offsets), np.bincount(chosen[there], minlength=experts))
    assert np.array_equal(slots >= 0, there)
    for t, k in zip(*np.nonzero(there)):
        s = slots[t, k]
        assert rows[s] == t and offsets[chosen[t, k]] <= s < offsets[chosen[t, k] + 1]
    assert len(set(slots[there])) == there.sum()
    for e in range(experts):  # a token's rows in its tokens' order
        assert np.all(np.diff(rows[offsets[e]:offsets[e + 1]]) >= 0)


@pytest.mark.parametrize("bad", [torch.zeros(4, dtype=torch.int64), torch.zeros(4, 2)])
def test_route_refuses(bad):
    with pytest.raises(ValueError):
        ff.route(bad, 4)


def test_blocks_refuse_weights_that_do_not_fit():
    for up, down, experts in ((Weights(8, 4), Weights(4, 8), 1), (None, None, None)):
        with pytest.raises(ValueError, match="PublicWeights"):
            ff._pair("FeedForward", up, down, experts)
    make = ff.PublicWeights.__new__

    def weights(K, N, experts=1):
        w = make(ff.PublicWeights)
        w.K, w.N, w.experts, w.d = K, N, experts, 0
        return w
    ff._pair("FeedForward", weights(8, 4), weights(4, 8), 1)
    ff._pair("ExpertFeedForward", weights(8, 4, 3), weights(4, 8, 3), None)
    for up, down in ((weights(8, 4), weights(4, 9)), (weights(8, 4), weights(5, 8)),
                     (weights(8, 4, 2), weights(4, 8, 3))):
        with pytest.raises(ValueError, match="fit"):
            ff._pair("ExpertFeedForward", up, down, None)
    with pytest.raises(ValueError, match="2 matrices"):
        ff._pair("FeedForward", weights(8, 4, 2), weights(4, 8, 2), 1)
