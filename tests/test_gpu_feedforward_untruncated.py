"""Products without truncation on the GPU, to shares and to digits.  Nothing is
opened in them, so each party's output is its own: x_p W (+ bias, party 0) +
residual_p, word for word."""
import ctypes

import numpy as np
import pytest
import torch

import feedforward_reference as ref
import oracle_lib as ol
from gpu_util import dev, say, u64
from suf_amd import feedforward as ff
from suf_amd import native, tasks

pytestmark = pytest.mark.gpu

STATE = ol.mt64_bytes(5, ol.PRG_STATE_BYTES).tobytes()

SHAPES = [
    # rows, K, N, weight digits, experts
    (1, 1, 1, 1, 1),
    (4, 100, 64, 2, 1),
    (17, 128, 33, 2, 1),
    (9, 130, 70, 3, 1),
    (400, 64, 2100, 2, 1),      # 256 columns a workgroup
    (3, 1000, 96, 2, 1),        # k-slices
    (16, 4096, 200, 4, 1),
    (40, 96, 50, 2, 5),
    (12, 700, 64, 1, 3),        # k-slices
    (2500, 64, 1000, 2, 4),
]


@pytest.fixture(scope="module", autouse=True)
def _init():
    native.call("sufhip_init", 0)


def _words(rng, *shape):
    return rng.integers(0, 1 << 64, shape, dtype=np.uint64)


def _pair(rng, *shape):
    return dev(_words(rng, *shape)), dev(_words(rng, *shape))


def _empty(*shape):
    return tuple(torch.full(shape, -7, dtype=torch.int64, device="cuda") for _ in range(2))


def _case(rng, rows, K, N, digits, experts, bias=True):
    """(the product, its offsets, want(xs, residual) of each party's rows)."""
    lo, hi = -(128 * (256 ** digits - 1) // 255), 127 * (256 ** digits - 1) // 255
    lead = (experts,) if experts > 1 else ()
    W = rng.integers(lo, hi + 1, lead + (K, N))
    W.flat[0], W.flat[-1] = lo, hi
    b = _words(rng, *lead, N).view(np.int64) if bias else None
    weights = ff.PublicWeights(W, b)
    assert weights.digits == digits
    lin = ff.Linear(weights, rows, STATE, trunc=False, seed=31)
    off = np.sort(rng.integers(0, rows + 1, experts + 1)) if experts > 1 else None
    at = None if off is None else torch.from_numpy(off.astype(np.int32)).cuda()

    def want(xs, residual=None):
        got = []
        for p in range(2):
            y, written = ref.linear(u64(xs[p]), W, b if p == 0 else None, 12,
                                    residual=None if residual is None else u64(residual[p]),
                                    offsets=off, trunc=False)
            got.append(y)
        return got, written
    return lin, at, want


@pytest.mark.parametrize("rows,K,N,digits,experts", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_to_shares_and_digits(rows, K, N, digits, experts, residual):
    say("untruncated %dx%dx%d digits=%d experts=%d residual=%s" % (rows, K, N, digits, experts,
                                                                  residual))
    rng = np.random.default_rng(rows + 10 * K + N)
    lin, off, want = _case(rng, rows, K, N, digits, experts)
    xs = _pair(rng, rows, K)
    res = _pair(rng, rows, N) if residual else None
    y, written = want(xs, res)
    there = torch.from_numpy(written).cuda()

    def check(out=None, digits=None):
        for got in ([] if out is None else [out]) + ([] if digits is None else [digits.values()]):
            for p in range(2):
                assert np.array_equal(u64(got[p])[written], y[p][written])
        if out is not None and out is not res:
            assert all(bool((o[~there] == -7).all()) for o in out)
        if digits is not None:
            assert not any(bool(v[~there].any()) for v in digits.values())

    src = ff.Digits(rows, K).split(xs)
    for x in (xs, src):
        out, both, alone = _empty(rows, N), ff.Digits(rows, N), ff.Digits(rows, N)
        lin.eval2(x, out, residual=res, offsets=off)
        check(out)
        out = _empty(rows, N)
        lin.eval2(x, out, residual=res, offsets=off, digits=both)
        check(out, both)
        assert lin.eval2(x, None, residual=res, offsets=off, digits=alone) is None
        check(digits=alone)
    if residual:  # in place
        again = ff.Digits(rows, N)
        lin.eval2(xs, res, residual=res, offsets=off, digits=again)
        check(res, again)


@pytest.mark.parametrize("rows,K,N", [(1, 64, 64), (5, 200, 300), (4, 1000, 70), (500, 64, 96)])
@pytest.mark.parametrize("to_digits", [False, True])
def test_with_walks(rows, K, N, to_digits):
    """Key-only halves of another operator's gates done by the call: its outputs
    stay right, the gates' tables are as in launches of their own, and the
    workspace is no larger than what was asked for."""
    say("untruncated with walks %dx%dx%d digits=%s" % (rows, K, N, to_digits))
    rng = np.random.default_rng(rows + K)
    lin, _, want = _case(rng, rows, K, N, 2, 1)
    xs, out, digits = _pair(rng, rows, K), _empty(rows, N), ff.Digits(rows, N)
    gate = tasks.Trunc(tasks.Dealer(32), 12, 100, STATE)
    gate.prepare()
    torch.cuda.synchronize()
    tables = [t.clone() for t in gate.work]
    for t in gate.work:
        t.fill_(-7)
    state, jobs, count = tasks.trunc_jobs([gate])
    a = native.Linear2Args.from_buffer_copy(lin._args)
    a.x_rows = rows
    ff._matrix(a.x, xs, (rows, K), 0, "x", "x")
    if to_digits:
        a.out_digits = digits.arg
    else:
        ff._out(a, out, (rows, N), 0, "out", "out")
    a.walk_jobs, a.walk_count = ctypes.addressof(jobs), count
    a.walk_prg_state = ctypes.addressof(state)
    words = native.load().sufhip_linear2_work_bytes(ctypes.byref(a)) // 8
    work = torch.full((words + 64,), -7, dtype=torch.int64, device="cuda")
    a.d_work, a.work_bytes = work.data_ptr(), words * 8
    native.call("sufhip_linear2", ctypes.byref(a), torch.cuda.current_stream().cuda_stream)
    y, _ = want(xs)
    got = digits.values() if to_digits else out
    assert all(np.array_equal(u64(got[p]), y[p]) for p in range(2))
    assert bool((work[words:] == -7).all())
    # The first 2^12 entries are the table; what lies behind is scratch.
    assert all(torch.equal(t[:1 << 12], w[:1 << 12]) for t, w in zip(gate.work, tables))
