"""What stands between one use of a feed-forward operator and the next, and what
its public values and its rows may be."""
import ctypes
import warnings

import numpy as np
import pytest
import torch

import feedforward_reference as ref
import oracle_lib as ol
from gpu_util import dev, say, u64
from suf_amd import feedforward as ff
from suf_amd import native, tables, tasks

pytestmark = pytest.mark.gpu

STATE = ol.mt64_bytes(6, ol.PRG_STATE_BYTES).tobytes()


@pytest.fixture(scope="module", autouse=True)
def _init():
    native.call("sufhip_init", 0)


def _pair(*shape):
    return tuple(torch.zeros(shape, dtype=torch.int64, device="cuda") for _ in range(2))


def _public(*shape):
    return ff.PublicWeights(np.arange(np.prod(shape)).reshape(shape) % 200 - 100)


def _tables(tokens, each, experts):
    chosen = torch.arange(tokens * each, device="cuda").reshape(tokens, each) % experts
    return (*ff.route(chosen, experts), torch.ones(tokens, each, dtype=torch.int64, device="cuda"))


def _norm():
    o = ff.RMSNorm(3, 40, STATE, seed=1)
    return (lambda: o.eval2(_pair(3, 40), _pair(3, 40))), (lambda: o.eval2(_pair(3, 41), None))


def _linear():
    o = ff.Linear(_public(40, 24), 3, STATE, act="relu", seed=1)
    return (lambda: o.eval2(_pair(3, 40), _pair(3, 24))), (lambda: o.eval2(_pair(3, 40), None))


def _mix():
    o, slots = ff.ExpertMix(3, 24, STATE, seed=1), torch.zeros(3, 2, dtype=torch.int32).cuda()
    w = torch.ones(3, 2, dtype=torch.int64, device="cuda")
    return (lambda: o.eval2(_pair(4, 24), slots, w, _pair(3, 24))), \
        (lambda: o.eval2(_pair(4, 24), slots, w, _pair(3, 25)))


def _block():
    o = ff.FeedForward(3, _public(40, 24), _public(24, 40), STATE, seed=1)
    return (lambda: o.eval2(_pair(3, 40), _pair(3, 40))), \
        (lambda: o.eval2(_pair(3, 41), _pair(3, 40))), (lambda: o.eval2(_pair(3, 40), None)), \
        (lambda: o.eval2(_pair(3, 40), _pair(3, 40), _pair(3, 39)))


def _experts():
    o = ff.ExpertFeedForward(3, 2, _public(4, 40, 24), _public(4, 24, 40), STATE, seed=1)
    tabs = _tables(3, 2, 4)
    return (lambda: o.eval2(_pair(3, 40), _pair(3, 40), *tabs)), \
        (lambda: o.eval2(_pair(3, 41), _pair(3, 40), *tabs)), \
        (lambda: o.eval2(_pair(3, 40), _pair(3, 41), *tabs)), \
        (lambda: o.eval2(_pair(3, 40), _pair(3, 40), tabs[0][1:], *tabs[1:])), \
        (lambda: o.eval2(_pair(3, 40), _pair(3, 40), tabs[0], tabs[1][1:], *tabs[2:])), \
        (lambda: o.eval2(_pair(3, 40), _pair(3, 40), *tabs[:2], tabs[2][:, :1], tabs[3])), \
        (lambda: o.eval2(_pair(3, 40), _pair(3, 40), *tabs[:3], tabs[3].int()))


@pytest.mark.parametrize("make", [_norm, _linear, _mix, _block, _experts])
def test_a_second_use_is_warned_of(make):
    """Once, where the call stands; a refused call is no use."""
    say("second use, %s" % make.__name__)
    call, *refused = make()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for bad in refused:
            with pytest.raises(ValueError):
                bad()
        call()
        for bad in refused:
            with pytest.raises(ValueError):
                bad()
    with pytest.warns(RuntimeWarning, match="one use") as seen:
        call()
    assert len(seen) == 1 and seen[0].filename == __file__
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        call()  # said once
    torch.cuda.synchronize()


def test_a_product_that_opens_nothing_may_be_used_again():
    say("untruncated product, twice")
    o = ff.Linear(_public(40, 24), 3, STATE, trunc=False)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for _ in range(2):
            o.eval2(_pair(3, 40), _pair(3, 24), digits=ff.Digits(3, 24))
    torch.cuda.synchronize()


def test_one_expert_needs_no_tables():
    """With one expert, one for each token, the tokens' own order will do; the
    sum may take fewer rows than there are."""
    say("one expert, no tables")
    up, down = _public(40, 24), _public(24, 40)
    x = tuple(torch.full((3, 40), v, dtype=torch.int64, device="cuda") for v in (5000, -77))
    slots = torch.arange(3, dtype=torch.int32, device="cuda")[:, None].contiguous()
    w = torch.full((3, 1), 4096, dtype=torch.int64, device="cuda")
    got = [ff.ExpertFeedForward(3, 1, up, down, STATE).eval2(x, _pair(3, 40), *t, slots, w)
           for t in ((None, None), ff.route(torch.zeros(3, 1, dtype=torch.int64).cuda(), 1)[:2])]
    assert torch.equal(*(a[0] + a[1] for a in got))
    two = ff.route(torch.zeros(3, 2, dtype=torch.int64).cuda(), 1)
    out = ff.ExpertFeedForward(3, 2, up, down, STATE).eval2(x, _pair(3, 40), *two[:2],
                                                            2 * slots, w)
    assert torch.equal(out[0] + out[1], got[0][0] + got[0][1])


@pytest.mark.parametrize("most,digits", [(127, 1), (128, 2), (32639, 2), (32640, 3), (32767, 3),
                                         (2139062143, 4), (2139062144, 5), (2 ** 31 - 1, 5)])
def test_digits_of_the_largest_weight(most, digits):
    """As many as the documentation says; a refusal names them and the range."""
    say("digits of %d" % most)
    W = np.array([[3, -5], [most, 0]])
    if digits <= 4:
        assert ff.PublicWeights(W).digits == digits
    else:
        with pytest.raises(ValueError, match=r"-2155905152, 2139062143\].* 5 digits"):
            ff.PublicWeights(W)


@pytest.mark.parametrize("name", ["sufhip_linear2", "sufhip_rmsnorm2"])
def test_walks_of_a_call_without_rows(name):
    """The key-only halves that come with a call are done though it has no rows."""
    say("walks without rows, %s" % name)
    gate = tasks.Trunc(tasks.Dealer(33), 12, 100, STATE)
    gate.prepare()
    torch.cuda.synchronize()
    tables = [t[:1 << 12].clone() for t in gate.work]
    for t in gate.work:
        t.fill_(-7)
    if name == "sufhip_linear2":
        a = native.Linear2Args.from_buffer_copy(ff.Linear(_public(40, 24), 3, STATE)._args)
    else:
        a = native.RmsNorm2Args.from_buffer_copy(ff.RMSNorm(3, 40, STATE)._args)
    a.rows = 0
    state, jobs, a.walk_count = tasks.trunc_jobs([gate])
    a.walk_jobs, a.walk_prg_state = ctypes.addressof(jobs), ctypes.addressof(state)
    native.call(name, ctypes.byref(a), torch.cuda.current_stream().cuda_stream)
    assert all(torch.equal(t[:1 << 12], w) for t, w in zip(gate.work, tables))


MADE = [
    lambda: ff.RMSNorm(3, 40, STATE), lambda: ff.RMSNorm(3, 40, STATE, weight=[4096] * 40),
    lambda: ff.Linear(_public(40, 24), 3, STATE), lambda: ff.ExpertMix(3, 24, STATE),
    lambda: ff.Linear(_public(40, 24), 3, STATE, act="relu"),
    lambda: ff.Linear(_public(40, 24), 3, STATE, act=tables.gelu_table(12)),
    lambda: ff.Linear(_public(40, 24), 3, STATE, trunc=False),
    lambda: ff.PublicWeights(torch.ones(40, 24, dtype=torch.int64, device="cuda")),
    lambda: ff.FeedForward(3, _public(40, 24), _public(24, 40), STATE),
    lambda: ff.ExpertFeedForward(3, 2, _public(4, 40, 24), _public(4, 24, 40), STATE),
]


@pytest.mark.parametrize("which", range(len(MADE)))
def test_objects_are_whole_when_they_are_made(which, monkeypatch):
    """Whatever their stream was doing, and however long the gates' keys take:
    another stream may use them at once."""
    say("made on a busy stream, %d" % which)
    gen = tasks.pfss.trunc_gen
    monkeypatch.setattr(tasks.pfss, "trunc_gen",
                        lambda *a: (torch.cuda._sleep(2000000), gen(*a))[1])
    busy = torch.cuda.Stream()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(2000000)
        made = MADE[which]()
        assert busy.query()
    assert made is not None


@pytest.mark.parametrize("act", [None, "relu"])
def test_another_stream_uses_them_at_once(act, monkeypatch):
    say("used on another stream, act=%s" % act)
    gen = tasks.pfss.trunc_gen
    monkeypatch.setattr(tasks.pfss, "trunc_gen",
                        lambda *a: (torch.cuda._sleep(2000000), gen(*a))[1])
    x = tuple(torch.full((3, 40), v, dtype=torch.int64, device="cuda") for v in (50000, -77))
    outs = [_pair(3, 24) for _ in range(2)]
    public = _public(40, 24)
    torch.cuda.synchronize()
    for out in outs:
        busy, other = torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(busy):
            o = ff.Linear(public, 3, STATE, act=act)
            with torch.cuda.stream(other):
                o.eval2(x, out)
        torch.cuda.synchronize()
    z = (50000 - 77) * (np.arange(40 * 24).reshape(40, 24) % 200 - 100).sum(0) >> 12
    want = torch.from_numpy(np.maximum(z, 0) if act else z).cuda().expand(3, 24)
    assert all(torch.equal(a + b, want) for a, b in outs)


def test_public_values_are_the_objects_own():
    """A buffer that weights were given in may be filled anew."""
    say("public values, given in tensors of the GPU")
    W = torch.arange(40 * 24, device="cuda").reshape(40, 24) % 200 - 100
    bias = torch.arange(24, device="cuda") << 14
    weight = torch.arange(40, device="cuda") * 300
    x = tuple(torch.full((3, 40), v, dtype=torch.int64, device="cuda") for v in (50000, -77))

    def run(spoil):
        lin = ff.Linear(ff.PublicWeights(W.clone(), given[0]), 3, STATE)
        norm = ff.RMSNorm(3, 40, STATE, weight=given[1])
        if spoil:
            for t in given:
                t.fill_(-1)
        return [a + b for a, b in (lin.eval2(x, _pair(3, 24)), norm.eval2(x, _pair(3, 40)))]
    given = bias.clone(), weight.clone()
    want = run(False)
    assert all(torch.equal(a, b) for a, b in zip(run(True), want))
    given = bias.cpu(), weight.cpu()
    assert all(torch.equal(a, b) for a, b in zip(run(True), want))


@pytest.mark.parametrize("rows,cols", [(9, 96), (2100, 1000)])
@pytest.mark.parametrize("eps", [1.0 / 1024.0, 2.0 ** -25])
def test_norm_of_rows_of_any_size(rows, cols, eps):
    """Rows whose mean squares go from 0 to 2^22, through tables of up to 64
    intervals: the definition, and outputs of their inputs' signs that saturate
    where the table ends."""
    say("norm %d x %d of rows of any size, eps %g" % (rows, cols, eps))
    rng = np.random.default_rng(rows)
    size = np.exp2(np.linspace(-14, 11, rows))[:, None]
    x = np.rint(rng.standard_normal((rows, cols)) * size * 4096).astype(np.int64)
    x[0] = 0
    s = rng.integers(0, 1 << 64, x.shape, dtype=np.uint64)
    norm = ff.RMSNorm(rows, cols, STATE, eps=eps)
    assert len(norm.table[0]) == (58 if eps > 1e-4 else 63)
    out = norm.eval2((dev(s), dev(x.view(np.uint64) - s)), _pair(rows, cols))
    got = u64(out[0] + out[1])
    assert np.array_equal(got, ref.rmsnorm(x.view(np.uint64), None, norm.inv_len, norm.eps_q,
                                           norm.table, 12)[1])
    # A floor takes a small value of either sign to -1 step at least.
    got = got.view(np.int64)
    assert np.all(np.where(x < 0, got <= 0, got >= 0))
    last = size[:, 0] ** 2 > 2 * 65536  # past the table's end by more than a row's own spread
    steps = int(norm.table[1][-1][0]) * 3 // 2
    assert last.any() and np.array_equal(got[last], (x[last] * steps) >> 12)
