"""Tables and the closed form of the softmax of long rows, on the CPU: how far
the reciprocals, the exponentials and the weights are from real numbers."""
import numpy as np
import pytest

import fixed_point as fp
import long_rows_reference as ref
from suf_amd import kv_attention as kv
from suf_amd import softmax, tables


@pytest.mark.parametrize("f,nmax", [(12, 1024.0), (13, 2048.0), (8, 1024.0), (12, 16.0),
                                    (28, 2.0 ** 18)])
def test_wide_reciprocal_table(f, nmax):
    """recip_table's pieces as far as their slopes are whole words."""
    wide, plain = tables.recip_wide_table(f, nmax), tables.recip_table(f, nmax)
    end = int(min(2.0 ** ((f + 1) // 2), nmax)) << f
    k = int((plain[0] < end).sum())
    assert np.array_equal(wide[0][:k], plain[0][:k]) and np.array_equal(wide[1][:k], plain[1][:k])
    assert (np.diff(wide[0].astype(np.int64)) > 0).all() and int(wide[0][-1]) == int(nmax) << f
    assert len(wide[0]) < 64  # one more at the wrap: a gate's most
    want = [2.0 ** f / (int(a) / 2.0 ** f) for a in wide[0][k:]]
    assert (wide[1][k:, 1] == 0).all()
    # Each constant against 1 / x where its piece starts: a quarter octave on.
    assert (abs(wide[1][k:, 0] - want) <= 0.09 * np.array(want) + 1).all()


def test_reciprocal_of_every_sum():
    """One Newton step in Q(12): within its first guess's error squared (0.09
    and half a step) and two steps of 2^-12 below 1 / x, never above it."""
    f, x = 12, np.arange(1 << 12, 1024 << 12, 7, dtype=np.int64)
    y = fp.recip_task(*tables.recip_wide_table(f, 1024.0), x, f)
    real = 2.0 ** (2 * f) / x
    guess = 0.125 + 0.5 / real
    assert (y <= real + 1).all() and (y >= real * (1 - guess ** 2) - 2).all()
    # The plain table has lost 1 / x there: at 127 and 255 the word is 1 and 0.
    plain = fp.recip_task(*tables.recip_table(f), np.array([127 << f, 255 << f]), f)
    assert (plain * 4 < 2.0 ** f / np.array([127, 255])).all()


def test_long_rows_reciprocal():
    """Three steps in Q(28): three floors, each of a step or of x steps."""
    f = softmax.INV_BITS
    x = np.rint(2.0 ** (f + np.linspace(-0.01, 17, 100001))).astype(np.int64)
    y = fp.recip_task(*tables.recip_wide_table(f, 2.0 ** 18), x, f, 3)
    real = x / 2.0 ** f
    assert (abs(y / 2.0 ** f * real - 1) <= 0.125 ** 8 + 3 * (real + 1) * 2.0 ** -f).all()


def test_fine_exponential():
    """h^4 / 384 of the value, and the words' rounding: half a step of c0, one
    of c1 h, one of c2 h^2 / 2, half of c3 h^3 / 8 and the floor."""
    f = softmax.HALF_BITS
    x = np.rint(np.linspace(0, 20, 300001) * 2 ** f).astype(np.int64)
    g = fp.cubic_task(*tables.nexp_fine_table(f), x, f)
    real = np.exp(-x / 2.0 ** f)
    real[x >= 16 << f] = 0.0
    assert (abs(g - real * 2 ** f) <= real * 2 ** f * 0.5 ** 4 / 384 * np.exp(0.5) + 3.0).all()
    assert g[0] == 1 << f and g.min() >= 0 and g.max() == 1 << f


def weights_l1(x, f=12):
    """Distance of the closed form's shares from softmax(x), and its bound."""
    q = np.rint(np.asarray(x) * 2 ** f).astype(np.int64)
    w, _, y = ref.weights(q, [0, len(q)], f)
    real = np.exp((q - q.max()) / 2.0 ** f)
    return np.abs(w * (y[0] / 2.0 ** 52) - real / real.sum()).sum(), ref.bound(real)


@pytest.mark.parametrize("n", [1, 2, 127, 255, 512, 2048, 4096, 30000, 131072])
@pytest.mark.parametrize("sigma", [0.0, 0.3, 1.0, 4.0])
def test_weights_of_long_rows(n, sigma):
    l1, bound = weights_l1(np.random.default_rng(n).normal(0, 1, n) * sigma)
    assert l1 <= bound and bound < 0.03, (l1, bound)


@pytest.mark.parametrize("t", [9.0, 14.0, 18.0, 33.0])
def test_one_key_among_many_small_ones(t):
    l1, bound = weights_l1([0.0] + [-t] * 65535)
    assert l1 <= bound and bound < 0.03, (l1, bound)


def test_long_rows_refusals():
    for off, f in (([0, (1 << 17) + 1], 12), ([0, 4], 0), ([0, 4], 20)):
        with pytest.raises(ValueError, match="LongRows"):
            softmax.LongRows(off, bytes(128), f, [0])


class Cache:
    """What CachedAttention asks of a cache before any device work."""
    kv_heads, device = 1, "cpu"

    class k:
        dim = 8


def test_softmax_chosen_by_positions(monkeypatch):
    """Six steps of 2^-f an equal share, and gates of at most 13 bits."""
    monkeypatch.setattr(kv.Rotary, "build", classmethod(lambda *a, **k: None))
    make = lambda *a, **k: kv.CachedAttention(Cache, 1, b"", *a, **k)  # noqa: E731
    for positions, f, long in ((64, 12, False), (682, 12, False), (683, 12, True),
                               (4096, 12, True), (600, 14, True), (10, 6, False), (11, 6, True)):
        assert make(positions, frac_bits=f).long_rows is long
    assert make(64, long_rows=True).long_rows and not make(64, long_rows=False).long_rows
    with pytest.raises(ValueError, match="long_rows"):
        make(4096, long_rows=False)
    with pytest.raises(ValueError, match="positions"):
        make((1 << 17) + 1)


@pytest.mark.parametrize("make", [
    lambda: softmax.SoftmaxBlock([0, 3, 5], bytes(128), device="cpu"),
    lambda: softmax.LongRows([0, 3, 5], bytes(128), 12, [0, 1, 1], device="cpu")])
def test_a_blocks_material_is_on_its_device(monkeypatch, make):
    """Every tensor of a block, also those of its exponentials' gate."""
    monkeypatch.setattr(softmax.torch.cuda, "Stream", lambda device=None: None)
    monkeypatch.setattr(softmax.spline.pfss, "trunc_gen",
                        lambda *a: [softmax.torch.empty(8, device=a[-1])] * 2)
    seen = []

    def walk(v):
        if isinstance(v, softmax.torch.Tensor):
            seen.append(v.device.type)
        elif isinstance(v, (list, tuple)):
            for w in v:
                walk(w)
        elif isinstance(v, dict):
            walk(list(v.values()))
        elif type(v).__module__.startswith("suf_amd") and hasattr(v, "__dict__"):
            walk(list(vars(v).values()))
    walk(make())
    assert len(seen) > 50 and set(seen) == {"cpu"}


def test_each_attention_has_a_dealer_of_its_own(monkeypatch):
    """Layers that open under the same masks tell their difference."""
    monkeypatch.setattr(kv.Rotary, "build", classmethod(lambda *a, **k: None))
    a, b, c, d = (kv.CachedAttention(Cache, 1, b"", 64, **kw).dealer
                  for kw in ({}, {}, {"seed": 5}, {"seed": 5}))
    wa, wb, wc, wd = (x.words(64) for x in (a, b, c, d))
    assert not (wa == wb).any() and (wc == wd).all()
