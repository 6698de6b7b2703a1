"""Cached attention at the edges of what a call may hold: wrong words in
device memory, empty batches, far pages."""
import gc

import numpy as np
import pytest
import torch

import kv_reference as ref
from gpu_util import dev, say, u64
from suf_amd import kv_attention as kv
from suf_amd import native

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    native.call("sufhip_init", 0)
    yield
    gc.collect()
    torch.cuda.empty_cache()


def dev2(pair):
    return tuple(dev(v) for v in pair)


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def eq(got, want, what):
    for p in range(2):
        g = u64(got[p])
        assert np.array_equal(g, want[p]), "%s: party %d, %d of %d differ" % (
            what, p, int((g != want[p]).sum()), g.size)


LOW, HIGH = -2 ** 31, 2 ** 31 - 1


@pytest.mark.parametrize("kind", ["scores", "values"])
@pytest.mark.parametrize("new,lens", [([2, 3], [70, 300]), ([2, 60], [70, 300])])
@pytest.mark.parametrize("ends", [(HIGH, LOW), (9999, -5), (HIGH, HIGH), (99, 0)])
def test_wrong_starts_stay_inside(kind, new, lens, ends):
    """Starts past the tokens, then far below them: the second sequence ends
    with the tokens, the third has no rows, whatever their difference is."""
    say("wrong starts %s %s new %s" % (kind, ends, new))
    rng = np.random.default_rng(sum(new))
    c = ref.Case(rng, new + [0], lens + [40], 16, 2, 64)
    H = 4
    off = c.causal(H)
    n = int(off[-1])
    shapes = ((c.tokens, H, 64), (n,)) if kind == "scores" else ((n,), (c.tokens, H, 64))
    x, a = ([ref.words(rng, *shapes[0]) for _ in range(2)] for _ in range(2))
    cc, out = ([ref.words(rng, *shapes[1]) for _ in range(2)] for _ in range(2))
    want = getattr(ref, kind)(c, H, off, x, a, cc, out)
    o = dev2(out)
    batch = kv.Batch(i32([0, new[0], ends[0], ends[1]]), i32(c.lens), i32(c.table),
                     tokens=c.tokens, max_new=max(new), max_keys=max(lens))
    op = kv.scores2 if kind == "scores" else kv.values2
    op(batch, kv.Pool(*(dev(w) for w in c.pool)), dev2(x), dev2(a), dev2(cc), i32(off), o)
    eq(o, want, kind)


def test_calls_on_no_tokens():
    """No sequences, sequences without new tokens, rows of padding alone."""
    cache = kv.PagedCache(4, 4, 1, 8)
    s = cache.open()
    cache.extend([s], [3])
    r = kv.Rotary.build(8, 4)
    z = lambda *n: torch.zeros(n, dtype=torch.int64, device="cuda")  # noqa: E731
    b = cache.extend([s], [0])
    none = kv.Batch(i32([0]), i32([]), i32([]).reshape(0, 1), tokens=2, max_new=1, max_keys=4)
    for batch, T in ((cache.extend([], []), 0), (b, 0), (none, 2)):
        x = tuple(torch.full((T, 1, 8), 5, dtype=torch.int64, device="cuda") for _ in range(2))
        p = (z(0), z(0))
        off = i32([0] * (T + 1))
        kv.append2(batch, cache.k, x, x, cache.v, x, x, rotary=r)
        kv.scores2(batch, cache.k, x, x, p, off, p)
        out = tuple(torch.full((T, 1, 8), 7, dtype=torch.int64, device="cuda") for _ in range(2))
        kv.values2(batch, cache.v, p, p, x, off, out)
        assert all(bool((t == 7).all()) for t in out)
    assert not any(bool(t.any()) for c in (cache.k, cache.v) for t in (c.e,) + c.b)


def test_one_pool_for_keys_and_values_is_refused():
    cache = kv.PagedCache(4, 4, 1, 8)
    b = cache.extend([cache.open()], [1])
    x = tuple(torch.ones((1, 1, 8), dtype=torch.int64, device="cuda") for _ in range(2))
    for pool in (cache.k, kv.Pool(cache.v.e, cache.v.b[0], cache.k.e)):
        with pytest.raises(native.SufHipError, match="share memory"):
            kv.append2(b, cache.k, x, x, pool, x, x)
    assert not any(bool(t.any()) for c in (cache.k, cache.v) for t in (c.e,) + c.b)
