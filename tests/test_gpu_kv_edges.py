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


def test_rotary_takes_rows_between_rows():
    """Outputs in the gaps of their inputs' buffers, in place, in the other
    party's place: taken exactly where no word is another row's."""
    from test_kv_arguments import meets
    rng = np.random.default_rng(11)
    r = kv.Rotary(i32(rng.integers(-99, 99, (50, 2, 2))), 5, pass_mul=3)
    table = r.table.cpu().numpy()
    taken = refusals = 0
    for _ in range(400):
        T, H, D = int(rng.integers(1, 4)), int(rng.integers(1, 4)), 5
        hs = int(rng.choice([5, 6, 10, 15, 20, 40]))
        ts = int(rng.choice([5, 10, 15, 30, 31, 60, 80]))
        like = rng.random() < 0.8
        os = (ts, hs) if like else (int(rng.choice([5, 20, 60])), int(rng.choice([5, 20, 60])))
        x = [(int(v), ts, hs) for v in rng.choice([0, 300], 2, replace=False)]
        out = [(b + int(rng.choice([0, 0, 5, 10, 20, 30, 7, 600])), *os) for b, _, _ in x]
        if rng.random() < 0.3:
            out = out[::-1]
        words = ref.words(rng, 1600)
        buf = dev(words)
        view = lambda rows: torch.as_strided(buf, (T, H, D), (*rows[1:], 1), rows[0])  # noqa: E731
        pos = rng.integers(0, 50, T)
        xs = [u64(view(w).contiguous()) for w in x]
        if len({w for a in x for w in [a[0] + t * ts + h * hs + i for t in range(T)
                                       for h in range(H) for i in range(D)]}) < 2 * T * H * D:
            continue  # the inputs themselves overlap: in place has no meaning
        want = [ref.rotary(v, table, pos, False, 3, v) for v in xs]
        bad = meets(T, H, D, x, out)
        try:
            kv.rotary2([view(w) for w in x], r, i32(pos), [view(w) for w in out])
        except native.SufHipError as e:
            assert "overlap" in str(e)
            assert bad or not like, (T, H, x, out)
            refusals += 1
            continue
        assert not bad, (T, H, x, out)
        after = words.copy()
        for p in range(2):
            for t in range(T):
                for h in range(H):
                    o = out[p][0] + t * os[0] + h * os[1]
                    after[o:o + D] = want[p][t, h]
        assert np.array_equal(u64(buf), after), (T, H, x, out)
        taken += 1
    assert taken > 50 and refusals > 50


@pytest.mark.parametrize("rot", [0, 4])
@pytest.mark.parametrize("given", [False, True])
def test_append_through_a_table_without_positions(rot, given):
    """Every place is outside the table: nothing is written."""
    cache = kv.PagedCache(4, 4, 2, 8)
    b = cache.extend([cache.open()], [3])
    x, m = (tuple(dev(ref.words(np.random.default_rng(i), 3, 2, 8)) for _ in range(2))
            for i in (1, 2))
    r = kv.Rotary(torch.zeros(0, rot // 2, 2, dtype=torch.int32, device="cuda"), 8)
    kv.append2(b, cache.k, x, m, cache.v, x, m, rotary=r,
               positions=i32([0, 1, 2]) if given else None)
    assert not any(bool(t.any()) for t in (cache.k.e,) + cache.k.b)
    rows = cache.v.b[0][cache.seqs[0]["pages"][0]].transpose(0, 1)[:3]
    assert torch.equal(rows, m[0])  # the values are not rotated
    kv.rotary2(x, r, i32([0, 1, 2]), x)
    assert np.array_equal(u64(x[0]), ref.words(np.random.default_rng(1), 3, 2, 8))


def test_append_through_a_table_that_rotates_nothing():
    """rot 0 with positions: the words times the table's 1, inside it alone."""
    cache = kv.PagedCache(4, 4, 1, 8)
    b = cache.extend([cache.open()], [3])
    x, m = ([ref.words(np.random.default_rng(i), 3, 1, 8) for _ in range(2)] for i in (1, 2))
    r = kv.Rotary(torch.zeros(2, 0, 2, dtype=torch.int32, device="cuda"), 8, pass_mul=5)
    kv.append2(b, cache.k, dev2(x), dev2(m), rotary=r)
    e = u64(cache.k.e[cache.seqs[0]["pages"][0]])[0]
    want = np.uint64(5) * (x[0] + x[1])[:, 0] - m[0][:, 0] - m[1][:, 0]
    assert np.array_equal(e[:2], want[:2]) and not e[2:].any()


def test_append_writes_each_array_of_a_far_page():
    """Pages whose words lie past 2^31 words, three arrays of their own."""
    pages, heads, page, dim = 9000, 8, 128, 256  # 18.9 GB an array
    if torch.cuda.mem_get_info()[0] < 70 << 30:
        pytest.skip("70 GiB of device memory wanted")
    rng = np.random.default_rng(1)
    arrays = [torch.empty((pages, heads, page, dim), dtype=torch.int64, device="cuda")
              for _ in range(3)]
    for t in arrays:
        t[-1].zero_()
        t[0].zero_()
    k, m = ([ref.words(rng, 2, heads, dim) for _ in range(2)] for _ in range(2))
    batch = kv.Batch(i32([0, 1, 2]), i32([page, 1]), i32([[pages - 1], [0]]), tokens=2, max_new=1,
                     max_keys=page)
    kv.append2(batch, kv.Pool(*arrays), dev2(k), dev2(m))
    for t, w in zip(arrays, (k[0] + k[1] - m[0] - m[1], m[0], m[1])):
        assert np.array_equal(u64(t[-1][:, -1]), w[0]) and np.array_equal(u64(t[0][:, 0]), w[1])
        assert not bool(t[-1][:, :-1].any()) and not bool(t[0][:, 1:].any())
    del arrays, t, batch
    torch.cuda.empty_cache()
