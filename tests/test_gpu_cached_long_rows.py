"""Cached attention over long rows: whole steps against softmax(q k^T /
sqrt(dim)) v in real numbers, and against the closed form of their stages."""
import gc
import math

import numpy as np
import pytest
import torch

import long_rows_reference as ref
import oracle_lib as ol
from gpu_util import dev, say, u64
from suf_amd import kv_attention as kv
from suf_amd import native, tasks
from suf_amd.softmax import WEIGHT_BITS, LongRows

pytestmark = pytest.mark.gpu

STATE = ol.mt64_bytes(3, ol.PRG_STATE_BYTES).tobytes()
F, ONE = 12, 4096.0


@pytest.fixture(scope="module", autouse=True)
def _init():
    native.call("sufhip_init", 0)
    yield
    gc.collect()
    torch.cuda.empty_cache()


def shares(rng, v):
    s = rng.integers(0, 1 << 64, v.shape, dtype=np.uint64)
    return dev(s), dev(v.view(np.uint64) - s)


def whole(pair):
    return (u64(pair[0]) + u64(pair[1])).view(np.int64)


def rotated(x, rotary, positions):
    """Exact words of trunc(rot(x)), x [tokens, heads, dim], halves paired."""
    cs = rotary.table.cpu().numpy().astype(np.int64)[positions][:, None]
    half = cs.shape[2]
    u, v = x[..., :half], x[..., half:2 * half]
    return np.concatenate([u * cs[..., 0] - v * cs[..., 1], u * cs[..., 1] + v * cs[..., 0],
                           x[..., 2 * half:] * rotary.pass_mul], -1) >> 12


def turned(x, positions):
    """The same in real numbers, and how far the words can be from it: half a
    step of 2^-12 for each of a pair's factors, one for the shift."""
    half = x.shape[-1] // 2
    ang = positions[:, None, None] * 10000.0 ** (-2.0 * np.arange(half) / (2 * half))
    c, s = np.cos(ang), np.sin(ang)
    u, v = x[..., :half], x[..., half:]
    off = (abs(u) + abs(v)) / (2 * ONE) + 1 / ONE
    return np.concatenate([u * c - v * s, u * s + v * c], -1), np.concatenate([off, off], -1)


def fill(att, rng, s, k, v):
    """k, v as the first keys of sequence s, appended without a step."""
    cache, n = att.cache, len(k)
    batch = cache.extend([s], [n])
    masks = [tuple(dev(rng.integers(0, 1 << 64, x.shape, dtype=np.uint64)) for _ in range(2))
             for x in (k, v)]
    kv.append2(batch, cache.k, shares(rng, rotated(k, att.k_rotary, np.arange(n))), masks[0],
               cache.v, shares(rng, v), masks[1])


def fixed_bound(real, short):
    """Most that a row's fixed-point shares can be from real / sum(real)."""
    if not short:
        return ref.bound(real)
    # Q(12): exponentials within e / 384 of themselves and 4 steps; the
    # reciprocal as in test_reciprocal_of_every_sum; a floor each.
    n, s = len(real), real.sum()
    e = (real * np.e / 384 + 4 / ONE).sum()
    guess = 0.125 + 0.5 * (s + e) / ONE
    return 2 * e / max(s - e, 0.5) + guess ** 2 + 2 * (s + e) / ONE + n / ONE


@pytest.mark.parametrize("positions,keys", [(300, 127), (300, 255), (300, 300), (600, 600),
                                            (1024, 1023), (2048, 2048), (4096, 3000),
                                            (4096, 4096), (16384, 16384)])
@pytest.mark.parametrize("sigma", [0.0, 0.3, 1.0, 4.0])
def test_step_against_real_attention(positions, keys, sigma):
    """One token over `keys` keys; sigma 0: equal scores."""
    say("long rows: %d keys, sigma %g" % (keys, sigma))
    rng = np.random.default_rng(keys)
    heads, dim = 2, 16
    cache = kv.PagedCache(-(-keys // 64), 64, 1, dim)
    att = kv.CachedAttention(cache, heads, STATE, positions)
    s = cache.open()
    word = lambda *n, by=1.0, at=0.0: np.rint(  # noqa: E731
        (rng.normal(0, 1, n) * by + at) * ONE).astype(np.int64)
    k, v = word(keys, 1, dim), word(keys, 1, dim, at=2.0)
    q = word(1, heads, dim, by=sigma)
    fill(att, rng, s, k[:-1], v[:-1])
    step = att.deal([s], [1])
    out = tuple(torch.empty((1, heads, dim), dtype=torch.int64, device="cuda") for _ in range(2))
    step.run(shares(rng, q), shares(rng, k[-1:]), shares(rng, v[-1:]), out)
    got = whole(out)[0] / ONE
    kr, k_off = (a[:, 0] for a in turned(k / ONE, np.arange(keys)))
    qr, q_off = (a[0] for a in turned(q / ONE, np.array([keys - 1])))
    # The query's factors are of the scaled table: the same half steps.
    qr = qr / math.sqrt(dim)
    vr = v[:, 0] / ONE
    for h in range(heads):
        x = kr @ qr[h]
        off = (abs(kr) + k_off) @ q_off[h] + k_off @ abs(qr[h]) + 1 / ONE
        real = np.exp(x - x.max())
        p = real / real.sum()
        # Scores off by up to `off` move a share by its own part of
        # exp(2 off), and the values' mean by no more than their range times that.
        move = np.exp(2 * off.max()) * (p * off).sum() * np.ptp(vr, axis=0)
        tol = move + abs(vr).max() * fixed_bound(real, positions <= 682) + 3 / ONE
        err = abs(got[h] - p @ vr)
        assert (err <= tol).all(), "head %d: off by %s, at most %s" % (h, err.max(), tol.min())


@pytest.mark.parametrize("f,lens", [(12, [1, 2, 600, 33, 5]), (14, [1000, 1, 70]), (8, [16])])
def test_long_rows_equal_their_closed_form(f, lens):
    rng = np.random.default_rng(f)
    off = np.concatenate([[0], np.cumsum(lens)])
    n, cols = int(off[-1]), 3
    x = np.rint(rng.normal(0, 2.0, n) * 2 ** f).astype(np.int64)
    x[0] = -1 << 40  # far below the rest
    row_of = np.repeat(np.arange(len(lens))[::-1], cols)
    block = LongRows(off, STATE, f, row_of)
    w = tasks.pair(n)
    out = tasks.pair(len(row_of))
    z = rng.integers(-1 << (f + 3), 1 << (f + 3), len(row_of)) << WEIGHT_BITS
    low = rng.integers(0, 1 << (WEIGHT_BITS - LongRows.z_bits()), len(row_of))
    z = (z >> LongRows.z_bits()) + low
    want_w, _, want_y = ref.weights(x, off, f)
    want = ref.quotient(z << LongRows.z_bits(), want_y[row_of])
    for _ in range(2):
        block.eval2(shares(rng, x), w)
        assert np.array_equal(whole(w), want_w)
        assert np.array_equal(whole(block.recip.y), want_y)
        block.divide2(shares(rng, z), out)
        assert np.array_equal(whole(out), want)


class Plain:
    """Keys and values in the clear, and a step's stages as exact words."""

    def __init__(self, att):
        self.att, self.k, self.v = att, {}, {}

    def step(self, seqs, new, q, k, v):
        att, at = self.att, 0
        H, g = att.heads, att.heads // att.cache.kv_heads
        out = np.zeros((sum(new), H, v.shape[2]), np.int64)
        for s, n in zip(seqs, new):
            start = len(self.k.get(s, ()))
            pos, rows = np.arange(start, start + n), slice(at, at + n)
            kk = rotated(k[rows], att.k_rotary, pos)
            self.k[s] = np.concatenate([self.k[s], kk]) if s in self.k else kk
            self.v[s] = np.concatenate([self.v[s], v[rows]]) if s in self.v else v[rows]
            qq = rotated(q[rows], att.q_rotary, pos)
            for h in range(H):
                for i in range(n):
                    m = start + i + 1
                    x = (self.k[s][:m, h // g] @ qq[i, h]) >> F
                    # The reciprocal's table goes as far as the step's longest
                    # row; a sum's own pieces do not depend on that.
                    w, _, y = ref.weights(x, [0, m], F)
                    out[at + i, h] = ref.quotient(w @ self.v[s][:m, h // g], y[0])
            at += n
        return out


def run(att, plain, rng, seqs, new, v_dim):
    say("long rows %s new %s" % (seqs, new))
    T, Hk, D = sum(new), att.cache.kv_heads, att.cache.k.dim
    q, k, v = (np.rint(rng.normal(0, 1.5, n) * ONE).astype(np.int64)
               for n in ((T, att.heads, D), (T, Hk, D), (T, Hk, v_dim)))
    step = att.deal(seqs, new)
    parts = [shares(rng, x) for x in (q, k, v)]
    out = tuple(torch.empty((T, att.heads, v_dim), dtype=torch.int64, device="cuda")
                for _ in range(2))
    step.run(*parts, out)
    assert np.array_equal(whole(out), plain.step(seqs, new, q, k, v)), "step of %s" % (new,)
    return step, parts, out


def test_prompts_then_tokens_of_long_rows():
    rng = np.random.default_rng(1)
    cache = kv.PagedCache(20, 8, 2, 24, 10)
    att = kv.CachedAttention(cache, 6, STATE, 4096, rot=16)
    plain = Plain(att)
    a, b = cache.open(), cache.open()
    run(att, plain, rng, [a, b], [30, 1], 10)
    run(att, plain, rng, [b, a], [5, 1], 10)
    cache.close(a)
    c = cache.open()
    run(att, plain, rng, [c, b], [17, 1], 10)


def test_long_rows_on_request_replay():
    """long_rows for short contexts, as a graph with other shares each time."""
    rng = np.random.default_rng(2)
    cache = kv.PagedCache(16, 4, 1, 16)
    att = kv.CachedAttention(cache, 2, STATE, 64, long_rows=True)
    plain = Plain(att)
    s = cache.open()
    run(att, plain, rng, [s], [21], 16)
    keys, vals = plain.k[s], plain.v[s]
    step, parts, out = run(att, plain, rng, [s], [1], 16)
    graph = tasks.capture(lambda: step.run(*parts, out))
    for _ in range(3):
        plain.k[s], plain.v[s] = keys, vals
        x = [np.rint(rng.normal(0, 1.5, tuple(p[0].shape)) * ONE).astype(np.int64) for p in parts]
        for pair, v in zip(parts, x):
            for t, w in zip(pair, shares(rng, v)):
                t.copy_(w)
        graph.replay()
        torch.cuda.synchronize()
        got = whole(out)
        assert np.array_equal(got, plain.step([s], [1], *x))
        step.run(*parts, out)
        assert np.array_equal(whole(out), got)


def test_step_refuses_a_wrong_output():
    cache = kv.PagedCache(4, 4, 1, 8)
    att = kv.CachedAttention(cache, 2, STATE, 16, long_rows=True)
    s = cache.open()
    step = att.deal([s], [1])
    z = lambda *n: torch.zeros(n, dtype=torch.int64, device="cuda")  # noqa: E731
    q, k = (z(1, 2, 8), z(1, 2, 8)), (z(1, 1, 8), z(1, 1, 8))
    for out in ((z(1, 2, 7), z(1, 2, 7)), (z(1, 2, 8), z(1, 2, 8).float()), z(1, 2, 8),
                (z(1, 2, 8), z(1, 2, 16)[..., :8])):
        with pytest.raises(ValueError, match="out"):
            step.run(q, k, k, out)
    assert not bool(cache.k.e.any())  # nothing was opened
