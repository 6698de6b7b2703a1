"""Attention over the paged cache as a decoder runs it: prompts, then single
tokens, sequences that come and go, pages used again.  Every step's
reconstructed output equals the closed form of its stages: exact products and
shifts, the softmax block of the fixed-point oracle."""
import gc

import numpy as np
import pytest
import torch

import fixed_point as fp
import kv_reference as ref
import oracle_lib as ol
from gpu_util import dev, say, u64
from suf_amd import kv_attention as kv
from suf_amd import native, tables, tasks

pytestmark = pytest.mark.gpu

STATE = ol.mt64_bytes(3, ol.PRG_STATE_BYTES).tobytes()
F = 12


@pytest.fixture(scope="module", autouse=True)
def _init():
    native.call("sufhip_init", 0)
    yield
    # Nothing of these tests' stays in the allocator: what a later test is
    # handed, and so the size that is counted for it, depends on free blocks.
    gc.collect()
    torch.cuda.empty_cache()


def split(rng, v):
    s = rng.integers(0, 1 << 64, v.shape, dtype=np.uint64)
    return s, v.view(np.uint64) - s


def whole(pair):
    return (u64(pair[0]) + u64(pair[1])).view(np.int64)


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


class Plain:
    """The keys and values of every sequence in the clear, and the stages."""

    def __init__(self, att):
        self.att, self.k, self.v = att, {}, {}

    def rotated(self, x, rotary, positions):
        t = rotary.table.cpu().numpy()
        out = np.stack([np.stack([ref.rotate_row(h.view(np.uint64), t[p], rotary.interleaved,
                                                 rotary.pass_mul) for h in row])
                        for row, p in zip(x, positions)])
        return out.view(np.int64) >> self.att.fc

    def step(self, seqs, new, q, k, v):
        H, Hk = self.att.heads, self.att.cache.kv_heads
        scores, at, where = {}, 0, []
        for s, n in zip(seqs, new):
            start = len(self.k.get(s, ()))
            pos = np.arange(start, start + n)
            rows = slice(at, at + n)
            kk = self.rotated(k[rows], self.att.k_rotary, pos)
            self.k[s] = np.concatenate([self.k[s], kk]) if s in self.k else kk
            self.v[s] = np.concatenate([self.v[s], v[rows]]) if s in self.v else v[rows]
            qq = self.rotated(q[rows], self.att.q_rotary, pos)
            for h in range(H):
                g = h // (H // Hk)
                full = (qq[:, h] @ self.k[s][:, g].T) >> F
                for i in range(n):
                    scores[h, at + i] = full[i, :start + i + 1]
            where += [s] * n
            at += n
        order = [(h, t) for h in range(H) for t in range(at)]
        off = np.concatenate([[0], np.cumsum([len(scores[o]) for o in order])])
        prob, _ = fp.softmax_block(np.concatenate([scores[o] for o in order]), off,
                                   tables.nexp_table(F), tables.recip_table(F), F)
        out = np.zeros((at, H, self.v[where[0]].shape[2]), np.int64)
        for i, (h, t) in enumerate(order):
            p = prob[off[i]:off[i + 1]]
            out[t, h] = (p @ self.v[where[t]][:len(p), h // (H // Hk)]) >> F
        return out


def run(att, plain, rng, seqs, new):
    say("cached attention %s new %s" % (seqs, new))
    cache, T = att.cache, sum(new)
    step = att.deal(seqs, new)
    mk = lambda heads, dim, sigma: np.rint(  # noqa: E731
        rng.normal(0, sigma, (T, heads, dim)) * (1 << F)).astype(np.int64)
    q, k = mk(att.heads, cache.k.dim, 2.0), mk(cache.kv_heads, cache.k.dim, 2.0)
    v = mk(cache.kv_heads, cache.v.dim, 1.0)
    # The three as parts of one buffer, like a fused product's rows.
    width = q[0].size + k[0].size + v[0].size
    bufs = [np.zeros((T, width), np.uint64) for _ in range(2)]
    o = 0
    for x in (q, k, v):
        for buf, s in zip(bufs, split(rng, x)):
            buf[:, o:o + x[0].size] = s.reshape(T, -1)
        o += x[0].size
    bufs = [dev(b) for b in bufs]
    parts, o = [], 0
    for x in (q, k, v):
        parts.append([b[:, o:o + x[0].size].view(T, x.shape[1], x.shape[2]) for b in bufs])
        o += x[0].size
    out = tuple(torch.empty((T, att.heads, cache.v.dim), dtype=torch.int64, device="cuda")
                for _ in range(2))
    step.run(*parts, out)
    want = plain.step(seqs, new, q, k, v)
    assert np.array_equal(whole(out), want), "step of %s" % (new,)
    return step, parts, out, want


@pytest.mark.parametrize("kv_heads,group,dim,v_dim,page,rot,neigh,scaling", [
    (2, 2, 32, None, 4, None, False, None),
    (1, 4, 64, 40, 16, 48, True, ("linear", 4)),
    (3, 1, 20, None, 2, 8, False, ("parts", 4, 16, 1, 4)),
])
def test_prompts_then_tokens(kv_heads, group, dim, v_dim, page, rot, neigh, scaling):
    rng = np.random.default_rng(dim)
    cache = kv.PagedCache(60 // page + 8, page, kv_heads, dim, v_dim)
    att = kv.CachedAttention(cache, kv_heads * group, STATE, 64, rot=rot, interleaved=neigh,
                             scaling=scaling)
    plain = Plain(att)
    a, b, c = cache.open(), cache.open(), cache.open()
    run(att, plain, rng, [a, b], [9, 1])
    run(att, plain, rng, [a, b], [1, 1])
    run(att, plain, rng, [c, a], [7, 3])       # another prompt beside a few tokens
    run(att, plain, rng, [b, a, c], [1, 1, 1])
    cache.close(a)                             # its pages go to the next ones
    d = cache.open()
    run(att, plain, rng, [d, c], [21, 1])
    run(att, plain, rng, [c, d, b], [1, 1, 1])


def test_rows_past_the_one_launch_softmax():
    """More keys than the softmax block takes in its one launch."""
    rng = np.random.default_rng(8)
    cache = kv.PagedCache(10, 64, 1, 8)
    att = kv.CachedAttention(cache, 2, STATE, 600)
    plain = Plain(att)
    s = cache.open()
    run(att, plain, rng, [s], [40])
    run(att, plain, rng, [s], [500])
    run(att, plain, rng, [s], [1])


def test_captured_step_replays():
    """A step's launches as a graph, replayed with other shares of other
    values, beside eager work."""
    rng = np.random.default_rng(4)
    cache = kv.PagedCache(16, 4, 2, 32)
    att = kv.CachedAttention(cache, 4, STATE, 64)
    plain = Plain(att)
    s = cache.open()
    run(att, plain, rng, [s], [13])
    keys, vals = plain.k[s], plain.v[s]
    step, parts, out, want = run(att, plain, rng, [s], [1])
    graph = tasks.capture(lambda: step.run(*parts, out))
    for _ in range(3):
        plain.k[s], plain.v[s] = keys, vals
        x = [np.rint(rng.normal(0, 1.5, p[0].shape) * (1 << F)).astype(np.int64) for p in parts]
        for pair, v in zip(parts, x):
            for t, w in zip(pair, split(rng, v)):
                t.copy_(dev(w))
        graph.replay()
        torch.cuda.synchronize()
        got = whole(out)
        assert np.array_equal(got, plain.step([s], [1], *x))
        step.run(*parts, out)
        assert np.array_equal(whole(out), got)


def test_a_key_is_opened_under_its_own_mask():
    """The same value twice: E is value - mask with the dealer's whole mask,
    another one each time."""
    cache = kv.PagedCache(4, 4, 1, 16)
    att = kv.CachedAttention(cache, 1, STATE, 16)
    opens = []
    for _ in range(2):
        s = cache.open()
        step = att.deal([s], [1])
        one = tuple(torch.ones((1, 1, 16), dtype=torch.int64, device="cuda") for _ in range(2))
        out = tuple(torch.empty((1, 1, 16), dtype=torch.int64, device="cuda") for _ in range(2))
        step.run(one, one, one, out)
        page = cache.seqs[s]["pages"][0]
        opens.append(cache.v.e[page, 0, 0].clone())
        assert torch.equal(opens[-1], 2 - step.v_mask[0][0, 0] - step.v_mask[1][0, 0])
    assert not bool((opens[0] == opens[1]).any())


def test_dealing_opens_nothing():
    """The masks are in their pages before the step's values are, beside an E
    that does not depend on them."""
    cache = kv.PagedCache(4, 4, 2, 8, 6)
    att = kv.CachedAttention(cache, 2, STATE, 16)
    s = cache.open()
    step = att.deal([s], [5])
    for pool, mask in ((cache.k, step.k_mask), (cache.v, step.v_mask)):
        assert not bool(pool.e.any())
        for p in (0, 1):
            rows = torch.cat([pool.b[p][i].transpose(0, 1) for i in cache.seqs[s]["pages"]])
            assert torch.equal(rows[:5], mask[p]) and not bool(rows[5:].any())


def test_cache_bookkeeping():
    cache = kv.PagedCache(6, 4, 1, 8)
    att = kv.CachedAttention(cache, 2, STATE, 20)
    a, b = cache.open(), cache.open()
    cache.extend([a, b], [5, 1])
    assert [cache.length(s) for s in (a, b)] == [5, 1] and len(cache.free) == 3
    before = (list(cache.free), {s: dict(v, pages=list(v["pages"])) for s, v in cache.seqs.items()})
    with pytest.raises(RuntimeError, match="pages"):
        cache.extend([a, b], [12, 4])
    assert (cache.free, cache.seqs) == before  # nothing changed
    for seqs, new in (([a, a], [1, 1]), ([a], [1, 1]), ([a], [-1])):
        with pytest.raises(ValueError):
            cache.extend(seqs, new)
    with pytest.raises(ValueError, match="max_positions"):
        att.deal([a], [16])
    with pytest.raises(ValueError, match="new token"):
        att.deal([a], [0])
    assert cache.extend([], []).tokens == 0
    cache.close(a)
    assert len(cache.free) == 5 and a not in cache.seqs
    with pytest.raises(ValueError, match="multiple"):
        kv.CachedAttention(kv.PagedCache(1, 1, 2, 8), 3, STATE, 4)


def test_sizes_past_32_bits_are_refused():
    """Counts that the library would take modulo 2^32."""
    z = lambda *n: torch.zeros(n, dtype=torch.int64, device="cuda")  # noqa: E731
    cache = kv.PagedCache(4, 4, 1, 8)
    s = cache.open()
    b = cache.extend([s], [1])
    for kw in ({"tokens": 1 << 32}, {"max_new": 1 << 31}, {"max_keys": 1 << 31}, {"tokens": -1}):
        with pytest.raises(ValueError, match="2\\^31"):
            kv.Batch(b.cu, b.kv_lens, b.pages, **dict({"tokens": 1, "max_new": 1, "max_keys": 1},
                                                      **kw))
    with pytest.raises(ValueError, match="2\\^31"):
        kv.Pool(*(z(1 << 32, 0, 4, 8) for _ in range(3)))
    r = kv.Rotary.build(8, 4)
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    for shape in ((1, 1 << 32, 8), (1 << 32, 1, 8)):
        x = tuple(z(1, 1, 8).expand(shape) for _ in range(2))
        with pytest.raises(ValueError, match="2\\^31"):
            kv.rotary2(x, r, pos.expand(shape[0]), out=x)
    x = tuple(z(1, 1, 8).expand(1, 1 << 32, 8) for _ in range(2))
    with pytest.raises(ValueError, match="2\\^31"):
        kv.scores2(b, cache.k, x, x, (z(1), z(1)), pos, (z(1), z(1)))


def test_a_step_of_too_many_scores_changes_nothing():
    n = 1 << 16  # n (n + 1) / 2 scores a head
    cache = kv.PagedCache(n // 64, 64, 1, 2)
    att = kv.CachedAttention(cache, 1, STATE, n)
    s = cache.open()
    with pytest.raises(ValueError, match="2\\^31"):
        att.deal([s], [n])
    assert cache.length(s) == 0 and len(cache.free) == n // 64
    for bits in ({"frac_bits": 0}, {"frac_bits": 15}, {"table_bits": 0}, {"table_bits": 15}):
        with pytest.raises(ValueError, match="bits"):
            kv.CachedAttention(cache, 1, STATE, 4, **bits)


class OtherDevice:
    """A prepared gate whose table is not on the tensors' GPU."""
    n, mask, work = 1 << 20, 0, [torch.zeros(2, dtype=torch.int64)] * 2

    def has_table(self):
        return True

    def epilogue(self, y):
        raise AssertionError("used")


def test_gates_on_another_device_are_refused():
    cache = kv.PagedCache(4, 4, 1, 8)
    s = cache.open()
    b = cache.extend([s], [1])
    z = lambda *n: torch.zeros(n, dtype=torch.int64, device="cuda")  # noqa: E731
    x, p, off = (z(1, 1, 8), z(1, 1, 8)), (z(1), z(1)), i32([0, 1])
    gate = OtherDevice()
    for call in (lambda: kv.rotary2(x, kv.Rotary.build(8, 4), i32([0]), trunc=gate),
                 lambda: kv.append2(b, cache.k, x, x, k_trunc=gate),
                 lambda: kv.scores2(b, cache.k, x, x, p, off, p, trunc=gate),
                 lambda: kv.values2(b, cache.v, p, p, x, off, x, trunc=gate)):
        with pytest.raises(ValueError, match="another device"):
            call()


def test_calls_refuse_wrong_tensors():
    """What the calls say of a wrong tensor, before any launch."""
    cache = kv.PagedCache(4, 4, 2, 16)
    s = cache.open()
    b = cache.extend([s], [3])
    z = lambda *n: torch.zeros(n, dtype=torch.int64, device="cuda")  # noqa: E731
    x, kx = (z(3, 4, 16), z(3, 4, 16)), (z(3, 2, 16), z(3, 2, 16))
    off = torch.tensor(kv.causal_row_offsets([3], [3], 4), dtype=torch.int32, device="cuda")
    n = int(off[-1])
    p = (z(n), z(n))
    r = kv.Rotary.build(16, 8)
    pos = torch.arange(3, dtype=torch.int32, device="cuda")
    gate = tasks.Trunc(tasks.Dealer(1), 12, 5, STATE)
    wide = tasks.Trunc(tasks.Dealer(1), 20, 500, STATE)
    bad = [
        lambda: kv.rotary2(x, r, pos.long()),
        lambda: kv.rotary2(x, r, pos[:2]),
        lambda: kv.rotary2((x[0], x[1][:2]), r, pos),
        lambda: kv.rotary2((x[0], z(3, 8, 16)[:, ::2]), r, pos),
        lambda: kv.rotary2((x[0], x[1].cpu()), r, pos),
        lambda: kv.rotary2(x[0], r, pos),
        lambda: kv.rotary2((z(3, 4, 8), z(3, 4, 8)), r, pos),
        lambda: kv.rotary2(tuple(v.transpose(1, 2).contiguous().transpose(1, 2) for v in x), r, pos),
        lambda: kv.rotary2(x, r, pos, out=tuple(z(1, 4, 16).expand(3, 4, 16) for _ in range(2))),
        lambda: kv.rotary2(x, r, pos, trunc=gate),
        lambda: kv.rotary2(x, r, pos, trunc=wide),
        lambda: kv.append2(b, cache.k, x, x),
        lambda: kv.append2(b, cache.k, kx, (kx[0], kx[1].float())),
        lambda: kv.append2(b, cache.k, kx, kx, rotary=kv.Rotary.build(32, 8)),
        lambda: kv.append2(b, cache.k, kx, kx, rotary=r, positions=pos[:1]),
        lambda: kv.append2(b, cache.k, kx, kx, cache.v, x, kx),
        lambda: kv.scores2(b, cache.k, x, kx, p, off, p),
        lambda: kv.scores2(b, cache.k, x, x, p, off[1:], p),
        lambda: kv.scores2(b, cache.k, x, x, (z(n - 1), z(n - 1)), off, p),
        lambda: kv.scores2(b, cache.k, x, x, p, off, p, trunc=gate),
        lambda: kv.values2(b, cache.v, p, (z(n + 1), z(n + 1)), x, off, x),
        lambda: kv.values2(b, cache.v, p, p, kx, off, x),
        lambda: kv.values2(b, cache.v, p, p, x, off, (x[0], z(3, 4, 32)[..., :16])),
        lambda: kv.values2(b, cache.v, p, p, x, off, x, work=z(4)[::2]),
        lambda: kv.Pool(cache.k.e, cache.k.b[0], z(4, 2, 4, 8)),
        lambda: kv.Rotary(r.table, 8),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(native.SufHipError, match="power of two"):
        odd = kv.Pool(*(z(4, 2, 3, 16) for _ in range(3)))
        kv.append2(b, odd, kx, kx)
    with pytest.raises(native.SufHipError, match="d_work"):
        long = kv.Batch(b.cu, b.kv_lens, b.pages, tokens=3, max_new=3, max_keys=1000)
        kv.values2(long, cache.v, p, p, x, off, x, work=z(2))
