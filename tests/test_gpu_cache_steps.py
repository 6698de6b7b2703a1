"""The cache's state and the order of its steps: what raises leaves it as it
was, and no step runs on pages that are not its own."""
import gc
import warnings

import pytest
import torch

import oracle_lib as ol
from suf_amd import kv_attention as kv
from suf_amd import native, tasks

pytestmark = pytest.mark.gpu

STATE = ol.mt64_bytes(3, ol.PRG_STATE_BYTES).tobytes()


@pytest.fixture(scope="module", autouse=True)
def _init():
    native.call("sufhip_init", 0)
    yield
    gc.collect()
    torch.cuda.empty_cache()


def z(*n):
    return torch.zeros(n, dtype=torch.int64, device="cuda")


def one(att, tokens=1):
    """Inputs of a step of `tokens` tokens, and its output."""
    c = att.cache
    kvs = [tuple(torch.ones((tokens, c.kv_heads, c.k.dim), dtype=torch.int64, device="cuda")
                 for _ in range(2)) for _ in range(2)]
    q = tuple(torch.ones((tokens, att.heads, c.k.dim), dtype=torch.int64, device="cuda")
              for _ in range(2))
    return (q, *kvs, (z(tokens, att.heads, c.v.dim), z(tokens, att.heads, c.v.dim)))


def state_of(cache):
    return list(cache.free), {s: dict(v, pages=list(v["pages"])) for s, v in cache.seqs.items()}


def fail(*args, **kw):
    raise MemoryError("injected")


@pytest.mark.parametrize("where", ["Batch", "values_work", "Trunc", "SoftmaxBlock"])
def test_a_deal_that_fails_changes_nothing(monkeypatch, where):
    cache = kv.PagedCache(8, 4, 1, 8)
    att = kv.CachedAttention(cache, 2, STATE, 20)
    a, b = cache.open(), cache.open()
    att.deal([a], [6]).run(*one(att, 6))
    att.deal([b], [1]).run(*one(att))
    before = state_of(cache)
    with monkeypatch.context() as m:
        m.setattr(kv, where, fail)
        with pytest.raises(MemoryError):
            att.deal([b, a], [9, 3])
    assert state_of(cache) == before
    step = att.deal([b, a], [9, 3])
    assert [cache.length(s) for s in (a, b)] == [9, 10] and len(cache.free) == 8 - 3 - 3
    step.run(*one(att, 12))


def test_steps_run_in_the_order_of_their_deal():
    cache = kv.PagedCache(8, 4, 1, 8)
    att = kv.CachedAttention(cache, 2, STATE, 20)
    a, b = cache.open(), cache.open()
    first, other = att.deal([a], [3]), att.deal([b], [2])
    second = att.deal([b, a], [1, 1])
    with pytest.raises(RuntimeError, match="earlier step"):
        second.run(*one(att, 2))
    first.run(*one(att, 3))
    with pytest.raises(RuntimeError, match="earlier step"):
        second.run(*one(att, 2))
    assert not bool(cache.k.e[cache.seqs[b]["pages"][0]].any())  # nothing was opened
    other.run(*one(att, 2))
    second.run(*one(att, 2))
    e = cache.k.e.clone()
    for late, n in ((first, 3), (other, 2)):
        with pytest.raises(RuntimeError, match="later step"):
            late.run(*one(att, n))
    assert torch.equal(cache.k.e, e)


def test_a_closed_sequences_step_does_not_run():
    """Its pages are another sequence's by then."""
    cache = kv.PagedCache(2, 4, 1, 8)
    att = kv.CachedAttention(cache, 2, STATE, 8)
    a = cache.open()
    old = att.deal([a], [8])
    cache.close(a)
    b = cache.open()
    att.deal([b], [8]).run(*one(att, 8))
    words = [t.clone() for p in (cache.k, cache.v) for t in (p.e,) + p.b]
    with pytest.raises(RuntimeError, match="closed"):
        old.run(*one(att, 8))
    assert all(torch.equal(t, w) for t, w in
               zip([t for p in (cache.k, cache.v) for t in (p.e,) + p.b], words))


def test_a_second_run_is_warned_of():
    cache = kv.PagedCache(4, 4, 1, 8)
    att = kv.CachedAttention(cache, 2, STATE, 8)
    step = att.deal([cache.open()], [1])
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        step.run(*one(att))
    with pytest.warns(RuntimeWarning, match="one use"):
        step.run(*one(att))


def test_a_refused_call_does_not_use_a_step():
    cache = kv.PagedCache(4, 4, 1, 8)
    att = kv.CachedAttention(cache, 2, STATE, 8)
    step = att.deal([cache.open()], [1])
    q, k, v, out = one(att)
    for bad in ((q, k, v, q[0]), (k, k, v, out), (q, q, v, out), (q, k, q, out),
                (q[0], k, v, out), (q, k, None, out), (q, k, [t.float() for t in v], out)):
        with pytest.raises((ValueError, TypeError)):
            step.run(*bad)
    assert not bool(cache.k.e.any())
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        step.run(q, k, v, out)


def test_a_step_is_dealt_and_run_on_the_caches_device(monkeypatch):
    """Launches that go to the current device and its stream (the gates', the
    softmax's) are issued with the cache's as the current one."""
    real, inside, seen = torch.cuda.device, [], []

    class Spy(real):
        def __enter__(self):
            inside.append(self.idx)
            return super().__enter__()

        def __exit__(self, *a):
            inside.pop()
            return super().__exit__(*a)

    prepare, gen = kv.prepare_batch, tasks.pfss.trunc_gen
    monkeypatch.setattr(torch.cuda, "device", Spy)
    monkeypatch.setattr(kv, "prepare_batch", lambda t: (seen.append(list(inside)), prepare(t))[1])
    monkeypatch.setattr(tasks.pfss, "trunc_gen",
                        lambda *a, **k: (seen.append(list(inside)), gen(*a, **k))[1])
    cache = kv.PagedCache(4, 4, 1, 8, device="cuda:0")
    att = kv.CachedAttention(cache, 2, STATE, 8)
    att.deal([cache.open()], [2]).run(*one(att, 2))
    assert len(seen) > 4 and all(s and s[-1] == 0 for s in seen)
