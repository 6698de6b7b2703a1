"""The cache's state and the order of its steps: what raises leaves it as it
was, and no step runs on pages that are not its own."""
import gc

import pytest
import torch

import oracle_lib as ol
from suf_amd import kv_attention as kv
from suf_amd import native

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
