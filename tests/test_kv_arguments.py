"""Arguments of the cached-attention calls at their edges, on the CPU: what is
taken and what is refused before any device work."""
import ctypes

import pytest

from suf_amd import kv_attention as kv
from suf_amd import native
from test_kv_attention import append_args, batch, refused


@pytest.mark.parametrize("none", [{"seqs": 0}, {"tokens": 0}, {"seqs": 0, "tokens": 0}])
def test_an_append_of_no_tokens_does_nothing(none):
    """A tensor without elements has no address."""
    a = append_args()
    batch(a.batch, **none)
    for p in a.part:
        for i in range(2):
            p.x.p[i] = p.mask[i] = None
    assert native.load().sufhip_kv_append2(ctypes.byref(a), None) == 0
    batch(a.batch)
    refused("sufhip_kv_append2", a, "rows")


@pytest.mark.parametrize("k", range(3))
@pytest.mark.parametrize("v", range(3))
def test_pools_that_share_memory_are_refused(k, v):
    """Keys and values of one call are written in no order."""
    a = append_args()
    words = 4 * 2 * 16 * 64  # of each array of the pools
    at = [[1 << 20 | i << 24 for i in range(3)], [1 << 20 | (i + 1) << 28 for i in range(3)]]
    for p, q in zip(a.part, at):
        p.pool.e, p.pool.b[0], p.pool.b[1] = q
    # The last word of one array is the first of another.
    at[1][v] = at[0][k] + 8 * (words - 1)
    a.part[1].pool.e, a.part[1].pool.b[0], a.part[1].pool.b[1] = at[1]
    refused("sufhip_kv_append2", a, "share memory")


class Anything:
    """Not read before the refusal."""


@pytest.mark.parametrize("kw", [{"v": 1}, {"v_mask": 1}, {"v_trunc": 1}, {"positions": 1}])
def test_append_arguments_without_their_part_are_refused(kw):
    with pytest.raises(ValueError, match="need"):
        kv.append2(Anything(), None, None, None, **kw)
