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


class Anything:
    """Not read before the refusal."""


@pytest.mark.parametrize("kw", [{"v": 1}, {"v_mask": 1}, {"v_trunc": 1}, {"positions": 1}])
def test_append_arguments_without_their_part_are_refused(kw):
    with pytest.raises(ValueError, match="need"):
        kv.append2(Anything(), None, None, None, **kw)
