"""The feed-forward operators on the CPU: workspaces, and what stands between
one use of an object and the next."""
import ctypes

import pytest

from suf_amd import native
from test_feedforward_arguments import at, linear_args


@pytest.mark.parametrize("rows,K,N", [(4, 64, 32), (1, 1, 1), (500, 64, 96), (4, 1000, 70)])
def test_a_product_without_a_gate_hands_over_both_shares(rows, K, N):
    """Nothing is opened in it, so an epilogue of its own reads two words an
    output at least; a product that writes its outputs itself reads none."""
    lib = native.load()

    def words(gate, **kw):
        a = linear_args(w__K=K, w__N=N, rows=rows, x_rows=rows, **kw)
        if not gate:
            a.trunc = None
        return lib.sufhip_linear2_work_bytes(ctypes.byref(a)) // 8

    for kw in (dict(out_digits__d_digits=at(9)), dict(walk_count=2)):
        assert words(False, **kw) >= 2 * rows * N
        assert words(True, **kw) >= rows * N
    assert words(False) in (0, words(False, walk_count=2))
