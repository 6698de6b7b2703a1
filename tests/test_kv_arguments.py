"""Arguments of the cached-attention calls at their edges, on the CPU: what is
taken and what is refused before any device work."""
import ctypes

import pytest
import torch

from suf_amd import kv_attention as kv
from suf_amd import native
from test_kv_attention import append_args, batch, pool, product_args, refused, rotary_args


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


# ---- a rotation's outputs ----

def meets(T, H, D, x, out):
    """By every word: whether an output word is another output's, or an input
    word of another row or place (x, out: (address, token, head stride) of each
    party, in words)."""
    def words(rows):
        base, ts, hs = rows
        return {(t, h, i): base + t * ts + h * hs + i
                for t in range(T) for h in range(H) for i in range(D)}
    o = [words(r) for r in out]
    if len(set(o[0].values()) | set(o[1].values())) < 2 * T * H * D:
        return True
    for q in o:
        at = {w: k for k, w in q.items()}
        for r in x:
            if any(w in at and at[w] != k for k, w in words(r).items()):
                return True
    return False


def rotary_of(T, H, D, x, out):
    a = rotary_args(tokens=T, heads=H, dim=D)
    a.rot.rot = 0
    for p in range(2):
        a.x.p[p], a.out[p] = 8 * x[p][0], 8 * out[p][0]
    _, a.x.token_stride, a.x.head_stride = x[0]
    _, a.out_token_stride, a.out_head_stride = out[0]
    return a


BASE = 1 << 20
OVERLAPS = [
    # tokens, heads, dim, strides of x, offset and strides of out in party 0's buffer
    (3, 2, 8, (16, 8), 1, (16, 8)),       # a word further
    (3, 2, 8, (16, 8), 8, (16, 8)),       # a head further
    (3, 2, 8, (16, 8), 16, (16, 8)),      # a token further
    (3, 2, 8, (16, 8), 0, (8, 24)),       # in place with the axes exchanged
    (3, 2, 8, (48, 8), 12, (48, 8)),      # half a head into the next part
    (3, 2, 8, (48, 24), 4, (48, 24)),
    (5, 1, 8, (8, 8), 32, (8, 8)),
    (1, 4, 6, (0, 6), 3, (0, 6)),
]


@pytest.mark.parametrize("T,H,D,xs,at,os", OVERLAPS)
def test_rotary_refuses_outputs_over_other_inputs(T, H, D, xs, at, os):
    x = [(BASE, *xs), (BASE + 5000, *xs)]
    out = [(BASE + at, *os), (BASE + 9000, *os)]
    assert meets(T, H, D, x, out)
    refused("sufhip_rotary2", rotary_of(T, H, D, x, out), "overlap")
    refused("sufhip_rotary2", rotary_of(T, H, D, x, out[::-1]), "overlap")


@pytest.mark.parametrize("T,H,D,ts,hs", [(2, 2, 8, 8, 8), (3, 2, 8, 16, 7), (2, 3, 8, 4, 100),
                                         (3, 4, 4, 12, 8), (2, 2, 8, 0, 8), (5, 7, 3, 9, 6)])
def test_rotary_refuses_output_rows_over_each_other(T, H, D, ts, hs):
    x = [(BASE, 1000, 100), (BASE + 10000, 1000, 100)]
    out = [(BASE + 20000, ts, hs), (BASE + 30000, ts, hs)]
    assert meets(T, H, D, x, out)
    refused("sufhip_rotary2", rotary_of(T, H, D, x, out), "output rows overlap")


@pytest.mark.parametrize("by", [0, 1, 8, 60])
def test_rotary_refuses_one_output_for_both_parties(by):
    x = [(BASE, 64, 8), (BASE + 10000, 64, 8)]
    out = [(BASE + 20000, 64, 8), (BASE + 20000 + by, 64, 8)]
    if meets(2, 6, 8, x, out):
        refused("sufhip_rotary2", rotary_of(2, 6, 8, x, out), "output rows overlap")
    else:
        assert by == 48


# ---- strides of axes of one ----

@pytest.mark.parametrize("shape", [(1, 4, 8), (4, 1, 8), (1, 1, 8), (3, 4, 1), (1, 1, 1), (0, 4, 8)])
def test_strides_along_an_axis_of_one_do_not_matter(shape):
    """A single token out of wider rows beside one of its own."""
    base = torch.zeros(4096, dtype=torch.int64)
    st = [1]
    for n in shape[:0:-1]:
        st.insert(0, st[0] * max(n, 1))
    odd = [999 if n <= 1 else s for n, s in zip(shape, st)]
    pair = (torch.as_strided(base, shape, st), torch.as_strided(base, shape, odd, 2048))
    for p in (pair, pair[::-1]):
        arr = [0, 0]
        ts, hs = kv._rows(arr, p, shape, -1, "here", "x", written=True)
        assert arr == [t.data_ptr() for t in p]
        assert (shape[0] <= 1 or ts == st[0]) and (shape[1] <= 1 or hs == st[1])


@pytest.mark.parametrize("shape,a,b", [((2, 3, 4), (12, 4, 1), (24, 4, 1)),
                                       ((2, 3, 4), (12, 4, 1), (12, 8, 1)),
                                       ((1, 3, 4), (12, 4, 1), (12, 8, 1)),
                                       ((2, 3, 4), (12, 4, 1), (12, 1, 3)),
                                       ((2, 3, 4), (12, 1, 3), (12, 1, 3))])
def test_strides_that_differ_are_refused(shape, a, b):
    base = torch.zeros(256, dtype=torch.int64)
    for u, v in ((a, b), (b, a)):
        with pytest.raises(ValueError, match="strides|neighbours"):
            kv._rows([0, 0], (torch.as_strided(base, shape, u), torch.as_strided(base, shape, v)),
                     shape, -1, "here", "x")


# ---- rotary tables ----

def test_a_tables_one_fits_its_words():
    """2^31 - 1 is the largest word; a quarter more rounds to it, 2^31 does not."""
    top = 2.0 ** 31
    for one in (top - 1, top - 0.75, 1 - top):
        t, got = kv.rotary_table(3, 4, frac_bits=20, scale=one / 2.0 ** 20)
        assert got == round(one) and (t[0, :, 0] == round(one)).all() and abs(t[0, 0, 0]) < top
    for one in (top - 0.25, top, -top + 0.25, -top, float("nan"), float("inf"), -float("inf")):
        with pytest.raises(ValueError, match="2\\^31"):
            kv.rotary_table(3, 4, frac_bits=20, scale=one / 2.0 ** 20)


@pytest.mark.parametrize("kw", [{"base": 0.0}, {"base": -2.0}, {"base": float("nan")},
                                {"base": float("inf")}, {"scaling": ("linear", float("nan"))},
                                {"scaling": ("linear", float("inf"))},
                                {"scaling": ("parts", 2.0, float("nan"), 1, 4)},
                                {"scaling": ("parts", 2.0, 64, 1, float("nan"))},
                                {"scaling": ("parts", 2.0, 64)}, {"scaling": ()},
                                {"scaling": ("linear",)}])
def test_a_tables_angles_are_numbers(kw):
    with pytest.raises(ValueError, match="rotary_table"):
        kv.rotary_table(5, 8, **kw)


@pytest.mark.parametrize("pages,page,heads,dim,v_dim", [
    (4, 3, 1, 8, None), (4, 0, 1, 8, None), (4, -4, 1, 8, None), (-1, 4, 1, 8, None),
    (4, 4, 0, 8, None), (4, 4, 1, 0, None), (4, 4, 1, 257, None), (4, 4, 1, 8, 0),
    (4, 4, 1, 8, 257)])
def test_a_cache_of_pages_that_no_call_takes_is_refused(pages, page, heads, dim, v_dim):
    """When it is made, not at its first step."""
    with pytest.raises(ValueError, match="PagedCache"):
        kv.PagedCache(pages, page, heads, dim, v_dim, device="cpu")


def work_bytes(heads, **kw):
    a = product_args()
    batch(a.batch, **kw)
    pool(a.pool, pages=16, kv_heads=2, dim=128)
    return native.load().sufhip_kv_values2_work_bytes(ctypes.byref(a.batch),
                                                      ctypes.byref(a.pool), heads)


@pytest.mark.parametrize("heads", [2, 1 << 10, 1 << 20, 1 << 28])
@pytest.mark.parametrize("seqs", [1, 64, 1 << 16, 1 << 20])
def test_any_bounds_lay_a_launch_out(heads, seqs):
    """Products of bounds do not wrap: more new tokens than the batch has are
    as many as it has, and more keys never take the layout of fewer."""
    top = 2 ** 31 - 1
    for keys in (32, 300, 1 << 20, top):
        at = [work_bytes(heads, seqs=seqs, tokens=1, max_new=n, max_keys=keys)
              for n in (1, 2, 1 << 16, top)]
        assert len(set(at)) == 1, at
        # Two slots of 16 KB for each of two workgroups a CU, 16 bytes a row.
        assert at[0] <= (2 << 30) + 2 * 2 * 256 * 16384 + heads * 2 * 16, at
