"""Rotary positions, the append to a paged cache and the two products of
attention over it, against plain numpy forms: bit-equal shares (everything is
an integer mod 2^64), and every word that a call must not touch as it was."""
import gc

import numpy as np
import pytest
import torch

import kv_reference as ref
import oracle_lib as ol
from gpu_util import dev, say, u64
from suf_amd import kv_attention as kv
from suf_amd import native, tasks

pytestmark = pytest.mark.gpu

STATE = ol.mt64_bytes(3, ol.PRG_STATE_BYTES).tobytes()


@pytest.fixture(scope="module", autouse=True)
def _init():
    native.call("sufhip_init", 0)
    yield
    # Nothing of these tests' stays in the allocator: what a later test is
    # handed, and so the size that is counted for it, depends on free blocks.
    gc.collect()
    torch.cuda.empty_cache()


def dev2(pair):
    return tuple(dev(v) for v in pair)


def eq(got, want, what):
    for p in range(2):
        g = u64(got[p])
        assert np.array_equal(g, want[p]), "%s: party %d, %d of %d differ" % (
            what, p, int((g != want[p]).sum()), g.size)


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def batch_of(c, max_new=None, max_keys=None):
    return kv.Batch(i32(c.cu), i32(np.array(c.lens).reshape(-1)), i32(c.table), tokens=c.tokens,
                    max_new=max(c.new + [0]) if max_new is None else max_new,
                    max_keys=max(c.lens + [0]) if max_keys is None else max_keys)


def view_of(x, lead=0, gap_t=0, gap_h=0):
    """A device copy of x [tokens, heads, dim] as a view into a larger buffer:
    `lead` words before it, gaps behind every head and token.  (view, buffer)"""
    T, H, D = x.shape
    ts = H * (D + gap_h) + gap_t
    buf = torch.full((lead + T * ts + 1,), -77, dtype=torch.int64, device="cuda")
    v = torch.as_strided(buf, (T, H, D), (ts, D + gap_h, 1), lead)
    v.copy_(dev(x))
    return v, buf


# ---- rotary ----

@pytest.mark.parametrize("T,H,D,rot,neigh,lead,gap_t,gap_h", [
    (1, 1, 2, 2, False, 0, 0, 0),
    (1, 12, 64, 64, False, 0, 0, 0),
    (5, 3, 64, 64, True, 0, 0, 0),
    (7, 2, 80, 32, True, 0, 64, 0),     # part of the head, a view of wider rows
    (7, 2, 80, 32, False, 2, 0, 6),
    (3, 5, 64, 20, False, 0, 0, 0),     # 10 pairs; a tail of 44
    (3, 5, 66, 20, True, 0, 0, 0),      # the last piece of the tail is half a unit
    (3, 2, 33, 6, False, 0, 0, 0),      # odd head, odd pairs
    (3, 2, 33, 32, True, 0, 0, 0),
    (4, 3, 64, 64, False, 1, 0, 0),     # 8-byte alignment only
    (4, 3, 64, 64, True, 0, 1, 0),      # odd token stride
    (4, 3, 64, 0, False, 0, 0, 0),      # nothing rotated
    (700, 9, 40, 40, False, 0, 0, 0),
])
def test_rotary_shapes(T, H, D, rot, neigh, lead, gap_t, gap_h):
    say("rotary T=%d H=%d D=%d rot=%d neigh=%d" % (T, H, D, rot, neigh))
    rng = np.random.default_rng(T * 1000 + D)
    x = [ref.words(rng, T, H, D) for _ in range(2)]
    table = rng.integers(-2 ** 31, 2 ** 31, (50, rot // 2, 2), dtype=np.int32)
    pos = rng.integers(0, 50, T)
    pos[rng.random(T) < 0.2] = rng.choice([-1, 50, 2 ** 31 - 1, -2 ** 31])
    r = kv.Rotary(i32(table).reshape(50, rot // 2, 2), D, interleaved=neigh, pass_mul=-12345)
    before = [ref.words(rng, T, H, D) for _ in range(2)]
    want = [ref.rotary(x[p], table, pos, neigh, -12345, before[p]) for p in range(2)]
    xv, ov = ([view_of(v, lead, gap_t, gap_h) for v in w] for w in (x, before))
    frames = [b.clone() for _, b in ov]
    kv.rotary2([v for v, _ in xv], r, i32(pos), [v for v, _ in ov])
    eq([v.contiguous() for v, _ in ov], want, "out")
    for (v, b), f in zip(ov, frames):  # the gaps are as they were
        inside = torch.zeros_like(b, dtype=torch.bool)
        torch.as_strided(inside, v.shape, v.stride(), v.storage_offset()).fill_(True)
        assert torch.equal(b[~inside], f[~inside])
    # In place, and into new tensors (zeros in padding rows).
    want_z = [ref.rotary(x[p], table, pos, neigh, -12345, np.zeros_like(x[p])) for p in range(2)]
    eq(kv.rotary2([v for v, _ in xv], r, i32(pos)), want_z, "new")
    want_i = [ref.rotary(x[p], table, pos, neigh, -12345, x[p]) for p in range(2)]
    kv.rotary2([v for v, _ in xv], r, i32(pos), [v for v, _ in xv])
    eq([v.contiguous() for v, _ in xv], want_i, "in place")


def test_rotary_empty():
    r = kv.Rotary(torch.zeros(0, 4, 2, dtype=torch.int32, device="cuda"), 8)
    x = tuple(torch.ones(3, 2, 8, dtype=torch.int64, device="cuda") for _ in range(2))
    kv.rotary2(x, r, i32([0, 1, 2]), x)  # no positions: every row is padding
    assert all(bool((v == 1).all()) for v in x)
    none = tuple(torch.empty(0, 2, 8, dtype=torch.int64, device="cuda") for _ in range(2))
    kv.rotary2(none, r, i32([]), none)


@pytest.mark.parametrize("D,rot,lead", [(64, 64, 0), (33, 10, 1)])
def test_rotary_truncates(D, rot, lead):
    """Through the gate: the shares of the unfused rotation, open and gate."""
    rng = np.random.default_rng(5)
    T, H = 9, 3
    val = rng.integers(-1 << 20, 1 << 20, (T, H, D)).astype(np.int64).view(np.uint64)
    s0 = ref.words(rng, T, H, D)
    x = dev2([s0, val - s0])
    r = kv.Rotary.build(D, 64, rot=rot)
    pos = i32(rng.integers(0, 64, T))
    gate = tasks.Trunc(tasks.Dealer(3), 12, T * H * D, STATE)
    gate.prepare()
    plain = kv.rotary2(x, r, pos)
    want = tasks.pair(T * H * D)
    flat = tuple(v.reshape(-1) for v in plain)
    tasks.lin2(tasks.operand(tasks.term(flat)), T * H * D, into=(gate, want))
    out = [view_of(np.zeros((T, H, D), np.uint64), lead)[0] for _ in range(2)]
    kv.rotary2(x, r, pos, out, trunc=gate)
    eq([o.contiguous().reshape(-1) for o in out], [u64(w) for w in want], "truncated")
    whole = (u64(plain[0]) + u64(plain[1])).view(np.int64) >> 12
    got = (u64(out[0].contiguous()) + u64(out[1].contiguous())).view(np.int64)
    assert np.array_equal(got, whole)


# ---- append ----

APPENDS = [
    # new, lens, page, kv_heads, dim, pad, rot, interleaved
    ([1], [1], 1, 1, 2, 0, 2, False),
    ([1, 1, 1], [17, 1, 300], 16, 2, 64, 0, 64, False),
    ([5, 0, 20, 1], [5, 7, 33, 64], 8, 3, 40, 4, 16, True),
    ([9, 2], [30, 2], 4, 2, 33, 1, 32, True),      # odd head
    ([70], [130], 64, 1, 128, 0, 128, False),
    ([6], [4], 2, 2, 16, 0, 0, False),             # more new tokens than keys: the first two have no place
    ([0, 0], [3, 0], 4, 1, 8, 2, 8, False),
]


@pytest.mark.parametrize("new,lens,page,hk,D,pad,rot,neigh", APPENDS)
@pytest.mark.parametrize("given", [False, True])
def test_append(new, lens, page, hk, D, pad, rot, neigh, given):
    say("append %s %s page=%d" % (new, lens, page))
    rng = np.random.default_rng(len(new) + D)
    ck, cv = (ref.Case(rng, new, lens, page, hk, D, pad) for _ in range(2))
    cv.table[:], cv.pages = ck.table, ck.pages
    if len(lens) > 1:  # a sequence whose last page is missing, and one of no page's number
        ck.table[0, -1] = cv.table[0, -1] = -5
        ck.table[-1, 0] = cv.table[-1, 0] = ck.pages
    T = ck.tokens
    k, v, mk, mv = ([ref.words(rng, T, hk, D) for _ in range(2)] for _ in range(4))
    table = rng.integers(-4096, 4097, (40, rot // 2, 2), dtype=np.int32)
    pos = rng.integers(-3, 43, T) if given else None
    want = (ref.append(ck, k, mk, table, neigh, 7, pos) + ref.append(cv, v, mv))
    r = kv.Rotary(i32(table).reshape(40, rot // 2, 2), D, interleaved=neigh, pass_mul=7)
    pk, pv = (kv.Pool(*(dev(a) for a in c.pool)) for c in (ck, cv))
    kview = [view_of(w, 2, 2, 0)[0] for w in k]
    kv.append2(batch_of(ck), pk, kview, dev2(mk), pv, dev2(v), dev2(mv), rotary=r,
               positions=None if pos is None else i32(pos))
    for got, w in zip((pk.e,) + pk.b + (pv.e,) + pv.b, want):
        assert np.array_equal(u64(got), w)


def test_append_keys_alone_and_truncated():
    rng = np.random.default_rng(8)
    c = ref.Case(rng, [4, 3], [10, 3], 4, 2, 16)
    shape = (c.tokens, 2, 16)
    val = rng.integers(-1 << 20, 1 << 20, shape).astype(np.int64).view(np.uint64)
    s0 = ref.words(rng, *shape)
    x, m = [s0, val - s0], [ref.words(rng, *shape) for _ in range(2)]
    r = kv.Rotary.build(16, 64)
    gate = tasks.Trunc(tasks.Dealer(4), 12, val.size, STATE)
    gate.prepare()
    want = ref.append(c, x, m, r.table.cpu().numpy(), False, r.pass_mul, shift=12)
    for given in (False, True):
        pool = kv.Pool(*(dev(a) for a in c.pool))
        y = tuple(torch.zeros(shape, dtype=torch.int64, device="cuda") for _ in range(2))
        kv.append2(batch_of(c), pool, dev2(x), dev2(m), rotary=r,
                   k_trunc=(gate, y) if given else gate)
        for got, w in zip((pool.e,) + pool.b, want):
            assert np.array_equal(u64(got), w)
        if given:
            turned = kv.rotary2(dev2(x), r, i32([6, 7, 8, 9, 0, 1, 2]))
            whole = (u64(turned[0]) + u64(turned[1])).view(np.int64) >> 12
            assert np.array_equal((u64(y[0]) + u64(y[1])).view(np.int64), whole)


# ---- products ----

PRODUCTS = [
    # new, lens, page, kv_heads, group, dim, pad
    ([1], [1], 1, 1, 1, 1, 0),
    ([1], [2], 16, 1, 1, 64, 0),
    ([1], [300], 16, 12, 1, 64, 0),
    ([1, 1, 1, 1], [64, 65, 1, 513], 64, 2, 4, 128, 0),
    ([1, 0, 1], [129, 0, 63], 32, 2, 7, 40, 2),
    ([3, 12, 1], [40, 200, 90], 8, 2, 3, 80, 1),
    ([33, 1], [33, 70], 16, 2, 2, 32, 0),
    ([150], [150], 64, 1, 3, 64, 0),
    ([70, 17], [90, 300], 4, 2, 1, 96, 3),
    ([5], [3], 2, 1, 2, 16, 0),          # the first two tokens see no key
    ([2], [50], 16, 1, 17, 33, 0),       # a group above 16, an odd head
    ([20], [70], 1, 1, 1, 3, 0),
    ([4], [100], 16, 2, 2, 130, 0),
    ([9], [260], 128, 1, 8, 256, 0),
    ([1], [4500], 64, 1, 2, 64, 0),
    ([0, 0], [5, 0], 4, 1, 2, 8, 3),
]


def product_case(new, lens, page, hk, group, D, pad, kind, seed=0):
    rng = np.random.default_rng(sum(lens) + D + seed)
    c = ref.Case(rng, new, lens, page, hk, D, pad)
    H = hk * group
    off = c.causal(H)
    n = int(off[-1])
    if kind == "scores":
        x, a = ([ref.words(rng, c.tokens, H, D) for _ in range(2)] for _ in range(2))
        cc, out = ([ref.words(rng, n) for _ in range(2)] for _ in range(2))
    else:
        x, a = ([ref.words(rng, n) for _ in range(2)] for _ in range(2))
        cc, out = ([ref.words(rng, c.tokens, H, D) for _ in range(2)] for _ in range(2))
    return c, H, off, x, a, cc, out


def run_product(c, H, off, x, a, cc, out, kind, **hints):
    o = dev2(out)
    op = kv.scores2 if kind == "scores" else kv.values2
    op(batch_of(c, **hints), kv.Pool(*(dev(w) for w in c.pool)), dev2(x), dev2(a), dev2(cc),
       i32(off), o)
    return o


@pytest.mark.parametrize("kind", ["scores", "values"])
@pytest.mark.parametrize("new,lens,page,hk,group,D,pad", PRODUCTS)
def test_product(kind, new, lens, page, hk, group, D, pad):
    say("%s %s %s page=%d heads=%d x %d dim=%d" % (kind, new, lens, page, hk, group, D))
    case = product_case(new, lens, page, hk, group, D, pad, kind)
    want = getattr(ref, kind)(*case)
    eq(run_product(*case, kind), want, kind)


@pytest.mark.parametrize("kind", ["scores", "values"])
@pytest.mark.parametrize("max_new,max_keys", [(0, 0), (1, 1), (1000, 100000)])
def test_product_bounds_do_not_matter(kind, max_new, max_keys):
    case = product_case([30, 1, 7], [130, 600, 7], 16, 2, 3, 64, 2, kind)
    want = getattr(ref, kind)(*case)
    eq(run_product(*case, kind, max_new=max_new, max_keys=max_keys), want, kind)


@pytest.mark.parametrize("kind", ["scores", "values"])
def test_product_any_row_lengths(kind):
    """Rows that are not causal: empty ones, whole ones, longer than the
    sequence, and rows that do not lie within the packed elements."""
    rng = np.random.default_rng(77)
    c = ref.Case(rng, [6, 2, 40], [50, 9, 130], 8, 2, 64)
    H = 4
    rows = rng.integers(0, 140, H * c.tokens)
    rows[rng.random(rows.size) < 0.3] = 0
    off = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    n = int(off[-1])
    off[10], off[20], off[-1] = -4, n + 5, n + 1  # wrong words: those rows count as empty
    shapes = ((c.tokens, H, 64), (n,)) if kind == "scores" else ((n,), (c.tokens, H, 64))
    x, a = ([ref.words(rng, *shapes[0]) for _ in range(2)] for _ in range(2))
    cc, out = ([ref.words(rng, *shapes[1]) for _ in range(2)] for _ in range(2))
    case = (c, H, off, x, a, cc, out)
    eq(run_product(*case, kind), getattr(ref, kind)(*case), kind)


@pytest.mark.parametrize("kind", ["scores", "values"])
def test_product_bad_pages_are_zeros(kind):
    case = product_case([8, 1, 1], [100, 70, 40], 8, 2, 2, 64, 0, kind)
    c = case[0]
    c.table[0, 3], c.table[0, 12], c.table[1, 0], c.table[2, 2] = -1, c.pages, 2 ** 31 - 1, -2 ** 31
    eq(run_product(*case, kind), getattr(ref, kind)(*case), kind)
    # Lengths past the pages: those keys count as zeros too.
    c.lens = [100, 200, 40]
    eq(run_product(*case, kind), getattr(ref, kind)(*case), kind)


@pytest.mark.parametrize("kind", ["scores", "values"])
def test_product_wrong_lengths_stay_inside(kind):
    """Lengths that no pages cover, the largest and negative ones: keys without
    a page are zeros, rows of a sequence without keys are empty."""
    case = product_case([3, 1, 2, 1], [70, 300, 20, 9], 8, 2, 3, 64, 1, kind)
    c = case[0]
    c.lens = [2 ** 31 - 1, 2 ** 31 - 1, -5, -2 ** 31]
    eq(run_product(*case, kind, max_keys=300), getattr(ref, kind)(*case), kind)


@pytest.mark.parametrize("kind", ["scores", "values"])
def test_product_of_many_sequences(kind):
    """More sequences than a workgroup has threads, some without new tokens."""
    rng = np.random.default_rng(3)
    lens = [int(v) for v in rng.integers(1, 30, 700)]
    lens[::50] = [257] * 14
    new = [int(v) for v in rng.integers(0, 3, 700)]
    new = [min(n, m) for n, m in zip(new, lens)]
    case = product_case(new, lens, 16, 1, 2, 16, 2, kind)
    eq(run_product(*case, kind), getattr(ref, kind)(*case), kind)


@pytest.mark.parametrize("page,hk,group,D", [(16, 4, 5, 64), (2, 8, 4, 33), (32, 3, 4, 80),
                                             (64, 2, 8, 200)])
@pytest.mark.parametrize("max_keys", [320, 256])
def test_values_of_many_rows(page, hk, group, D, max_keys):
    """Digits formed once for all row tiles (page numbers outside the pool
    among them); 256: bounds that one of the sequences does not keep to."""
    case = product_case([130, 0, 90, 3], [300, 5, 256, 70], page, hk, group, D, 2, "values")
    c = case[0]
    c.table[0, 1], c.table[2, 0] = -1, c.pages
    say("many rows page=%d heads=%d x %d dim=%d max_keys=%d" % (page, hk, group, D, max_keys))
    eq(run_product(*case, "values", max_keys=max_keys), ref.values(*case), "values")


def sparse_rows(c, H, long):
    """Offsets with rows only for the (head, token) pairs in `long`."""
    rows = np.zeros(H * c.tokens, np.int64)
    for (h, t), n in long.items():
        rows[h * c.tokens + t] = n
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


@pytest.mark.parametrize("page", [16, 4])
@pytest.mark.parametrize("new,hk,group,dim,hint", [(130, 1, 16, 16, 9000),    # an item a workgroup
                                                   (130, 1, 16, 80, 9000),
                                                   (1, 1, 2, 16, 256),        # even shares of five
                                                   (1, 2, 2, 2, 256)])
@pytest.mark.parametrize("extreme", [False, True])
def test_values_long_sums(page, new, hk, group, dim, hint, extreme):
    """More keys than int32 digit sums hold in one workgroup; extreme: every
    digit of the opened operand and of party 0's mask share is -128."""
    L = 8400 if new > 1 else 30000
    rng = np.random.default_rng(dim + L)
    c = ref.Case(rng, [new], [L], page, hk, dim)
    H = hk * group
    off = sparse_rows(c, H, {(0, 0): L, (H - 1, new - 1): L - 1, (H // 2, new // 2): 4097})
    n = int(off[-1])
    x, a = ([ref.words(rng, n) for _ in range(2)] for _ in range(2))
    if extreme:
        low = np.uint64(0x7f7f7f7f7f7f7f80)  # sum of -128 * 256^i
        x[0][:], x[1][:], a[0][:] = low, 0, 0
        a[1][:] = 0
        c.pool[0][:], c.pool[1][:] = low, low
    cc, out = ([ref.words(rng, c.tokens, H, dim) for _ in range(2)] for _ in range(2))
    case = (c, H, off, x, a, cc, out)
    eq(run_product(*case, "values", max_keys=hint), ref.values(*case), "values")


def test_scores_extreme_digits():
    """Every digit of the operands of one party is -128, in a wide head."""
    rng = np.random.default_rng(2)
    for new, dim in ((1, 256), (40, 128)):
        c = ref.Case(rng, [new], [130], 16, 1, dim)
        off = c.causal(2)
        n = int(off[-1])
        low = np.uint64(0x7f7f7f7f7f7f7f80)
        x = [np.full((new, 2, dim), v, np.uint64) for v in (low, 0)]
        a = [np.zeros((new, 2, dim), np.uint64) for _ in range(2)]
        c.pool[0][:], c.pool[1][:] = low, low
        cc, out = ([ref.words(rng, n) for _ in range(2)] for _ in range(2))
        case = (c, 2, off, x, a, cc, out)
        eq(run_product(*case, "scores"), ref.scores(*case), "scores")


def test_long_cache_offsets_pass_32_bits():
    """A pool whose words lie past 2^32 bytes, and past 2^31 words."""
    pages, page, dim = 9000, 128, 2048 // 8
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("30 GiB of device memory wanted")
    shape = (pages, 8, page, dim)  # 2.36e9 words, 18.9 GB: e, b0, b1 share them
    e = torch.empty(shape, dtype=torch.int64, device="cuda")
    rng = np.random.default_rng(1)
    pool = kv.Pool(e, e, e)  # written once below, only read by the products
    table = np.array([[pages - 1, 3, pages - 2]], np.int32)
    c = ref.Case.__new__(ref.Case)
    c.new, c.lens, c.page, c.kv_heads, c.dim, c.width = [1], [300], page, 8, dim, 3
    c.table, c.pages, c.cu, c.tokens = table, pages, np.array([0, 1], np.int32), 1
    words = {int(pg): ref.words(rng, 8, page, dim) for pg in table[0]}
    for pg, w in words.items():
        e[pg].copy_(dev(w))

    class Pages(dict):
        def __getitem__(self, key):
            return words[int(key[0])][key[1:]]
    c.pool = [Pages()] * 3
    off = c.causal(8)
    n = int(off[-1])
    for kind, shapes in (("scores", ((1, 8, dim), (n,))), ("values", ((n,), (1, 8, dim)))):
        x, a = ([ref.words(rng, *shapes[0]) for _ in range(2)] for _ in range(2))
        cc, out = ([ref.words(rng, *shapes[1]) for _ in range(2)] for _ in range(2))
        o = dev2(out)
        op = kv.scores2 if kind == "scores" else kv.values2
        op(batch_of(c), pool, dev2(x), dev2(a), dev2(cc), i32(off), o)
        eq(o, getattr(ref, kind)(c, 8, off, x, a, cc, out), kind)
    # The append's far words: the last place of the last page, which here all
    # three arrays of the pool share, so any of its words may be left there.
    m, k = ([ref.words(rng, 1, 8, dim) for _ in range(2)] for _ in range(2))
    c.lens, c.table = [page], np.array([[pages - 1, 0, 0]], np.int32)
    kv.append2(batch_of(c), pool, dev2(k), dev2(m))
    got = u64(e[pages - 1, :, page - 1])
    assert any(np.array_equal(got, w) for w in (m[0][0], m[1][0],
                                                 k[0][0] + k[1][0] - m[0][0] - m[1][0]))
    assert np.array_equal(u64(e[pages - 1, :, page - 2]), words[pages - 1][:, page - 2])


@pytest.mark.parametrize("D", [64, 100])
@pytest.mark.parametrize("n", [(1 << 29) - 1, (1 << 29) + 77])
def test_scores_of_long_packed_arrays(D, n):
    """Rows at the end of packed arrays on both sides of 2^29 elements, where
    byte offsets pass 32 bits; every other element is left alone."""
    rng = np.random.default_rng(D)
    c = ref.Case(rng, [40], [150], 16, 1, D)
    off = c.causal(1)
    m = int(off[-1] - off[1])          # elements of the rows but the first
    far = off.astype(np.int64) + (n - m - int(off[1]))
    far[0] = 0                         # the first row's start; its rest has no keys
    x, a = ([ref.words(rng, c.tokens, 1, D) for _ in range(2)] for _ in range(2))
    cc = [ref.words(rng, int(off[-1])) for _ in range(2)]
    want = ref.scores(c, 1, off, x, a, cc, [np.zeros(int(off[-1]), np.uint64)] * 2)
    say("scores of %d packed elements, dim %d" % (n, D))
    k0 = 150                           # the first row sees all of its sequence now
    big = [torch.zeros(n, dtype=torch.int64, device="cuda") for _ in range(4)]
    for p in range(2):
        big[p][n - m:] = dev(cc[p][int(off[1]):])
    out = (big[2], big[3])
    kv.scores2(batch_of(c), kv.Pool(*(dev(w) for w in c.pool)), dev2(x), dev2(a),
               (big[0], big[1]), i32(far), out)
    for p in range(2):
        assert np.array_equal(u64(out[p][n - m:]), want[p][int(off[1]):]), "party %d" % p
        assert int(out[p][k0:n - m].count_nonzero()) == 0
    del big, out
    torch.cuda.empty_cache()


def test_scores_of_a_view():
    """Queries inside the rows of a fused product, 8-byte aligned."""
    for lead, gap in ((0, 64), (1, 0), (0, 1)):
        case = product_case([20, 1], [60, 33], 16, 2, 2, 64, 0, "scores")
        c, H, off, x, a, cc, out = case
        o = dev2(out)
        kv.scores2(batch_of(c), kv.Pool(*(dev(w) for w in c.pool)),
                   [view_of(w, lead, gap, 0)[0] for w in x], dev2(a), dev2(cc), i32(off), o)
        eq(o, ref.scores(*case), "view")


def test_pool_not_16_byte_aligned():
    for kind in ("scores", "values"):
        case = product_case([5, 1], [60, 33], 16, 2, 2, 64, 0, kind)
        c, H, off, x, a, cc, out = case
        pool = []
        for w in c.pool:
            buf = torch.empty(w.size + 1, dtype=torch.int64, device="cuda")
            v = buf[1:].view(*w.shape)
            v.copy_(dev(w))
            pool.append(v)
        o = dev2(out)
        op = kv.scores2 if kind == "scores" else kv.values2
        op(batch_of(c), kv.Pool(*pool), dev2(x), dev2(a), dev2(cc), i32(off), o)
        eq(o, getattr(ref, kind)(*case), kind)


@pytest.mark.parametrize("kind", ["scores", "values"])
@pytest.mark.parametrize("new,lens,group,D", [([1, 1], [70, 300], 4, 64), ([40], [90], 2, 33),
                                              ([1], [3000], 2, 128),
                                              ([40], [90], 2, 64), ([3, 50], [9, 150], 3, 100),
                                              ([130], [300], 8, 128)])
def test_product_truncates(kind, new, lens, group, D):
    """Through the gate: the shares of the unfused product, open and gate,
    and rows in no sequence untouched."""
    case = product_case(new, lens, 16, 2, group, D, 2, kind)
    c, H, off, x, a, cc, out = case
    plain = run_product(*case, kind)
    n = plain[0].numel()
    gate = tasks.Trunc(tasks.Dealer(6), 12, n, STATE)
    gate.prepare()
    want = tasks.pair(n)
    tasks.lin2(tasks.operand(tasks.term(tuple(v.reshape(-1) for v in plain))), n,
               into=(gate, want))
    want = [u64(w).reshape(out[0].shape).copy() for w in want]
    if kind == "values":
        for p in range(2):
            want[p][c.cu[-1]:] = out[p][c.cu[-1]:]
    o = dev2(out)
    op = kv.scores2 if kind == "scores" else kv.values2
    op(batch_of(c), kv.Pool(*(dev(w) for w in c.pool)), dev2(x), dev2(a), dev2(cc), i32(off), o,
       trunc=gate)
    eq(o, want, "truncated " + kind)


@pytest.mark.parametrize("kind", ["scores", "values"])
def test_captured_step_follows_the_lengths(kind):
    """One captured call replayed while its inputs, lengths, pages and row
    offsets change in place, beside eager work of the same shapes."""
    D, H, hk, page, width = 64, 4, 2, 16, 40
    rng = np.random.default_rng(9)
    lens_of = [[300, 20, 77], [301, 21, 78], [600, 1, 16], [17, 640, 500]]
    big = ref.Case(rng, [1, 1, 1], [640, 640, 640], page, hk, D, width=width)
    cap = 3 * 640 * H
    shapes = ((3, H, D), (cap,)) if kind == "scores" else ((cap,), (3, H, D))
    cu, lens, table = i32(big.cu), i32([1, 1, 1]), i32(big.table)
    off = i32(np.zeros(H * 3 + 1))
    x, a = (tuple(torch.zeros(shapes[0], dtype=torch.int64, device="cuda") for _ in range(2))
            for _ in range(2))
    cc, out = (tuple(torch.zeros(shapes[1], dtype=torch.int64, device="cuda") for _ in range(2))
               for _ in range(2))
    pool = kv.Pool(*(dev(w) for w in big.pool))
    batch = kv.Batch(cu, lens, table, tokens=3, max_new=1, max_keys=640)
    op = kv.scores2 if kind == "scores" else kv.values2
    work = kv.values_work(batch, pool, H)
    kw = {} if kind == "scores" else {"work": work}
    graph = tasks.capture(lambda: op(batch, pool, x, a, cc, off, out, **kw))
    for lens_now in lens_of:
        c = ref.Case.__new__(ref.Case)
        c.__dict__.update(big.__dict__)
        c.lens, c.table = lens_now, rng.permutation(big.table.ravel()).reshape(big.table.shape)
        o = c.causal(H)
        host = [[ref.words(rng, *s) for _ in range(2)] for s in (shapes[0], shapes[0], shapes[1],
                                                                 shapes[1])]
        for d, h in zip((x, a, cc, out), host):
            for p in range(2):
                d[p].copy_(dev(h[p]))
        lens.copy_(i32(lens_now))
        table.copy_(i32(c.table))
        off.copy_(i32(o))
        graph.replay()
        got = tuple(v.clone() for v in out)
        eager = dev2(host[3])
        op(batch, pool, x, a, cc, off, eager)
        want = getattr(ref, kind)(c, H, o, host[0], host[1], host[2], host[3])
        eq(got, want, "replay")
        eq(eager, want, "eager")


def test_captured_values_of_many_rows():
    """The same for prompts, whose digits pass through the workspace: a length
    may leave the captured bounds and come back."""
    D, hk, group, page = 64, 4, 5, 16
    H, rng = hk * group, np.random.default_rng(19)
    big = ref.Case(rng, [130, 60], [400, 400], page, hk, D)
    cap = H * (130 + 60) * 400
    lens, off = i32([130, 60]), i32(np.zeros(H * 190 + 1))
    mk = lambda *n: tuple(torch.zeros(n, dtype=torch.int64, device="cuda")  # noqa: E731
                          for _ in range(2))
    x, a, cc, out = mk(cap), mk(cap), mk(190, H, D), mk(190, H, D)
    pool = kv.Pool(*(dev(w) for w in big.pool))
    batch = kv.Batch(i32(big.cu), lens, i32(big.table), tokens=190, max_new=130, max_keys=300)
    work = kv.values_work(batch, pool, H)
    graph = tasks.capture(lambda: kv.values2(batch, pool, x, a, cc, off, out, work=work))
    for lens_now in ([300, 130], [140, 400], [299, 61]):
        c = ref.Case.__new__(ref.Case)
        c.__dict__.update(big.__dict__)
        c.lens = lens_now
        o = c.causal(H)
        host = [[ref.words(rng, *s) for _ in range(2)] for s in ((cap,), (cap,), (190, H, D))]
        for d, h in zip((x, a, cc), host):
            for p in range(2):
                d[p].copy_(dev(h[p]))
        lens.copy_(i32(lens_now))
        off.copy_(i32(o))
        graph.replay()
        got = tuple(v.clone() for v in out)
        eager = mk(190, H, D)
        kv.values2(batch, pool, x, a, cc, off, eager)
        want = ref.values(c, H, o, *host, [np.zeros((190, H, D), np.uint64)] * 2)
        eq(got, want, "replay")
        eq(eager, want, "eager")


def test_two_streams_at_once():
    cases = [product_case([1, 1], [500 + s, 900], 16, 2, 4, 64, 0, "values", seed=s)
             for s in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    inputs = [(batch_of(c[0]), kv.Pool(*(dev(w) for w in c[0].pool)), dev2(c[3]), dev2(c[4]),
               dev2(c[5]), i32(c[2]), dev2(c[6])) for c in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, i in zip(streams, inputs):
            with torch.cuda.stream(s):
                kv.values2(*i)
    torch.cuda.synchronize()
    for c, i in zip(cases, inputs):
        eq(i[-1], ref.values(*c), "stream")
