"""Attention over a paged cache of keys and values for two parties on one GPU:
packed sequences of different lengths, grouped heads, rotary positions.

Operators (each one call of libsuf_hip.so, both parties, exact mod 2^64):
  rotary2   rotary positions on shares (sufhip_rotary2)
  append2   keys, rotated on the way, and values into the cache's pages
            (sufhip_kv_append2)
  scores2   queries times cached keys, ragged rows (sufhip_kv_scores2)
  values2   ragged rows of probabilities times cached values
            (sufhip_kv_values2)

A cached word is opened once, when it is appended: the pages hold the public
E = value - b and each party's share of the mask b, which is used for nothing
else.  A product then needs a fresh mask A of its left operand alone and the
dealer's C = A b:
  Z_p = C_p + D b_p + (A_p + [p = 0] D) E,   D = open(left - A)

On top of them:
  PagedCache       the pages of many sequences and the dealer's masks
  CachedAttention  one step (prompts or single tokens) of causal attention:
                   rotation, append, scores, softmax, values, each product
                   and rotation with its truncation gate (over long rows the
                   softmax's division after the values: softmax.LongRows)

The reference keeps a cache of shares (include/nn/kv_cache.hpp) and multiplies
it by a fresh triple for every new token; its attention is
src/nn/attention_block.cpp:931-1900.
"""
import ctypes
import itertools
import math
import warnings

import numpy as np
import torch

from . import native, tables
from .softmax import LONG_KEYS, LongRows, SoftmaxBlock
from .tasks import TABLE_BITS, Dealer, Trunc, dev, dev_i32, prepare_batch

M64 = (1 << 64) - 1
I32 = (1 << 31) - 1       # the library counts tokens, heads and pages in 32 bits
MAX_PACKED = (1 << 31) - 256


# ---- arguments ----

def _fail(what, msg):
    raise ValueError("%s: %s" % (what, msg))


def _refuse(t, shape, d, what, name, dtype, dense):
    """Says what is wrong with a tensor that _ptr did not take."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or tuple(t.shape) != tuple(shape):
        _fail(what, "%s must be a %s tensor of shape %s" % (name, dtype, list(shape)))
    if not t.is_cuda or t.get_device() != d:
        _fail(what, "%s must be on the GPU, on one device with the other tensors" % name)
    if dense and not t.is_contiguous():
        _fail(what, "%s must be contiguous" % name)
    _fail(what, "%s is not usable" % name)


def _refuse_pair(pair, shape, d, what, name, dense):
    if not isinstance(pair, (tuple, list)) or len(pair) != 2:
        _fail(what, "%s must be a pair (party 0, party 1)" % name)
    for t in pair:
        if not (isinstance(t, torch.Tensor) and t.dtype is torch.int64 and t.shape == shape and
                t.get_device() == d and (not dense or t.is_contiguous())):
            _refuse(t, shape, d, what, name, torch.int64, dense)
    _fail(what, "%s is not usable" % name)


# A step makes many calls of a few microseconds each, so a pair of tensors is
# checked in one expression; the functions above find the reason.

_I64 = torch.int64


def _ptr(t, shape, d, what, name, dtype=_I64):
    """Address of a contiguous tensor on GPU d (>= 0)."""
    try:
        if t.dtype is dtype and t.shape == shape and t.get_device() == d and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    _refuse(t, shape, d, what, name, dtype, True)


def _ptr2(arr, pair, shape, d, what, name):
    """Both parties' contiguous tensors into a void*[2]."""
    try:
        t0, t1 = pair
        if t0.dtype is _I64 and t1.dtype is _I64 and t0.shape == shape and t1.shape == shape and \
                t0.get_device() == d and t1.get_device() == d and t0.is_contiguous() and \
                t1.is_contiguous():
            arr[0], arr[1] = t0.data_ptr(), t1.data_ptr()
            return
    except (AttributeError, TypeError, ValueError):
        pass
    _refuse_pair(pair, shape, d, what, name, True)


def _rows(arr, pair, shape, d, what, name, written=False):
    """Both parties' [tokens, heads, dim] tensors into a void*[2]; their token
    and head stride."""
    try:
        t0, t1 = pair
        ok = t0.dtype is _I64 and t1.dtype is _I64 and t0.shape == shape and t1.shape == shape and \
            t0.get_device() == d and t1.get_device() == d
    except (AttributeError, TypeError, ValueError):
        ok = False
    if not ok:
        _refuse_pair(pair, shape, d, what, name, False)
    st = t0.stride()
    if st != t1.stride():
        # A stride along an axis of one says nothing.
        other = t1.stride()
        if shape[2] > 1 and other[2] != 1:
            _fail(what, "the values of a head of %s must be neighbours" % name)
        if t0.numel() and ((st[0] != other[0] and shape[0] > 1) or
                           (st[1] != other[1] and shape[1] > 1)):
            _fail(what, "both parties' %s must have the same strides" % name)
    if st[2] != 1 and shape[2] > 1:
        _fail(what, "the values of a head of %s must be neighbours" % name)
    if written and ((st[0] == 0 and shape[0] > 1) or (st[1] == 0 and shape[1] > 1)):
        _fail(what, "rows of %s must not overlap" % name)
    arr[0], arr[1] = t0.data_ptr(), t1.data_ptr()
    return st[0], st[1]


def _device(t, what, name):
    """Index of the GPU a call's first tensor is on."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _fail(what, "%s must be a tensor on the GPU" % name)
    return t.get_device()


_entries = {}


def _call(name, args, d):
    """One library call on GPU d's current stream."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(native.load(), name)
    if torch._C._cuda_getDevice() == d:
        rc = fn(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(d))
    else:
        with torch.cuda.device(d):
            rc = fn(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(d))
    if rc != native.OK:
        native.check(rc, name)


def _epilogue(args, trunc, out, n, d, what):
    """trunc: a prepared tasks.Trunc whose outputs go to `out`."""
    if trunc is None:
        return None
    if not trunc.has_table():
        _fail(what, "the truncation must be a GapARS gate of at most 14 bits")
    if trunc.n < n:
        _fail(what, "the truncation is for %d elements, not %d" % (trunc.n, n))
    if trunc.work[0].get_device() != d:
        _fail(what, "the truncation is on another device")
    epi = trunc.epilogue(out)
    args.trunc = ctypes.pointer(epi)
    return epi


class Rotary:
    """A public rotary table: int32 [positions, rot / 2, 2] fixed-point (cos,
    sin) on the GPU, for heads of `dim` values.  interleaved pairs neighbours
    (2i, 2i + 1), otherwise pair i is (i, rot / 2 + i).  pass_mul, the table's
    1, multiplies the values past the rotated part."""

    def __init__(self, table, dim, interleaved=False, pass_mul=1 << 12):
        _device(table, "Rotary", "the table")
        if table.dim() != 3 or table.shape[2] != 2 or 2 * table.shape[1] > dim:
            _fail("Rotary", "the table must be [positions, rot / 2, 2] with rot <= dim")
        _ptr(table, table.shape, _device(table, "Rotary", "the table"), "Rotary", "the table",
             torch.int32)
        self.table, self.dim, self.interleaved = table, int(dim), bool(interleaved)
        self.pass_mul, self.device = int(pass_mul), table.get_device()
        # A table of no elements has no address, and no address is no rotation.
        self._held = table if table.numel() else torch.zeros(2, dtype=torch.int32,
                                                             device=table.device)
        r = self.arg = native.RotaryTable()
        r.d_table = self._held.data_ptr()
        r.positions, r.rot = table.shape[0], 2 * table.shape[1]
        r.interleaved, r.pass_mul = int(self.interleaved), self.pass_mul

    @classmethod
    def build(cls, dim, positions, rot=None, base=10000.0, frac_bits=12, scale=1.0,
              interleaved=False, scaling=None, device="cuda"):
        """Table of Q(frac_bits) factors scale * cos, scale * sin of
        position * base^(-2 i / rot), the angles in float64.  scale: a public
        factor of every value (a query's 1 / sqrt(dim)).  scaling stretches
        the positions for contexts longer than trained ones:
          ("linear", s)     position / s
          ("base", s)       base * s^(rot / (rot - 2)): slow pairs are
                            stretched by s, the fastest not at all
          ("parts", s, n, slow, fast)   pairs that turn at most `slow` times in
                            the n trained positions are stretched by s, those
                            that turn at least `fast` times not, the others in
                            between; the table is scaled by 0.1 ln(s) + 1, its
                            1 for the values past the rotated part too"""
        rot = dim if rot is None else rot
        table, one = rotary_table(positions, rot, base, frac_bits, scale, scaling)
        return cls(torch.from_numpy(table).to(device), dim, interleaved, one)


def rotary_table(positions, rot, base=10000.0, frac_bits=12, scale=1.0, scaling=None):
    """(int32 [positions, rot / 2, 2], the table's 1): Rotary.build's factors."""
    if rot < 0 or rot % 2 or positions < 0 or not 0 < frac_bits <= 28:
        _fail("rotary_table", "rot must be even, positions >= 0 and frac_bits in [1, 28]")
    if not 0 < base < math.inf:
        _fail("rotary_table", "base must be a positive number")
    i = np.arange(rot // 2, dtype=np.float64)
    freq = float(base) ** (-2.0 * i / max(rot, 1))
    if scaling is not None:
        if len(scaling) != (5 if scaling and scaling[0] == "parts" else 2):
            _fail("rotary_table", "scaling must be (kind, s) or (\"parts\", s, n, slow, fast)")
        kind, s = scaling[0], float(scaling[1])
        if not 1 <= s < math.inf:
            _fail("rotary_table", "positions are stretched by a factor of at least 1")
        if kind == "linear":
            freq = freq / s
        elif kind == "base":
            if rot > 2:
                freq = (float(base) * s ** (rot / (rot - 2.0))) ** (-2.0 * i / rot)
        elif kind == "parts":
            trained, slow, fast = (float(v) for v in scaling[2:])
            if not (0 <= slow < fast < math.inf and 0 < trained < math.inf):
                _fail("rotary_table", "parts need positions trained and 0 <= slow < fast")
            turns = trained * freq / (2.0 * math.pi)
            keep = np.clip((turns - slow) / (fast - slow), 0.0, 1.0)
            freq = freq * keep + freq / s * (1.0 - keep)
            scale = scale * (0.1 * math.log(s) + 1.0)
        else:
            _fail("rotary_table", "unknown scaling %r" % (kind,))
    one = scale * (1 << frac_bits)
    if not abs(one) < (1 << 31) - 0.5:  # or it rounds past a word
        _fail("rotary_table", "scale * 2^frac_bits must stay below 2^31")
    ang = np.arange(positions, dtype=np.float64)[:, None] * freq
    table = np.rint(np.stack([np.cos(ang), np.sin(ang)], -1) * one).astype(np.int32)
    return table, int(round(one))


class Pool:
    """The pages of keys or of values: e, b0, b1 int64 [pages, kv_heads,
    page_tokens, dim] on the GPU (the open value - b, both parties' shares of
    b); page_tokens a power of two."""

    __slots__ = ("arg", "e", "b", "device", "shape", "kv_heads", "dim")

    def __init__(self, e, b0, b1):
        d, shape = _device(e, "Pool", "e"), e.shape
        if len(shape) != 4:
            _fail("Pool", "the arrays must be [pages, kv_heads, page_tokens, dim]")
        p = self.arg = native.KvPool()
        p.e = _ptr(e, shape, d, "Pool", "e")
        _ptr2(p.b, (b0, b1), shape, d, "Pool", "b")
        if max(shape) > I32:
            _fail("Pool", "at most 2^31 - 1 pages")
        p.pages, self.kv_heads, p.page_tokens, self.dim = shape
        p.kv_heads, p.dim = self.kv_heads, self.dim
        self.e, self.b, self.device, self.shape = e, (b0, b1), d, shape


class Batch:
    """The packed new tokens of some sequences and their pages: cu int32
    [seqs + 1] (first token of each sequence, the end last), kv_lens int32
    [seqs] (keys, the new ones included), pages int32 [seqs, max_pages] (pool
    page of each page_tokens keys, -1: none), all on the GPU.  tokens: rows of
    every token array; those from cu[-1] on are padding and are left alone.
    max_new, max_keys: bounds by which launches are laid out."""

    def __init__(self, cu, kv_lens, pages, tokens, max_new, max_keys):
        d = _device(kv_lens, "Batch", "kv_lens")
        if kv_lens.dim() != 1 or pages.dim() != 2:
            _fail("Batch", "kv_lens must be [seqs], pages [seqs, max_pages]")
        if not (0 <= tokens <= I32 and 0 <= max_new <= I32 and 0 <= max_keys <= I32):
            _fail("Batch", "tokens, max_new and max_keys must be in [0, 2^31)")
        seqs, width = kv_lens.shape[0], pages.shape[1]
        b = self.arg = native.KvBatch()
        b.d_cu_tokens = _ptr(cu, (seqs + 1,), d, "Batch", "cu", torch.int32)
        b.d_kv_lens = _ptr(kv_lens, (seqs,), d, "Batch", "kv_lens", torch.int32)
        b.d_pages = _ptr(pages, (seqs, width), d, "Batch", "pages", torch.int32)
        b.seqs, b.tokens, b.max_pages = seqs, int(tokens), width
        b.max_new, b.max_keys = int(max_new), int(max_keys)
        self.cu, self.kv_lens, self.pages = cu, kv_lens, pages
        self.tokens, self.device = int(tokens), d
        self._work_bytes = {}


def causal_row_offsets(new, lens, heads):
    """Host int64 [heads * tokens + 1]: packed rows of causal attention for
    sequences of new[s] new tokens at the end of lens[s] keys; row (h, t) is
    h * tokens + t and holds the keys up to the token's own."""
    rows = [np.arange(L - n + 1, L + 1) for n, L in zip(new, lens)]
    rows = np.concatenate(rows) if rows else np.zeros(0)
    return np.concatenate([[0], np.cumsum(np.tile(np.maximum(rows, 0), heads))]).astype(np.int64)


# ---- operators ----

def rotary2(x, rotary, positions, out=None, trunc=None):
    """Rotates both parties' shares x (pair of int64 [tokens, heads, dim], any
    token and head strides) by the tokens' positions (int32 [tokens]; a token
    outside the table is padding and its rows of out stay).  out: a pair like
    x, which may be x itself, or None for new ones (zeros in padding rows);
    its rows overlap no others of x and none of each other.
    trunc: a prepared tasks.Trunc the rotated values go through.  Returns
    out."""
    what = "rotary2"
    d, shape = _device(x[0], what, "x"), x[0].shape
    if len(shape) != 3 or shape[2] != rotary.dim:
        _fail(what, "x must be [tokens, heads, %d]" % rotary.dim)
    if shape[0] > I32 or shape[1] > I32:
        _fail(what, "at most 2^31 - 1 tokens and heads")
    if rotary.device != d:
        _fail(what, "the table is on another device than x")
    if out is None:
        out = tuple(torch.zeros(shape, dtype=torch.int64, device=x[0].device) for _ in range(2))
    a = native.Rotary2Args()
    r = a.x
    r.token_stride, r.head_stride = _rows(r.p, x, shape, d, what, "x")
    a.tokens, a.heads, a.dim = shape
    a.rot = rotary.arg
    a.d_positions = _ptr(positions, shape[:1], d, what, "positions", torch.int32)
    a.out_token_stride, a.out_head_stride = _rows(a.out, out, shape, d, what, "out", written=True)
    if trunc is not None:
        epi = _epilogue(a, trunc, out, x[0].numel(), d, what)
        a.mask = trunc.mask & M64
    _call("sufhip_rotary2", a, d)
    return out


def _append_part(part, batch, pool, x, mask, rotary, positions, trunc, what, name):
    T, d = batch.tokens, batch.device
    shape = (T, pool.kv_heads, pool.dim)
    if pool.device != d:
        _fail(what, "the pool and the batch are on different devices")
    r = part.x
    r.token_stride, r.head_stride = _rows(r.p, x, shape, d, what, name)
    _ptr2(part.mask, mask, shape, d, what, name + "_mask")
    part.pool = pool.arg
    if rotary is not None:
        if rotary.dim != pool.dim or rotary.device != d:
            _fail(what, "the rotary table must be for heads of %d, on the pool's device" % pool.dim)
        part.rot = rotary.arg
        if positions is not None:
            part.d_positions = _ptr(positions, (T,), d, what, "positions", torch.int32)
    if trunc is None:
        return None
    gate, y = trunc if isinstance(trunc, tuple) else (trunc, None)
    if y is not None:
        for t in y:
            _ptr(t, shape, d, what, "the truncated shares")
    epi = _epilogue(part, gate, y if y is not None else x, x[0].numel(), d, what)
    if y is None:
        epi.y[0] = epi.y[1] = None
        part.trunc = ctypes.pointer(epi)
    part.trunc_mask = gate.mask & M64
    return epi


def append2(batch, k_pool, k, k_mask, v_pool=None, v=None, v_mask=None, rotary=None,
            positions=None, k_trunc=None, v_trunc=None):
    """Appends the batch's new tokens to their pages: k (pair of int64
    [tokens, kv_heads, dim], any token and head strides), rotated by `rotary`
    if given (by the keys' places in their sequences, or by `positions`), and
    v if given.  k_mask, v_mask: pairs of the dealer's mask shares, contiguous
    [tokens, kv_heads, dim].  k_trunc, v_trunc: a prepared tasks.Trunc the rows
    go through before they are opened, or (Trunc, pair for the truncated
    shares).  The two pools share no memory."""
    what = "append2"
    if v_pool is None and not (v is None and v_mask is None and v_trunc is None):
        _fail(what, "v, v_mask and v_trunc need v_pool")
    if rotary is None and positions is not None:
        _fail(what, "positions need rotary")
    a = native.KvAppend2Args()
    a.batch = batch.arg
    keep = [_append_part(a.part[0], batch, k_pool, k, k_mask, rotary, positions, k_trunc, what,
                         "k")]
    if v_pool is not None:
        keep.append(_append_part(a.part[1], batch, v_pool, v, v_mask, None, None, v_trunc, what,
                                 "v"))
    _call("sufhip_kv_append2", a, batch.device)


def _product(batch, pool, offsets, heads, what):
    a = native.KvProduct2Args()
    if heads > I32:
        _fail(what, "at most 2^31 - 1 heads")
    a.batch, a.pool, a.heads = batch.arg, pool.arg, heads
    if pool.device != batch.device:
        _fail(what, "the pool and the batch are on different devices")
    a.d_row_offsets = _ptr(offsets, (heads * batch.tokens + 1,), batch.device, what, "offsets",
                           torch.int32)
    return a


def scores2(batch, pool, q, a, c, offsets, out, trunc=None):
    """Scores of the batch's new tokens against the cached keys: q (pair of
    int64 [tokens, heads, dim], any token and head strides), a (the dealer's
    mask shares of q, contiguous), c and out (pairs of packed int64 [n]: the
    shares of a's product with the keys' masks; the scores).  offsets: int32
    [heads * tokens + 1], row (h, t) first element h * tokens + t.  trunc: a
    prepared tasks.Trunc the scores go through.  Returns out."""
    what, d = "scores2", batch.device
    _device(q[0], what, "q")
    shape = q[0].shape
    if len(shape) != 3 or shape[0] != batch.tokens or shape[2] != pool.dim:
        _fail(what, "q must be [%d, heads, %d]" % (batch.tokens, pool.dim))
    g = _product(batch, pool, offsets, shape[1], what)
    r = g.x
    r.token_stride, r.head_stride = _rows(r.p, q, shape, d, what, "q")
    _ptr2(g.a, a, shape, d, what, "a")
    _device(out[0], what, "out")
    n = g.n = out[0].numel()
    _ptr2(g.c, c, (n,), d, what, "c")
    _ptr2(g.out, out, (n,), d, what, "out")
    if trunc is not None:
        epi = _epilogue(g, trunc, out, n, d, what)
        g.mask = trunc.mask & M64
    _call("sufhip_kv_scores2", g, d)
    return out


def _work_words(batch, pool, heads):
    key = (pool.shape, heads)
    n = batch._work_bytes.get(key)
    if n is None:
        with torch.cuda.device(batch.device):
            nb = native.load().sufhip_kv_values2_work_bytes(ctypes.byref(batch.arg),
                                                            ctypes.byref(pool.arg), heads)
        n = batch._work_bytes[key] = (nb + 7) // 8
    return n


def values_work(batch, pool, heads):
    """The workspace of a values2 call on this batch (None: none needed)."""
    n = _work_words(batch, pool, heads)
    return torch.empty(n, dtype=torch.int64, device=batch.kv_lens.device) if n else None


def values2(batch, pool, p, a, c, offsets, out, trunc=None, work=None):
    """Rows of probabilities times the cached values: p, a (pairs of packed
    int64 [n]; the dealer's mask shares of p), c and out (pairs of contiguous
    int64 [tokens, heads, dim]: the shares of a's product with the values'
    masks; the weighted values, heads side by side).  offsets as in scores2.
    work: values_work(...) of a batch and a pool with the same extents,
    allocated here if it is not given.  Returns out."""
    what, d = "values2", batch.device
    _device(out[0], what, "out")
    shape = out[0].shape
    if len(shape) != 3 or shape[0] != batch.tokens or shape[2] != pool.dim:
        _fail(what, "out must be [%d, heads, %d]" % (batch.tokens, pool.dim))
    g = _product(batch, pool, offsets, shape[1], what)
    _device(p[0], what, "p")
    n = g.n = p[0].numel()
    _ptr2(g.x.p, p, (n,), d, what, "p")
    _ptr2(g.a, a, (n,), d, what, "a")
    _ptr2(g.c, c, shape, d, what, "c")
    _ptr2(g.out, out, shape, d, what, "out")
    if trunc is not None:
        epi = _epilogue(g, trunc, out, out[0].numel(), d, what)
        g.mask = trunc.mask & M64
    if work is None:
        work = values_work(batch, pool, shape[1])
    if work is not None:
        g.d_work = _ptr(work, work.shape, d, what, "work")
        g.work_bytes = work.numel() * 8
    _call("sufhip_kv_values2", g, d)
    return out


# ---- a cache of many sequences, and a step of attention over it ----

class PagedCache:
    """Pages of keys and values for many sequences of any lengths.  open()
    starts a sequence, extend() gives its new tokens pages, close() takes its
    pages back; k and v are the Pools.  A page that is used again gets new
    masks with its new tokens."""

    def __init__(self, pages, page_tokens, kv_heads, dim, v_dim=None, device="cuda"):
        if not (pages >= 0 and kv_heads >= 1 and page_tokens >= 1 and
                page_tokens & (page_tokens - 1) == 0 and 1 <= dim <= native.KV_MAX_DIM and
                (v_dim is None or 1 <= v_dim <= native.KV_MAX_DIM)):
            _fail("PagedCache", "pages >= 0, kv_heads >= 1, page_tokens a power of two and heads "
                                "of 1 to %d values" % native.KV_MAX_DIM)
        shape = (pages, kv_heads, page_tokens)
        self.k, self.v = (
            Pool(*(torch.zeros(shape + (n,), dtype=torch.int64, device=device)
                   for _ in range(3))) for n in (dim, dim if v_dim is None else v_dim))
        self.page_tokens, self.kv_heads, self.device = page_tokens, kv_heads, device
        self.free = list(range(pages))[::-1]
        self.seqs = {}
        self._next = 0

    def open(self):
        """A new, empty sequence's number."""
        s, self._next = self._next, self._next + 1
        self.seqs[s] = {"pages": [], "length": 0, "dealt": 0, "run": 0}
        return s

    def close(self, seq):
        """Takes the sequence's pages back.  A step of it that was dealt and
        has not run does not run any more, nor does a later one of another
        sequence in that step, whose keys would miss: close that one too."""
        self.free += self.seqs.pop(seq)["pages"][::-1]

    def length(self, seq):
        return self.seqs[seq]["length"]

    def extend(self, seqs, new):
        """Room for new[i] more tokens of sequence seqs[i]; the Batch of these
        tokens.  What it raises (the pages do not suffice, the device's memory
        does not), it raises with nothing changed."""
        if len(seqs) != len(new) or len(set(seqs)) != len(seqs) or min(new, default=1) < 0:
            _fail("extend", "sequences must be different, each with a count of new tokens >= 0")
        state = [self.seqs[s] for s in seqs]
        lens = [st["length"] + n for st, n in zip(state, new)]
        need = [-(-n // self.page_tokens) - len(st["pages"]) for n, st in zip(lens, state)]
        if sum(need) > len(self.free):
            raise RuntimeError("PagedCache: %d pages wanted, %d free" % (sum(need), len(self.free)))
        # The last free pages first, as many as each sequence needs.
        ends = len(self.free) - np.concatenate([[0], np.cumsum(need, dtype=np.int64)])
        pages = [st["pages"] + self.free[e:b][::-1] for st, b, e in zip(state, ends, ends[1:])]
        width = max([len(p) for p in pages] + [1])
        table = np.full((len(seqs), width), -1, np.int32)
        for row, p in zip(table, pages):
            row[:len(p)] = p
        cu = np.concatenate([[0], np.cumsum(np.asarray(new, dtype=np.int64))])
        batch = Batch(dev_i32(cu, self.device), dev_i32(np.asarray(lens), self.device),
                      dev_i32(table, self.device), tokens=int(cu[-1]), max_new=max(new, default=0),
                      max_keys=max(lens, default=0))
        for st, n, p in zip(state, lens, pages):
            st["pages"], st["length"] = p, n
        del self.free[ends[-1]:]
        return batch

    def _shrink(self, seqs, lens):
        """Takes back what the last extend() gave: seqs[i] has lens[i] tokens
        again, the pages past them are free."""
        for s, n in reversed(list(zip(seqs, lens))):
            st = self.seqs[s]
            keep = -(-n // self.page_tokens)
            self.free += st["pages"][keep:][::-1]
            st["pages"], st["length"] = st["pages"][:keep], n


def _shares(dealer, shape, device):
    """Uniform shares of a uniform value (a mask), both parties."""
    n = int(np.prod(shape))
    return tuple(dev(dealer.words(n), device).view(shape) for _ in range(2))


_seeds = itertools.count(21)


class CachedAttention:
    """Causal attention of new tokens over a PagedCache, grouped heads, with
    rotary positions; Q(frac_bits) shares in and out:
      q', k' = trunc(rot(q) / sqrt(dim)), trunc(rot(k))
      scores = trunc(q' k'^T), p = Softmax(scores), out = trunc(p v)
    The queries' 1 / sqrt(dim) is part of their rotary table, so q' holds
    frac_bits bits of the scaled query: each of its values is off by up to
    2^-frac_bits and 2^-table_bits of the query's pair.

    Softmax: steps of 2^-frac_bits in probabilities and reciprocals
    (SoftmaxBlock) while an equal share of max_positions keys is at least six
    of them; a row of n keys so loses up to about 2 n 2^-frac_bits of its
    weight when its scores are close to each other (5 % at 100 keys, 29 % at
    600, frac_bits 12), and long_rows asks for the other form there.  Beyond,
    and wherever long_rows is given, weights of 24 bits are divided after the product
    with the values (LongRows): off by less than 0.1 % up to 8192 keys, 1.3 %
    at LONG_KEYS; the values have to stay below 2^(38 - frac_bits) over the
    keys in size.
    deal(seqs, new) makes a step's dealer material and room in the cache,
    step.run(q, k, v, out) computes it.

    seed: of the dealer's words, another one for each object unless given (two
    with one seed, a model's layers say, would open their keys under the same
    masks)."""

    def __init__(self, cache, heads, prg_state, max_positions, frac_bits=12, table_bits=12,
                 rot=None, base=10000.0, interleaved=False, scaling=None, seed=None,
                 long_rows=None):
        dim = cache.k.dim
        if heads % cache.kv_heads:
            _fail("CachedAttention", "heads must be a multiple of the cache's %d" % cache.kv_heads)
        if not (0 < frac_bits <= TABLE_BITS and 0 < table_bits <= TABLE_BITS):
            _fail("CachedAttention", "frac_bits and table_bits must be in [1, %d]" % TABLE_BITS)
        # The block's gates have tables of up to 13 bits.
        short = 6 * max_positions <= 1 << frac_bits and frac_bits < TABLE_BITS
        self.long_rows = not short if long_rows is None else bool(long_rows)
        if not self.long_rows and not short:
            _fail("CachedAttention", "max_positions needs long_rows")
        if max_positions > LONG_KEYS:
            _fail("CachedAttention", "at most %d positions" % LONG_KEYS)
        self.cache, self.heads, self.f, self.fc = cache, heads, frac_bits, table_bits
        self.prg_state = bytes(prg_state)
        self.max_positions = max_positions
        kw = dict(rot=rot, base=base, frac_bits=table_bits, interleaved=interleaved,
                  scaling=scaling, device=cache.device)
        self.q_rotary = Rotary.build(dim, max_positions, scale=1.0 / math.sqrt(dim), **kw)
        self.k_rotary = Rotary.build(dim, max_positions, **kw)
        # Of rows that the block takes, a reciprocal that holds at every sum.
        self.recip_table = None if self.long_rows else tables.recip_wide_table(
            frac_bits, 2.0 ** max(10, int(max_positions).bit_length()))
        self.dealer = Dealer(next(_seeds) if seed is None else seed)

    def deal(self, seqs, new):
        """A step of new[i] tokens of sequence seqs[i].  Its material takes
        about 340 bytes of host memory a score while it is drawn, 260 of the
        device's while the step lives.  What deal raises, it raises with the
        cache as it was."""
        if min(new, default=0) < 1:
            _fail("CachedAttention.deal", "every sequence needs a new token")
        if max(self.cache.length(s) + n for s, n in zip(seqs, new)) > self.max_positions:
            _fail("CachedAttention.deal", "a sequence grows past max_positions")
        keys = sum(n * self.cache.length(s) + n * (n + 1) // 2 for s, n in zip(seqs, new))
        if self.heads * keys > MAX_PACKED:
            _fail("CachedAttention.deal", "more than 2^31 - 256 scores in one step")
        before = [self.cache.length(s) for s in seqs]
        batch = self.cache.extend(seqs, new)
        try:
            with torch.cuda.device(self.cache.device):
                step = AttentionStep(self, batch, seqs, new)
        except BaseException:  # out of memory, an interrupt: no tokens without a step
            self.cache._shrink(seqs, before)
            raise
        for _, st, _ in step.turns:
            st["dealt"] += 1
        return step


class AttentionStep:
    """One step's tokens: its Batch, the dealer's masks, products and gates.
    For one use, in the order in which the steps of a sequence were dealt."""

    def __init__(self, att, batch, seqs, new):
        cache, deal, H, f = att.cache, att.dealer, att.heads, att.f
        device, Hk = cache.device, cache.kv_heads
        self.att = att
        self.batch = b = batch
        # Which step of each of its sequences this is.
        self.turns = [(s, cache.seqs[s], cache.seqs[s]["dealt"]) for s in seqs]
        lens = [cache.length(s) for s in seqs]
        T, D, Dv = b.tokens, cache.k.dim, cache.v.dim
        self.offsets = causal_row_offsets(new, lens, H)
        self.off = dev_i32(self.offsets, device)
        n = int(self.offsets[-1])
        self.positions = dev_i32(np.concatenate([np.arange(L - k, L)
                                                 for k, L in zip(new, lens)]), device)
        self.work = values_work(b, cache.v, H)
        # The new words' masks go to their pages at once, so that the products
        # below see all masks: appended as the values too, they leave E = 0
        # there, which says nothing of them.
        self.k_mask = _shares(deal, (T, Hk, D), device)
        self.v_mask = _shares(deal, (T, Hk, Dv), device)
        append2(b, cache.k, self.k_mask, self.k_mask, cache.v, self.v_mask, self.v_mask)
        self.q_a, self.p_a = _shares(deal, (T, H, D), device), _shares(deal, (n,), device)
        self.s_c = self._triple(scores2, cache.k, self.q_a, (n,), deal, {})
        self.o_c = self._triple(values2, cache.v, self.p_a, (T, H, Dv), deal, {"work": self.work})
        self.tr = {name: Trunc(deal, bits, size, att.prg_state, device=device)
                   for name, bits, size in (("q", att.fc, T * H * D), ("k", att.fc, T * Hk * D),
                                            ("s", f, n),
                                            ("o", LongRows.z_bits() if att.long_rows else f,
                                             T * H * Dv))}
        seed = deal.word() >> 1
        if att.long_rows:
            row = np.arange(H) * T + np.arange(T)[:, None]  # of out's [tokens, heads]
            self.softmax = LongRows(self.offsets, att.prg_state, f, np.repeat(row.ravel(), Dv),
                                    seed=seed, device=device)
            self.z = tuple(torch.empty((T, H, Dv), dtype=torch.int64, device=device)
                           for _ in range(2))
        else:
            self.softmax = SoftmaxBlock(self.offsets, att.prg_state, f, seed=seed,
                                        recip=att.recip_table, device=device)
        self.q = tuple(torch.empty((T, H, D), dtype=torch.int64, device=device) for _ in range(2))
        self.s, self.p = (tuple(torch.empty(n, dtype=torch.int64, device=device)
                                for _ in range(2)) for _ in range(2))

    def _triple(self, op, pool, a, shape, deal, kw):
        """Shares of A b for the product's left mask A: the product itself with
        b_1 in E's place, A opened and nothing else: Z_0 = A b_0 + A b_1."""
        zero = tuple(torch.zeros_like(a[0]) for _ in range(2))
        out = tuple(torch.zeros(shape, dtype=torch.int64, device=a[0].device) for _ in range(2))
        op(self.batch, Pool(pool.b[1], pool.b[0], pool.b[0]), (a[0] + a[1], zero[1]), zero,
           tuple(torch.zeros_like(v) for v in out), self.off, out, **kw)
        c0 = dev(deal.words(out[0].numel()), out[0].device).view(shape)
        return c0, out[0] - c0

    def truncs(self):
        return list(self.tr.values())

    def _take_turn(self):
        """Refuses a step whose keys would land in pages that are not its
        sequences' any more, beside keys that are not there yet, or under keys
        that a later step has used."""
        again = False
        for s, st, k in self.turns:
            if self.att.cache.seqs.get(s) is not st:
                raise RuntimeError("AttentionStep.run: sequence %d has been closed" % s)
            if st["run"] < k:
                raise RuntimeError("AttentionStep.run: an earlier step of sequence %d has not run"
                                   % s)
            if st["run"] > k + 1:
                raise RuntimeError("AttentionStep.run: a later step of sequence %d has run" % s)
            again = again or st["run"] > k
        if again:
            warnings.warn("AttentionStep.run: a step is for one use; a second one opens other "
                          "values under the same masks, whose difference is then public",
                          RuntimeWarning, stacklevel=3)
        for _, st, k in self.turns:
            st["run"] = k + 1

    def run(self, q, k, v, out):
        """q [tokens, heads, dim], k, v [tokens, kv_heads, dim]: pairs of shares
        with any token and head strides (the parts of a fused product's rows);
        out: contiguous [tokens, heads, dim of v].  Returns out.  Raises for a
        step out of its order or of a closed sequence, and warns of a second
        run (a captured one's replays are not seen here)."""
        att, cache, b = self.att, self.att.cache, self.batch
        T, at = b.tokens, [0, 0]
        _rows(at, q, (T, att.heads, cache.k.dim), b.device, "run", "q")
        _rows(at, k, (T, cache.kv_heads, cache.k.dim), b.device, "run", "k")
        _rows(at, v, (T, cache.kv_heads, cache.v.dim), b.device, "run", "v")
        _ptr2(at, out, (T, att.heads, cache.v.dim), b.device, "run", "out")
        self._take_turn()
        with torch.cuda.device(b.device):  # the gates' launches go to the current one
            return self._run(q, k, v, out)

    def _run(self, q, k, v, out):
        att, cache, b, tr = self.att, self.att.cache, self.batch, self.tr
        prepare_batch(self.truncs())
        rotary2(q, att.q_rotary, self.positions, self.q, trunc=tr["q"])
        append2(b, cache.k, k, self.k_mask, cache.v, v, self.v_mask, rotary=att.k_rotary,
                k_trunc=tr["k"])
        scores2(b, cache.k, self.q, self.q_a, self.s_c, self.off, self.s, trunc=tr["s"])
        self.softmax.eval2(self.s, self.p)
        if not att.long_rows:
            return values2(b, cache.v, self.p, self.p_a, self.o_c, self.off, out, trunc=tr["o"],
                           work=self.work)
        z = values2(b, cache.v, self.p, self.p_a, self.o_c, self.off, self.z, trunc=tr["o"],
                    work=self.work)
        return self.softmax.divide2(z, out)
