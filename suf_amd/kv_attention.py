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
                   and rotation with its truncation gate

The reference keeps a cache of shares (include/nn/kv_cache.hpp) and multiplies
it by a fresh triple for every new token; its attention is
src/nn/attention_block.cpp:931-1900.
"""
import ctypes
import math

import numpy as np
import torch

from . import native, pfss
from .softmax import SoftmaxBlock
from .tasks import Dealer, Trunc, dev, dev_i32, prepare_batch

M64 = (1 << 64) - 1


# ---- arguments ----

def _fail(what, msg):
    raise ValueError("%s: %s" % (what, msg))


def _check(t, shape, dtype, device, what, name):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or tuple(t.shape) != tuple(shape):
        _fail(what, "%s must be a %s tensor of shape %s" % (name, dtype, list(shape)))
    if t.device != device or device.type != "cuda":
        _fail(what, "%s must be on the GPU, with the other tensors (%s)" % (name, device))
    return t


def _dense(t, shape, device, what, name, dtype=torch.int64):
    if not _check(t, shape, dtype, device, what, name).is_contiguous():
        _fail(what, "%s must be contiguous" % name)
    return t.data_ptr()


def _dense2(arr, pair, shape, device, what, name):
    """Both parties' contiguous tensors into a void*[2]."""
    if len(pair) != 2:
        _fail(what, "%s must be a pair (party 0, party 1)" % name)
    arr[0] = _dense(pair[0], shape, device, what, name)
    arr[1] = _dense(pair[1], shape, device, what, name)


def _strides(pair, shape, device, what, name, written=False):
    """Token and head stride of both parties' [tokens, heads, dim] tensors."""
    if len(pair) != 2:
        _fail(what, "%s must be a pair (party 0, party 1)" % name)
    for t in pair:
        _check(t, shape, torch.int64, device, what, name)
        if shape[2] > 1 and t.stride(2) != 1:
            _fail(what, "the values of a head of %s must be neighbours" % name)
    st = pair[0].stride()[:2]
    if pair[1].stride()[:2] != st and pair[0].numel():
        _fail(what, "both parties' %s must have the same strides" % name)
    if written and any(n > 1 and s == 0 for n, s in zip(shape[:2], st)):
        _fail(what, "rows of %s must not overlap" % name)
    return st


def _rows(out, pair, shape, device, what, name):
    out.token_stride, out.head_stride = _strides(pair, shape, device, what, name)
    out.p[0], out.p[1] = pair[0].data_ptr(), pair[1].data_ptr()


class _Launch:
    """The stream of `device`, and that device current while a call is made."""

    def __init__(self, device):
        self.guard = None if device.index == torch.cuda.current_device() else \
            torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _call(name, args, device):
    with _Launch(device) as stream:
        native.call(name, ctypes.byref(args), stream)


def _epilogue(args, trunc, out, n, what):
    """trunc: a prepared tasks.Trunc whose outputs go to `out`."""
    if trunc is None:
        return None
    if not trunc.has_table():
        _fail(what, "the truncation must be a GapARS gate of at most 14 bits")
    if trunc.n < n:
        _fail(what, "the truncation is for %d elements, not %d" % (trunc.n, n))
    epi = trunc.epilogue(out)
    args.trunc = ctypes.pointer(epi)
    return epi


class Rotary:
    """A public rotary table: int32 [positions, rot / 2, 2] fixed-point (cos,
    sin) on the GPU, for heads of `dim` values.  interleaved pairs neighbours
    (2i, 2i + 1), otherwise pair i is (i, rot / 2 + i).  pass_mul, the table's
    1, multiplies the values past the rotated part."""

    def __init__(self, table, dim, interleaved=False, pass_mul=1 << 12):
        if table.dim() != 3 or table.shape[2] != 2 or 2 * table.shape[1] > dim:
            _fail("Rotary", "the table must be [positions, rot / 2, 2] with rot <= dim")
        _dense(table, table.shape, table.device, "Rotary", "the table", torch.int32)
        self.table, self.dim, self.interleaved = table, int(dim), bool(interleaved)
        self.pass_mul = int(pass_mul)
        r = self.arg = native.RotaryTable()
        r.d_table = table.data_ptr() or None
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
                            between; the table is scaled by 0.1 ln(s) + 1"""
        rot = dim if rot is None else rot
        table, one = rotary_table(positions, rot, base, frac_bits, scale, scaling)
        return cls(torch.from_numpy(table).to(device), dim, interleaved, one)


def rotary_table(positions, rot, base=10000.0, frac_bits=12, scale=1.0, scaling=None):
    """(int32 [positions, rot / 2, 2], the table's 1): Rotary.build's factors."""
    if rot < 0 or rot % 2 or positions < 0 or not 0 < frac_bits <= 28:
        _fail("rotary_table", "rot must be even, positions >= 0 and frac_bits in [1, 28]")
    i = np.arange(rot // 2, dtype=np.float64)
    freq = float(base) ** (-2.0 * i / max(rot, 1))
    if scaling is not None:
        kind, s = scaling[0], float(scaling[1])
        if s < 1:
            _fail("rotary_table", "positions are stretched by a factor of at least 1")
        if kind == "linear":
            freq = freq / s
        elif kind == "base":
            if rot > 2:
                freq = (float(base) * s ** (rot / (rot - 2.0))) ** (-2.0 * i / rot)
        elif kind == "parts":
            trained, slow, fast = (float(v) for v in scaling[2:])
            if not 0 <= slow < fast:
                _fail("rotary_table", "parts need 0 <= slow < fast")
            turns = trained * freq / (2.0 * math.pi)
            keep = np.clip((turns - slow) / (fast - slow), 0.0, 1.0)
            freq = freq * keep + freq / s * (1.0 - keep)
            scale = scale * (0.1 * math.log(s) + 1.0)
        else:
            _fail("rotary_table", "unknown scaling %r" % (kind,))
    one = scale * (1 << frac_bits)
    if abs(one) >= 1 << 31:
        _fail("rotary_table", "scale * 2^frac_bits must stay below 2^31")
    ang = np.arange(positions, dtype=np.float64)[:, None] * freq
    table = np.rint(np.stack([np.cos(ang), np.sin(ang)], -1) * one).astype(np.int32)
    return table, int(round(one))


class Pool:
    """The pages of keys or of values: e, b0, b1 int64 [pages, kv_heads,
    page_tokens, dim] on the GPU (the open value - b, both parties' shares of
    b); page_tokens a power of two."""

    def __init__(self, e, b0, b1):
        if e.dim() != 4:
            _fail("Pool", "the arrays must be [pages, kv_heads, page_tokens, dim]")
        p = self.arg = native.KvPool()
        p.e = _dense(e, e.shape, e.device, "Pool", "e")
        p.b[0] = _dense(b0, e.shape, e.device, "Pool", "b0")
        p.b[1] = _dense(b1, e.shape, e.device, "Pool", "b1")
        p.pages, p.kv_heads, p.page_tokens, p.dim = e.shape
        self.e, self.b, self.device = e, (b0, b1), e.device
        self.kv_heads, self.dim = e.shape[1], e.shape[3]


class Batch:
    """The packed new tokens of some sequences and their pages: cu int32
    [seqs + 1] (first token of each sequence, the end last), kv_lens int32
    [seqs] (keys, the new ones included), pages int32 [seqs, max_pages] (pool
    page of each page_tokens keys, -1: none), all on the GPU.  tokens: rows of
    every token array; those from cu[-1] on are padding and are left alone.
    max_new, max_keys: bounds by which launches are laid out."""

    def __init__(self, cu, kv_lens, pages, tokens, max_new, max_keys):
        if kv_lens.dim() != 1 or pages.dim() != 2:
            _fail("Batch", "kv_lens must be [seqs], pages [seqs, max_pages]")
        seqs, d = kv_lens.shape[0], kv_lens.device
        b = self.arg = native.KvBatch()
        b.d_cu_tokens = _dense(cu, (seqs + 1,), d, "Batch", "cu", torch.int32)
        b.d_kv_lens = _dense(kv_lens, (seqs,), d, "Batch", "kv_lens", torch.int32)
        b.d_pages = _dense(pages, (seqs, pages.shape[1]), d, "Batch", "pages", torch.int32)
        b.seqs, b.tokens, b.max_pages = seqs, int(tokens), pages.shape[1]
        b.max_new, b.max_keys = int(max_new), int(max_keys)
        self.cu, self.kv_lens, self.pages = cu, kv_lens, pages
        self.tokens, self.device = int(tokens), d


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
    x, which may be x itself, or None for new ones (zeros in padding rows).  trunc: a prepared
    tasks.Trunc the rotated values go through.  Returns out."""
    what = "rotary2"
    shape, d = tuple(x[0].shape), x[0].device
    if len(shape) != 3 or shape[2] != rotary.dim:
        _fail(what, "x must be [tokens, heads, %d]" % rotary.dim)
    if rotary.table.device != d:
        _fail(what, "the table is on another device than x")
    if out is None:
        out = tuple(torch.zeros(shape, dtype=torch.int64, device=d) for _ in range(2))
    a = native.Rotary2Args()
    _rows(a.x, x, shape, d, what, "x")
    a.tokens, a.heads, a.dim = shape
    a.rot = rotary.arg
    a.d_positions = _dense(positions, shape[:1], d, what, "positions", torch.int32)
    a.out_token_stride, a.out_head_stride = _strides(out, shape, d, what, "out", written=True)
    a.out[0], a.out[1] = out[0].data_ptr(), out[1].data_ptr()
    epi = _epilogue(a, trunc, out, x[0].numel(), what)
    if epi is not None:
        a.mask = trunc.mask & M64
    _call("sufhip_rotary2", a, d)
    return out


def _append_part(part, batch, pool, x, mask, rotary, positions, trunc, what, name):
    T, d = batch.tokens, batch.device
    shape = (T, pool.kv_heads, pool.dim)
    if pool.device != d:
        _fail(what, "the pool and the batch are on different devices")
    _rows(part.x, x, shape, d, what, name)
    _dense2(part.mask, mask, shape, d, what, name + "_mask")
    part.pool = pool.arg
    if rotary is not None:
        if rotary.dim != pool.dim or rotary.table.device != d:
            _fail(what, "the rotary table is for heads of %d on %s" %
                  (rotary.dim, rotary.table.device))
        part.rot = rotary.arg
        if positions is not None:
            part.d_positions = _dense(positions, (T,), d, what, "positions", torch.int32)
    if trunc is None:
        return None
    gate, y = trunc if isinstance(trunc, tuple) else (trunc, None)
    if y is not None:
        for t in y:
            _dense(t, shape, d, what, "the truncated shares")
    epi = _epilogue(part, gate, y if y is not None else x, x[0].numel(), what)
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
    shares)."""
    what = "append2"
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
    a.batch, a.pool, a.heads = batch.arg, pool.arg, heads
    if pool.device != batch.device:
        _fail(what, "the pool and the batch are on different devices")
    a.d_row_offsets = _dense(offsets, (heads * batch.tokens + 1,), batch.device, what, "offsets",
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
    if q[0].dim() != 3 or q[0].shape[0] != batch.tokens or q[0].shape[2] != pool.dim:
        _fail(what, "q must be [%d, heads, %d]" % (batch.tokens, pool.dim))
    shape = tuple(q[0].shape)
    g = _product(batch, pool, offsets, shape[1], what)
    _rows(g.x, q, shape, d, what, "q")
    _dense2(g.a, a, shape, d, what, "a")
    g.n = out[0].numel()
    _dense2(g.c, c, (g.n,), d, what, "c")
    _dense2(g.out, out, (g.n,), d, what, "out")
    epi = _epilogue(g, trunc, out, g.n, what)
    if epi is not None:
        g.mask = trunc.mask & M64
    _call("sufhip_kv_scores2", g, d)
    return out


def values_work(batch, pool, heads):
    """The workspace of a values2 call on this batch (None: none needed)."""
    nb = native.load().sufhip_kv_values2_work_bytes(ctypes.byref(batch.arg),
                                                    ctypes.byref(pool.arg), heads)
    return torch.empty((nb + 7) // 8, dtype=torch.int64, device=batch.device) if nb else None


def values2(batch, pool, p, a, c, offsets, out, trunc=None, work=None):
    """Rows of probabilities times the cached values: p, a (pairs of packed
    int64 [n]; the dealer's mask shares of p), c and out (pairs of contiguous
    int64 [tokens, heads, dim]: the shares of a's product with the values'
    masks; the weighted values, heads side by side).  offsets as in scores2.
    work: values_work(...) of a batch with the same extents, allocated here if
    it is not given.  Returns out."""
    what, d = "values2", batch.device
    if out[0].dim() != 3 or out[0].shape[0] != batch.tokens or out[0].shape[2] != pool.dim:
        _fail(what, "out must be [%d, heads, %d]" % (batch.tokens, pool.dim))
    shape = tuple(out[0].shape)
    g = _product(batch, pool, offsets, shape[1], what)
    g.n = p[0].numel()
    _dense2(g.x.p, p, (g.n,), d, what, "p")
    _dense2(g.a, a, (g.n,), d, what, "a")
    _dense2(g.c, c, shape, d, what, "c")
    _dense2(g.out, out, shape, d, what, "out")
    epi = _epilogue(g, trunc, out, out[0].numel(), what)
    if epi is not None:
        g.mask = trunc.mask & M64
    with _Launch(d) as stream:
        if work is None:
            work = values_work(batch, pool, shape[1])
        if work is not None:
            g.d_work, g.work_bytes = work.data_ptr(), work.numel() * 8
        native.call("sufhip_kv_values2", ctypes.byref(g), stream)
    return out
