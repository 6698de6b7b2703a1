"""The parts of a decoder around its attention for two parties on one GPU: the
root-mean-square norm of the residual stream, products with public weights for
any number of rows, products grouped by expert, the experts' weighted sum.

  RMSNorm        s = x + residual, out = s / sqrt(mean(s s) + eps) (* weight)
                 (sufhip_rmsnorm2)
  PublicWeights  one matrix, or one for each expert, with a bias
  Linear         out = act(trunc(x W + bias)) + residual, dense or by expert
                 (sufhip_linear2)
  ExpertMix      out[t] = trunc(sum_k weight[t, k] z[slot[t, k]]) + residual[t]
                 (sufhip_expert_mix2)
  FeedForward    norm, up with an activation, down with the residual's addition
  ExpertFeedForward  the same with each token's experts
  Digits         rows as 8-bit digits, what a norm or a Linear writes and the
                 next Linear reads

Values are shares in Q(frac_bits); weights are public.  Which experts a token
takes is public too, as are their weights in the sum: both parties learn them.
A program that has to hide the choice runs every token through every expert
(a Linear each) and adds them up by shared weights.

Each object holds one use's dealer material, drawn by its own Dealer unless it
is given a seed (two with one seed would open under the same masks; a block's
parts draw from the block's one Dealer).  eval2
issues the key-only halves of its gates first, or waits for `prep` =
(tasks.Prepared, batch) where they were issued before.  Calls of one object go
one after the other (they share its workspace), in one stream or in streams
that wait for each other; on another stream than it was made on, it has to
live until they have run.  A second call of an object with gates opens other
values under the same masks: eval2 warns of it once, and not of a captured
call's replays, of which each is one.

The reference has LayerNorm (include/runtime/phase_tasks.hpp:2186-2668) and
dense public products (src/nn/matmul_publicW.cpp:17-36); it has no experts.
"""
import contextlib
import ctypes
import warnings

import numpy as np
import torch

from . import native, tables
from .kv_attention import _call, _fail, _ptr
from .tasks import (M64, RELU_ALPHA, TABLE_BITS, CoeffLut, Dealer, Triples, Trunc, chain2_args,
                    dev, own_seed, relu_coeffs_for, trunc_jobs)

MAX_ROWS = 1 << 24
LEN_BITS = 26  # of a norm's public 1 / cols, truncated by two gates of 13 bits

_seeds = iter(own_seed, None)


def _dealer(seed):
    """The Dealer of a seed; a block's parts are given its own, from which they
    draw one after the other."""
    if isinstance(seed, Dealer):
        return seed
    return Dealer(next(_seeds) if seed is None else seed)


# ---- arguments ----

def _matrix(arg, t2, shape, d, what, name, written=False):
    """Both parties' [rows, cols] tensors, rows with any stride, into a
    sufhip_matrix2."""
    try:
        t0, t1 = t2
        ok = t0.dtype is torch.int64 and t1.dtype is torch.int64 and t0.shape == shape and \
            t1.shape == shape and t0.get_device() == d and t1.get_device() == d
    except (AttributeError, TypeError, ValueError):
        ok = False
    if not ok:
        _fail(what, "%s must be a pair of int64 tensors of shape %s on the object's device" %
              (name, list(shape)))
    s0, s1 = t0.stride(), t1.stride()
    if shape[1] > 1 and (s0[1] != 1 or s1[1] != 1):
        _fail(what, "the values of a row of %s must be neighbours" % name)
    if shape[0] > 1 and s0[0] != s1[0]:
        _fail(what, "both parties' %s must have the same row stride" % name)
    if written and shape[0] > 1 and s0[0] < shape[1]:
        _fail(what, "rows of %s must not overlap" % name)
    arg.p[0], arg.p[1] = t0.data_ptr(), t1.data_ptr()
    arg.row_stride = s0[0]


def _out(a, t2, shape, d, what, name):
    """An output's addresses and stride into a's fields name, name_stride."""
    m = native.Matrix2()
    _matrix(m, t2, shape, d, what, name, written=True)
    getattr(a, name)[:] = m.p[:]
    setattr(a, name + "_stride", m.row_stride)


def _gate_bits(frac_bits, most, what):
    _extent(frac_bits, 1, most, what, "frac_bits")


def _extent(v, least, most, what, name):
    if not (isinstance(v, (int, np.integer)) and least <= v <= most):
        _fail(what, "%s must be a whole number in [%d, %d]" % (name, least, most))
    return int(v)


def _settle(device):
    """Waits for the current stream: any stream may use what it has written, and
    the memory that it had before."""
    if not torch.cuda.is_current_stream_capturing():
        torch.cuda.current_stream(device).synchronize()


def _gpu(device, what):
    """The GPU that a name or number stands for, with its index."""
    device = torch.device(device)
    if device.type != "cuda":
        _fail(what, "device must be a GPU, not %s" % device)
    return torch.device("cuda", torch.cuda.current_device() if device.index is None
                        else device.index)


class _Block:
    """What the operators share: a dealer, the key-only halves of the gates,
    the device."""

    def __init__(self, prg_state, seed, device):
        self.device = _gpu(device, type(self).__name__)
        self.d = self.device.index
        self.prg_state = bytes(prg_state)
        self.dealer = _dealer(seed)
        self._walks = None
        self.spent = False  # whether its masks have hidden a value
        # Who warns of a second use, and how far above _use its caller stands: of
        # a block's parts the first one, for the block.
        self.warns = (type(self).__name__, 3)

    def _guard(self):
        """Makes the object's device the current one, where it is not."""
        if torch._C._cuda_getDevice() == self.d:
            return contextlib.nullcontext()
        return torch.cuda.device(self.d)

    def _use(self):
        """Warns of a second use, once (a warning takes some microseconds)."""
        if self.spent and self.warns:
            warnings.warn("%s.eval2: an object is for one use; a second one opens other values "
                          "under the same masks, whose difference is then public" % self.warns[0],
                          RuntimeWarning, stacklevel=self.warns[1])
            self.warns = None

    def _gate(self, bits, n):
        return Trunc(self.dealer, bits, n, self.prg_state, device=self.device)

    def _shares(self, v):
        s = self.dealer.words(v.size).reshape(v.shape)
        return dev(s, self.device), dev(v - s, self.device)

    def _jobs(self):
        """(PRG state, jobs, count) of the gates' key-only halves."""
        if self._walks is None:
            self._walks = trunc_jobs(self.truncs())
        return self._walks

    def _walks_of(self, a, prep):
        """The gates' key-only halves: done by the call a, or waited for."""
        if prep is not None:
            prep[0].wait(prep[1])
            return
        state, jobs, a.walk_count = self._jobs()
        a.walk_jobs, a.walk_prg_state = ctypes.addressof(jobs), ctypes.addressof(state)

    def _ready(self, prep):
        """The gates' key-only halves: issued here, or waited for."""
        if prep is not None:
            prep[0].wait(prep[1])
            return
        state, jobs, count = self._jobs()
        native.call("sufhip_trunc_prepare_batch", state, jobs, count,
                    torch._C._cuda_getCurrentRawStream(self.d))


class Digits:
    """Rows of both parties as balanced base-256 digits (sufhip_digits2)."""

    def __init__(self, rows, cols, device="cuda"):
        rows = _extent(rows, 1, MAX_ROWS, "Digits", "rows")
        cols = _extent(cols, 1, MAX_ROWS, "Digits", "cols")
        device = _gpu(device, "Digits")
        nb = native.load().sufhip_digits2_bytes(rows, cols)
        # Zeros: rows that no call writes stand for 0.
        self.buffer = torch.zeros(nb, dtype=torch.int8, device=device)
        _settle(device)
        self.shape, self.d = (rows, cols), self.buffer.get_device()
        self.arg = native.Digits2()
        self.arg.d_digits, self.arg.rows, self.arg.cols = self.buffer.data_ptr(), rows, cols

    def split(self, x):
        """Writes the digits of x (a pair of [rows, cols], any row stride)."""
        m = native.Matrix2()
        _matrix(m, x, self.shape, self.d, "Digits.split", "x")
        with torch.cuda.device(self.d):
            native.call("sufhip_digits2_split", ctypes.byref(m), ctypes.byref(self.arg),
                        torch._C._cuda_getCurrentRawStream(self.d))
        return self

    def values(self):
        """The rows that the digits stand for, a pair of int64 [rows, cols]."""
        rows, cols = self.shape
        d = self.buffer.view(-1, 2, rows, 8, 32).to(torch.int64)
        scale = torch.tensor([1 << 8 * i for i in range(8)], device=d.device)
        v = (d * scale[:, None]).sum(3).permute(1, 2, 0, 3).reshape(2, rows, -1)[:, :, :cols]
        return v[0].contiguous(), v[1].contiguous()


def _digits(arg, digits, shape, d, what, name):
    if not isinstance(digits, Digits) or digits.shape != tuple(shape) or digits.d != d:
        _fail(what, "%s must be Digits(%d, %d) on the object's device" % ((name,) + tuple(shape)))
    arg.d_digits, arg.rows, arg.cols = digits.arg.d_digits, shape[0], shape[1]


# ---- operators ----

class RMSNorm(_Block):
    """Root-mean-square norm of [rows, cols] values with the residual's
    addition: s = x + residual; out = s / sqrt(mean(s s) + eps), times weight.

    In whole numbers, with >> a floor: ms = (((sum s s) >> f) inv) >> 26 with inv
    = round(2^26 / cols); y from `table` (pieces' starts and words (c0, c1) in
    the unsigned order of ms + eps: tables.rsqrt_wide_table, for mean squares up
    to 4096, rougher up to 65536, where y stops falling) and a Newton step; out =
    (s y) >> f, then (out weight) >> f.  The gates take 62 bits: a row's sum of
    squares has to stay below 2^(62 - 2 f), its mean square below 2^(36 - f).
    y is a Q(f) number: at a mean square of 4096 it is 2^(f - 6) steps.  So are
    ms and eps: an eps of less than half a step is 0, and a row whose ms + eps is
    n steps has its y off by a share of up to 0.75 / n (default eps, 12 bits: n
    is 4 at least; a model's 1e-5 is none).  eps must be positive, and at least
    2^-25 for the default table; a table has at most 63 pieces.
    weight: public int64 [cols] in Q(f), or None.  frac_bits at most 13."""

    def __init__(self, rows, cols, prg_state, frac_bits=12, weight=None, eps=1.0 / 1024.0,
                 table=None, seed=None, device="cuda"):
        what = "RMSNorm"
        self.rows = rows = _extent(rows, 1, MAX_ROWS, what, "rows")
        self.cols = cols = _extent(cols, 1, 1 << 20, what, "cols")
        _gate_bits(frac_bits, TABLE_BITS - 1, what)
        if table is None:
            table = tables.rsqrt_wide_table(frac_bits, eps)
        if len(table[0]) > 63:  # 64 intervals, one of them wrapped by the mask
            _fail(what, "a table of %d pieces (eps %r), at most 63 are taken" %
                  (len(table[0]), eps))
        super().__init__(prg_state, seed, device)
        with self._guard():
            self._deal(rows, cols, frac_bits, weight, eps, table, what)
            _settle(self.device)

    def _deal(self, rows, cols, f, weight, eps, table, what):
        deal, n = self.dealer, rows * cols
        self.table, self.f = table, f
        self.inv_len = tables.llround(2.0 ** LEN_BITS / cols)
        self.eps_q = tables.eps_qf(eps, f)
        self.weight = None
        if weight is not None:
            w = torch.as_tensor(weight)
            if w.dtype is not torch.int64 or tuple(w.shape) != (cols,):
                _fail(what, "weight must be int64 [%d]" % cols)
            self.weight = w.to(self.device, copy=True).contiguous()
        # a is the mask of s in both products: s - a is opened once.
        a = deal.words(n).reshape(rows, cols)
        b = deal.words(rows)
        self.a = self._shares(a)
        self.a2 = self._shares((a * a).sum(1, dtype=np.uint64))
        self.b = self._shares(b)
        self.ab = self._shares(a * b[:, None])
        self.tr_ms = [self._gate(bits, rows) for bits in (f, LEN_BITS // 2, LEN_BITS // 2)]
        self.lut = CoeffLut(deal, table[0], table[1], self.device)
        self.tri = [Triples(deal, rows, device=self.device) for _ in range(4)]
        self.tr_rsqrt = [self._gate(bits, rows) for bits in (f, f, f + 1, f)]
        self.tr_norm = self._gate(f, n)
        self.tr_weight = self._gate(f, n) if weight is not None else None
        none = (None, None)
        a = self._args = native.RmsNorm2Args()
        a.rows, a.cols = rows, cols
        a.inv_len, a.eps = self.inv_len, self.eps_q & M64
        for p in (0, 1):
            a.a[p], a.a2[p], a.b[p], a.ab[p] = (t[p].data_ptr() for t in
                                                (self.a, self.a2, self.b, self.ab))
        for q, tr in enumerate(self.tr_ms):
            a.tr_ms[q], a.ms_mask[q] = _epi(tr), tr.mask & M64
        a.rsqrt = chain2_args(native.CHAIN_RSQRT, f, None, rows, self.lut.keys,
                              self.lut.key_bytes, self.lut.intervals, self.lut.mask, self.tri,
                              self.tr_rsqrt, self.b)
        a.rsqrt.out[:] = none
        a.tr_norm, a.norm_mask = _epi(self.tr_norm), self.tr_norm.mask & M64
        nb = native.load().sufhip_rmsnorm2_work_bytes(rows, cols)
        self.work = torch.empty((nb + 7) // 8, dtype=torch.int64, device=self.device)
        a.d_work, a.work_bytes = (self.work.data_ptr() if nb else None), nb
        if weight is not None:
            a.d_weight = self.weight.data_ptr()
            a.tr_weight, a.weight_mask = _epi(self.tr_weight), self.tr_weight.mask & M64

    def truncs(self):
        return self.tr_ms + self.tr_rsqrt + [self.tr_norm] + \
            ([self.tr_weight] if self.tr_weight is not None else [])

    def eval2(self, x, out, residual=None, total=None, digits=None, prep=None):
        """x, residual: pairs of int64 [rows, cols] with any row stride.  out:
        a pair like x, or None; total: a pair for s, or None; digits: a Digits
        for the output, or None.  out and total may each be x or residual
        itself.  Returns out."""
        what, shape, d = "RMSNorm.eval2", (self.rows, self.cols), self.d
        a = native.RmsNorm2Args.from_buffer_copy(self._args)
        _matrix(a.x, x, shape, d, what, "x")
        if residual is not None:
            _matrix(a.residual, residual, shape, d, what, "residual")
        if total is not None:
            _out(a, total, shape, d, what, "total")
        if out is not None:
            _out(a, out, shape, d, what, "out")
        if digits is not None:
            _digits(a.out_digits, digits, shape, d, what, "digits")
        if out is None and digits is None and total is None:
            _fail(what, "no output")
        self._use()
        with self._guard():
            self._walks_of(a, prep)
            _call("sufhip_rmsnorm2", a, d)
        self.spent = True
        return out


def _epi(tr):
    """A gate folded into an operator, which has its own outputs."""
    e = tr.epilogue(tr.work)
    e.y[0] = e.y[1] = None
    return e


class PublicWeights:
    """Public weights on the GPU as int8 digits: W int64 [K, N], or [experts,
    K, N], a numpy array or a tensor; bias int64 [N] or [experts, N] in the
    scale of the products (twice the fractional bits of a Q(f) W and x), or
    None.  Every weight takes as many digits, a byte each, as the largest one:
    1 hold [-128, 127], 2 [-32896, 32639], 3 [-8421504, 8355711], 4
    [-2155905152, 2139062143], so that 15 bits and a sign take 3 where some are
    past 32639 (21 int8 products where 2 take 15).  At most 4, and digits
    K < 2^17."""

    def __init__(self, W, bias=None, device="cuda"):
        what = "PublicWeights"
        W = torch.as_tensor(W)
        if W.dtype is not torch.int64 or W.dim() not in (2, 3) or W.numel() == 0:
            _fail(what, "W must be int64 [K, N] or [experts, K, N]")
        lead = tuple(W.shape[:-2])
        self.experts, (self.K, self.N) = (lead[0] if lead else 1), W.shape[-2:]
        if bias is not None:
            bias = torch.as_tensor(bias)
            if bias.dtype is not torch.int64 or tuple(bias.shape) != lead + (self.N,):
                _fail(what, "bias must be int64 %s" % (list(lead + (self.N,)),))
        device = _gpu(W.device if W.is_cuda else device, what)
        with torch.cuda.device(device):
            W = W.to(device).contiguous()
            self.d = W.get_device()
            self.bias = None if bias is None else bias.to(W.device, copy=True).contiguous()
            self.digits = self._digits_of(int(W.min()), int(W.max()))
            lib = native.load()
            nb = lib.sufhip_linear_planes_bytes(self.experts, self.K, self.N, self.digits)
            if nb == 0:
                _fail(what, "1 to 4096 experts, K up to 65536, N up to 2^24, weights in "
                            "[-2155905152, 2139062143] (4 digits), digits K < 2^17; these %d x "
                            "%d x %d take %d digits" % (self.experts, self.K, self.N, self.digits))
            self.planes = torch.empty((nb + 7) // 8, dtype=torch.int64, device=W.device)
            native.call("sufhip_linear_prepare", W.data_ptr(), self.experts, self.K, self.N,
                        self.digits, self.planes.data_ptr(),
                        torch._C._cuda_getCurrentRawStream(self.d))
            _settle(W.device)
        a = self.arg = native.LinearWeights()
        a.d_planes, a.experts, a.K, a.N, a.digits = (self.planes.data_ptr(), self.experts, self.K,
                                                     self.N, self.digits)
        a.d_bias = None if self.bias is None else self.bias.data_ptr()

    @staticmethod
    def _digits_of(lo, hi):
        """Balanced base-256 digits of every number in [lo, hi]."""
        n, least, most = 1, -128, 127
        while n < 8 and not least <= lo <= hi <= most:
            least, most, n = least * 256 - 128, most * 256 + 127, n + 1
        return n


class Linear(_Block):
    """out = act(trunc(x W + bias)) + residual for both parties and `rows`
    output rows (1 and up).

    act: None, "relu", or a table of cubics (starts, words [pieces, 4]), e.g.
    tables.gelu_table().  With several experts, output row i takes the weights
    of the expert e with offsets[e] <= i < offsets[e + 1]; rows says which x row
    each output row reads.  trunc False: the product itself, at the scale of x
    times W (without an activation).
    x_rows: the most rows of x (rows, unless given)."""

    def __init__(self, weights, rows, prg_state, frac_bits=12, act=None, trunc=True, x_rows=None,
                 seed=None):
        what = "Linear"
        self.weights = weights
        self.rows = _extent(rows, 1, MAX_ROWS, what, "rows")
        self.x_rows = self.rows if x_rows is None else _extent(x_rows, 1, MAX_ROWS, what, "x_rows")
        if self.rows * weights.N >= 1 << 31:
            _fail(what, "rows times N must stay below 2^31")
        _gate_bits(frac_bits, TABLE_BITS if act is None or isinstance(act, str)
                   else TABLE_BITS - 1, what)
        if isinstance(act, str) and act != "relu":
            _fail(what, "act must be None, \"relu\" or a table (starts, words)")
        if act is not None and not trunc:
            _fail(what, "an activation needs the truncation")
        super().__init__(prg_state, seed, torch.device("cuda", weights.d))
        with self._guard():
            self._deal(frac_bits, act, trunc)
            _settle(self.device)

    def _deal(self, f, act, trunc):
        n = self.rows * self.weights.N
        self.f, self.act = f, act
        self.tr = self._gate(f, n) if trunc else None
        self.tr_act, self.tri = [], []
        a = self._args = native.Linear2Args()
        a.w, a.rows = self.weights.arg, self.rows
        if trunc:
            self._epi = _epi(self.tr)
            a.trunc, a.mask = ctypes.pointer(self._epi), self.tr.mask & M64
        if isinstance(act, str):
            lut = self.lut = CoeffLut(self.dealer, RELU_ALPHA, np.zeros((2, 2), np.int64),
                                      self.device, coeffs_for_rin=relu_coeffs_for)
            a.act = native.ACT_RELU
            a.relu.key[0], a.relu.key[1] = (k.data_ptr() for k in lut.keys)
            a.relu.key_bytes, a.relu.intervals, a.relu.mask = (lut.key_bytes, lut.intervals,
                                                              lut.mask & M64)
        elif act is not None:
            lut = self.lut = CoeffLut(self.dealer, act[0], act[1], self.device)
            for _ in range(3):
                tri = Triples(self.dealer, n, device=self.device)
                tri.host = None  # three products of rows N elements: not kept on the host
                self.tri.append(tri)
            self.tr_act = [self._gate(f, n) for _ in range(3)]
            self._cubic = chain2_args(native.CHAIN_CUBIC, f, None, n, lut.keys, lut.key_bytes,
                                      lut.intervals, lut.mask, self.tri, self.tr_act,
                                      self.tri[0].a)
            self._cubic.out[:] = (None, None)
            a.act, a.cubic = native.ACT_CUBIC, ctypes.pointer(self._cubic)
        # The largest workspace of any call of this object.
        a.x_rows = self.x_rows
        some = torch.empty(2, dtype=torch.int64, device=self.device).data_ptr()
        nb = 0
        for offsets in (None, some):
            for digits in (None, some):  # with an epilogue of its own, as walks have it
                a.d_offsets, a.out_digits.d_digits = offsets, digits
                nb = max(nb, native.load().sufhip_linear2_work_bytes(ctypes.byref(a)))
        a.d_offsets = a.out_digits.d_digits = None
        self.work = torch.empty(max(2, (nb + 7) // 8), dtype=torch.int64, device=self.device)
        a.d_work, a.work_bytes = self.work.data_ptr(), self.work.numel() * 8

    def truncs(self):
        return ([self.tr] if self.tr is not None else []) + self.tr_act

    def eval2(self, x, out, residual=None, offsets=None, rows=None, digits=None, prep=None):
        """x: a pair of int64 [x rows, K] with any row stride, or Digits.  out:
        a pair of [rows, N] with any row stride, or None; digits: a Digits for
        the outputs, or None; residual: a pair of [rows, N], which may be out
        itself.  offsets: int32 [experts + 1] on the GPU, not decreasing, needed
        with several experts; rows in no expert are left as they were.  rows:
        int32 [rows] on the GPU, the x row of each output row; one outside x
        stands for a row of zeros.  Returns out."""
        what, d, w = "Linear.eval2", self.d, self.weights
        a = native.Linear2Args.from_buffer_copy(self._args)
        if isinstance(x, Digits):
            n = x.shape[0]
            _digits(a.x_digits, x, (n, w.K), d, what, "x")
        else:
            try:
                n = x[0].shape[0]
            except (AttributeError, TypeError, IndexError):
                _fail(what, "x must be a pair of tensors or Digits")
            _matrix(a.x, x, (n, w.K), d, what, "x")
        if not 1 <= n <= self.x_rows:
            _fail(what, "x has %d rows, at most %d (x_rows) are taken" % (n, self.x_rows))
        a.x_rows = n
        if rows is not None:
            a.d_rows = _ptr(rows, (self.rows,), d, what, "rows", torch.int32)
        elif n < self.rows:
            _fail(what, "x has %d rows for %d: rows says which" % (n, self.rows))
        if offsets is not None:
            a.d_offsets = _ptr(offsets, (w.experts + 1,), d, what, "offsets", torch.int32)
        elif w.experts > 1:
            _fail(what, "several experts need offsets")
        shape = (self.rows, w.N)
        if residual is not None:
            _matrix(a.residual, residual, shape, d, what, "residual")
        if out is not None:
            _out(a, out, shape, d, what, "out")
        if digits is not None:
            _digits(a.out_digits, digits, shape, d, what, "digits")
        elif out is None:
            _fail(what, "no output")
        self._use()
        with self._guard():
            if prep is not None or self.tr is not None:
                self._walks_of(a, prep)
            _call("sufhip_linear2", a, d)
        self.spent = self.tr is not None
        return out


class ExpertMix(_Block):
    """out[t] = trunc(sum_k weights[t, k] z[slots[t, k]]) + residual[t] for both
    parties: each token's experts' outputs by public weights in Q(frac_bits)."""

    def __init__(self, tokens, cols, prg_state, frac_bits=12, seed=None, device="cuda"):
        what = "ExpertMix"
        self.tokens = _extent(tokens, 1, MAX_ROWS, what, "tokens")
        self.cols = _extent(cols, 1, MAX_ROWS, what, "cols")
        if self.tokens * self.cols >= 1 << 31:
            _fail(what, "tokens times cols must stay below 2^31")
        _gate_bits(frac_bits, TABLE_BITS, what)
        super().__init__(prg_state, seed, device)
        a = self._args = native.ExpertMix2Args()
        a.tokens, a.cols = self.tokens, self.cols
        with self._guard():
            self.tr = self._gate(frac_bits, self.tokens * self.cols)
            _settle(self.device)
        self._epi = _epi(self.tr)
        a.trunc, a.mask = ctypes.pointer(self._epi), self.tr.mask & M64

    def truncs(self):
        return [self.tr]

    def eval2(self, z, slots, weights, out, residual=None, prep=None):
        """z: a pair of int64 [rows, cols] with any row stride; slots: int32
        [tokens, each] on the GPU, rows of z (one outside adds nothing);
        weights: int64 [tokens, each] on the GPU.  out, residual: pairs of
        [tokens, cols] with any row stride, which may be the same.  Returns
        out."""
        what, d, shape = "ExpertMix.eval2", self.d, (self.tokens, self.cols)
        a = native.ExpertMix2Args.from_buffer_copy(self._args)
        try:
            n, each = z[0].shape[0], slots.shape[1]
        except (AttributeError, TypeError, IndexError):
            _fail(what, "z must be a pair of [rows, cols], slots [tokens, each]")
        if n > MAX_ROWS or each > 1024:
            _fail(what, "at most 2^24 rows of z, and 1024 of them a token")
        _matrix(a.z, z, (n, self.cols), d, what, "z")
        a.z_rows, a.each = n, each
        a.d_slots = _ptr(slots, (self.tokens, each), d, what, "slots", torch.int32)
        a.d_weights = _ptr(weights, (self.tokens, each), d, what, "weights")
        if residual is not None:
            _matrix(a.residual, residual, shape, d, what, "residual")
        _out(a, out, shape, d, what, "out")
        self._use()
        with self._guard():
            self._ready(prep)
            _call("sufhip_expert_mix2", a, d)
        self.spent = True
        return out


# ---- blocks ----

def route(experts_of, experts):
    """The tables of a public choice: experts_of int [tokens, each], on any
    device.  Returns int32 tensors there: offsets [experts + 1] and rows
    [tokens * each] for Linear (the pairs in the order of their experts, a
    token's before the next one's), slots [tokens, each] for ExpertMix.  A
    number outside [0, experts) is in no expert and adds nothing to its
    token's sum.  Sorts, so not for a captured stream."""
    if experts_of.dim() != 2 or experts_of.dtype not in (torch.int32, torch.int64):
        _fail("route", "experts_of must be int32 or int64 [tokens, each]")
    tokens, each = experts_of.shape
    e = experts_of.reshape(-1).to(torch.int64)
    e = torch.where((e >= 0) & (e < experts), e, experts)
    order = torch.argsort(e, stable=True)
    offsets = torch.searchsorted(e[order], torch.arange(experts + 1, device=e.device))
    place = torch.empty_like(order)
    place[order] = torch.arange(tokens * each, device=e.device)
    slots = torch.where(e < experts, place, -1).view(tokens, each)
    rows = torch.div(order, max(each, 1), rounding_mode="floor")
    return offsets.to(torch.int32), rows.to(torch.int32), slots.to(torch.int32)


class FeedForward:
    """out = s + down(act(up(norm(s)))) with s = x + residual, over rows tokens:
    what follows a decoder's attention, from its output and the residual
    stream.  The norm hands its output on as digits, up its activations.
    up, down: PublicWeights of [cols, hidden] and [hidden, cols]; act as in
    Linear; weight, eps, table as in RMSNorm.  seed: of the block's dealer, from
    which its parts draw."""

    def __init__(self, rows, up, down, prg_state, frac_bits=12, act="relu", weight=None,
                 eps=1.0 / 1024.0, table=None, seed=None):
        _pair("FeedForward", up, down, 1)
        dev_ = torch.device("cuda", up.d)
        deal = _dealer(seed)
        self.rows, self.cols = rows, up.K
        self.norm = RMSNorm(rows, up.K, prg_state, frac_bits, weight, eps, table, deal, dev_)
        self.up = Linear(up, rows, prg_state, frac_bits, act, seed=deal)
        self.down = Linear(down, rows, prg_state, frac_bits, seed=deal)
        self.total = [torch.empty(rows, up.K, dtype=torch.int64, device=dev_) for _ in range(2)]
        self.normed, self.hidden = Digits(rows, up.K, dev_), Digits(rows, up.N, dev_)
        self.norm.warns, self.up.warns, self.down.warns = ("FeedForward", 4), None, None

    def truncs(self):
        return self.norm.truncs() + self.up.truncs() + self.down.truncs()

    def eval2(self, x, out, residual=None, prep=None):
        """x, out, residual: pairs of int64 [rows, cols] with any row stride;
        out may be x or residual.  Returns out."""
        # Before the norm uses up its masks.
        _matrix(native.Matrix2(), out, (self.rows, self.cols), self.norm.d, "FeedForward.eval2",
                "out", written=True)
        self.norm.eval2(x, None, residual, self.total, self.normed, prep)
        self.up.eval2(self.normed, None, digits=self.hidden, prep=prep)
        return self.down.eval2(self.hidden, out, self.total, prep=prep)


class ExpertFeedForward:
    """out[t] = s[t] + sum_k weights[t, k] down_e(act(up_e(norm(s)[t]))), e the
    k-th expert of token t, with s = x + residual: FeedForward with `each`
    experts a token.  up, down: PublicWeights of [experts, cols, hidden] and
    [experts, hidden, cols]; the rest as in FeedForward."""

    def __init__(self, tokens, each, up, down, prg_state, frac_bits=12, act="relu", weight=None,
                 eps=1.0 / 1024.0, table=None, seed=None):
        what = "ExpertFeedForward"
        tokens = _extent(tokens, 1, MAX_ROWS, what, "tokens")
        each = _extent(each, 1, 1024, what, "each")
        _pair(what, up, down, None)
        dev_ = torch.device("cuda", up.d)
        deal = _dealer(seed)
        n = tokens * each
        self.tokens, self.each, self.cols = tokens, each, up.K
        self.norm = RMSNorm(tokens, up.K, prg_state, frac_bits, weight, eps, table, deal, dev_)
        self.up = Linear(up, n, prg_state, frac_bits, act, x_rows=tokens, seed=deal)
        self.down = Linear(down, n, prg_state, frac_bits, seed=deal)
        self.mix = ExpertMix(tokens, up.K, prg_state, frac_bits, deal, dev_)
        self.total = [torch.empty(tokens, up.K, dtype=torch.int64, device=dev_)
                      for _ in range(2)]
        # Pairs in no expert are not written, nor read by the sum.
        self.z = [torch.empty(n, up.K, dtype=torch.int64, device=dev_) for _ in range(2)]
        self.normed, self.hidden = Digits(tokens, up.K, dev_), Digits(n, up.N, dev_)
        self.norm.warns = ("ExpertFeedForward", 4)
        self.up.warns = self.down.warns = self.mix.warns = None

    def truncs(self):
        return self.norm.truncs() + self.up.truncs() + self.down.truncs() + self.mix.truncs()

    def eval2(self, x, out, offsets, rows, slots, weights, residual=None, prep=None):
        """x, out, residual as in FeedForward; offsets, rows, slots: route() of
        the tokens' experts, on the GPU; weights: int64 [tokens, each] in
        Q(frac_bits) on the GPU.  Returns out."""
        what, d, experts = "ExpertFeedForward.eval2", self.norm.d, self.up.weights.experts
        # Before the norm uses up its masks.
        _matrix(native.Matrix2(), out, (self.tokens, self.cols), d, what, "out", written=True)
        if experts > 1 or offsets is not None:
            _ptr(offsets, (experts + 1,), d, what, "offsets", torch.int32)
        if self.each > 1 or rows is not None:
            _ptr(rows, (self.up.rows,), d, what, "rows", torch.int32)
        each = slots.shape[1] if getattr(slots, "ndim", 0) == 2 else self.each
        _ptr(slots, (self.tokens, each), d, what, "slots", torch.int32)
        _ptr(weights, (self.tokens, each), d, what, "weights")
        self.norm.eval2(x, None, residual, self.total, self.normed, prep)
        self.up.eval2(self.normed, None, offsets=offsets, rows=rows, digits=self.hidden,
                      prep=prep)
        self.down.eval2(self.hidden, self.z, offsets=offsets, prep=prep)
        return self.mix.eval2(self.z, slots, weights, out, self.total, prep)


def _pair(what, up, down, experts):
    """up and down fit each other."""
    if not isinstance(up, PublicWeights) or not isinstance(down, PublicWeights):
        _fail(what, "up and down must be PublicWeights")
    if (up.K, up.N, up.experts, up.d) != (down.N, down.K, down.experts, down.d):
        _fail(what, "up [%d, %d] and down [%d, %d] do not fit" % (up.K, up.N, down.K, down.N))
    if experts is not None and up.experts != experts:
        _fail(what, "of %d matrices ExpertFeedForward makes one" % up.experts)
