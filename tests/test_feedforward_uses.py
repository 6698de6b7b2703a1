"""The feed-forward operators on the CPU: workspaces, and what stands between
one use of an object and the next."""
import contextlib
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import feedforward_reference as ref
from suf_amd import feedforward as ff
from suf_amd import native, pfss, tables, tasks
from test_feedforward_arguments import at, gate, linear_args, mix_args, norm_args, put, refused

M64 = (1 << 64) - 1


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


@pytest.mark.parametrize("name,args", [("sufhip_linear2", lambda **kw: linear_args(rows=0, **kw)),
                                       ("sufhip_rmsnorm2", lambda **kw: norm_args(rows=0, **kw)),
                                       ("sufhip_rmsnorm2", lambda **kw: norm_args(cols=0, **kw))])
def test_walks_of_a_call_without_rows(name, args):
    """They are issued all the same: a job that no launch takes is refused."""
    refused(name, args(walk_count=1), "walk_jobs")
    refused(name, args(walk_count=-1), "walk_jobs")
    state, jobs = ctypes.create_string_buffer(pfss.PRG_STATE_BYTES), (native.TruncJob * 1)()
    jobs[0].kind = 77
    a = args(walk_count=1, walk_jobs=ctypes.addressof(jobs),
             walk_prg_state=ctypes.addressof(state))
    assert getattr(native.load(), name)(ctypes.byref(a), None) == -1


# ---- outputs over what the gates are read from ----

def cubic_args(stride=1, **kw):
    """A product of 4 x 32 outputs with a cubic's chain: gates at 40 to 43, the
    LUT at 50, triples at 52 and 53."""
    a = linear_args(act=native.ACT_CUBIC)
    c = native.Chain2Args()
    c.kind, c.frac_bits, c.n = native.CHAIN_CUBIC, 12, 4 * 32
    c.lut[0], c.lut[1], c.intervals = at(50), at(51), 4
    c.lut_key_bytes = native.load().sufhip_interval_lut_key_bytes(4, 4)
    for t in list(c.a[:3]) + list(c.b[:3]) + list(c.c[:3]):
        t.p[0], t.p[1], t.len, t.stride, t.mul = at(52), at(53), 4 * 32, stride, 1
    for e in c.trunc[:3]:
        gate(e)
    a.cubic = ctypes.pointer(c)
    return put(a, **kw)


def relu_args(**kw):
    size = native.load().sufhip_interval_lut_key_bytes(3, 2)
    return linear_args(act=native.ACT_RELU, relu__key0=at(20), relu__key1=at(21),
                       relu__intervals=3, relu__key_bytes=size, **kw)


def large_norm(**kw):
    return norm_args(rows=1 << 12, cols=1 << 9, x__row_stride=1 << 9, out_stride=1 << 9,
                     rsqrt__n=1 << 12, **{"d_work": at(30), "work_bytes": 1 << 20, **kw})


def digits(p, rows, cols):
    return dict(out_digits__d_digits=p, out_digits__rows=rows, out_digits__cols=cols)


OVER = [("sufhip_linear2", f, kw) for f, places in
        ((linear_args, (40, 41, 42, 43)), (relu_args, (20, 21, 40)),
         (cubic_args, (40, 42, 50, 51, 52, 53)))
        for k in places for kw in (dict(out0=at(k)), dict(out1=at(k)), dict(d_work=at(k)),
                                   digits(at(k), 4, 32))
        if "d_work" not in kw or f is not linear_args]
OVER += [("sufhip_linear2", cubic_args, dict(out0=at(52) + 8 * 127)),
         ("sufhip_linear2", lambda **kw: cubic_args(stride=3, **kw),
          dict(out0=at(53) + 8 * 3 * 127)),
         ("sufhip_linear2", linear_args, dict(out0=at(42) + (8 << 12) - 8)),
         ("sufhip_linear2", linear_args, dict(d_work=at(43), **digits(at(9), 4, 32)))]
OVER += [("sufhip_rmsnorm2", f, kw) for k in (40, 41, 42, 43, 50, 51, 52, 53)
         for f, kw in ((norm_args, dict(out0=at(k))), (norm_args, digits(at(k), 3, 40)),
                       (norm_args, dict(total0=at(k), total1=at(31), total_stride=40)),
                       (large_norm, dict(d_work=at(k))))]
OVER += [("sufhip_expert_mix2", mix_args, dict([(o, at(k))])) for k in (40, 41, 42, 43)
         for o in ("out0", "out1")]


@pytest.mark.parametrize("name,args,kw", OVER)
def test_outputs_over_keys_tables_and_triples(name, args, kw):
    refused(name, args(**kw), "gate")


# ---- whose words are whose ----

class HostWeights(ff.PublicWeights):
    """The extents of public weights."""

    def __init__(self, K, N, experts=1):
        self.K, self.N, self.experts, self.digits, self.d = K, N, experts, 2, -1
        a = self.arg = native.LinearWeights()
        a.experts, a.K, a.N, a.digits = experts, K, N, 2


@pytest.fixture
def on_host(monkeypatch):
    """Material is dealt on the host; here it stays there."""
    cpu = torch.device("cpu")
    monkeypatch.setattr(ff, "_gpu", lambda device, what: cpu)
    monkeypatch.setattr(ff._Block, "_guard", lambda self: contextlib.nullcontext())
    monkeypatch.setattr(ff, "Digits", lambda *a: None)
    monkeypatch.setattr(ff, "_settle", lambda device: None, raising=False)
    monkeypatch.setattr(torch, "device", lambda *a: cpu)
    monkeypatch.setattr(tasks.pfss, "trunc_gen",
                        lambda *a: [torch.zeros(8, dtype=torch.uint8)] * 2)


def words_of(o, names):
    """All words that an object's dealer drew or derived, by part, without the
    small numbers of layouts and headers."""
    out = set()

    def walk(v):
        if isinstance(v, torch.Tensor):
            if v.dtype is torch.int64:
                out.update(v.reshape(-1).tolist())
        elif isinstance(v, np.ndarray):
            if v.dtype in (np.uint64, np.int64):
                out.update(v.reshape(-1).view(np.int64).tolist())
        elif isinstance(v, (list, tuple)):
            for w in v:
                walk(w)
        elif isinstance(v, (ff.Trunc, ff.Triples, ff.CoeffLut)):
            walk([w for k, w in vars(v).items() if k not in ("work", "blobs", "keys")])
    walk([vars(o)[k] for k in names if k in vars(o)])
    return {w for w in out if abs(w) > 1 << 40}


MATERIAL = ("a", "a2", "b", "ab", "tr_ms", "tr_rsqrt", "tr_norm", "tr_weight", "tri", "tr",
            "tr_act")


def parts(block):
    return [words_of(p, MATERIAL) for p in
            (block.norm, block.up, block.down) + ((block.mix,) if hasattr(block, "mix") else ())]


@pytest.mark.parametrize("experts", [1, 3])
def test_blocks_of_neighbouring_seeds_share_no_material(on_host, experts):
    """A model's layers, seeded 0, 1, 2 and so on: no word of one part's masks,
    triples and gates is another's, in a block or between two."""
    up, down = HostWeights(8, 6, experts), HostWeights(6, 8, experts)
    kw = dict(act=tables.gelu_table(12), weight=torch.full((8,), 5000))
    make = (lambda s: ff.FeedForward(3, up, down, bytes(range(128)), seed=s, **kw)) if experts == 1 else \
        (lambda s: ff.ExpertFeedForward(3, 2, up, down, bytes(range(128)), seed=s, **kw))
    sets = [p for s in range(6) for p in parts(make(s))]
    assert all(len(p) > 8 for p in sets)
    assert len(set().union(*sets)) == sum(len(p) for p in sets)
    again = parts(make(2))  # one seed, one material
    assert again == sets[2 * len(again):3 * len(again)]


def test_unseeded_objects_differ_between_processes():
    """Two runs of a program do not open their values under the same masks."""
    code = ("from suf_amd import feedforward as ff, kv_attention as kv\n"
            "kv.Rotary.build = classmethod(lambda *a, **k: None)\n"
            "class Cache:\n"
            "    class k: dim = 8\n"
            "    kv_heads, device = 1, 'cpu'\n"
            "att = kv.CachedAttention(Cache, 1, b'', 64).dealer.seed\n"
            "print(next(ff._seeds), next(ff._seeds), att)\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    runs = [subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                           check=True).stdout.split() for _ in range(2)]
    assert len(runs[0]) == 3 and len(set(runs[0] + runs[1])) == 6


# ---- the norm's range ----

@pytest.mark.parametrize("f", [8, 10, 12, 13])
@pytest.mark.parametrize("eps", [1.0 / 1024.0, 1e-5, 1e-6])
def test_norm_of_large_mean_squares(f, eps):
    """Past the table's range y neither turns negative nor grows, up to sums that
    wrap; at 12 bits it is as near as the table says."""
    alpha, words = tables.rsqrt_wide_table(f, eps)
    assert np.all(alpha[1:] > alpha[:-1]) and len(alpha) <= 63
    v = np.concatenate([np.exp2(np.linspace(12, 16, 4001)), np.exp2(np.arange(16, 63 - f))])
    v = np.concatenate([np.rint(v * 2.0 ** f).astype(np.uint64),
                        np.array([1 << 63, M64], np.uint64)])
    y = ref.rsqrt(v, (alpha, words), f).view(np.int64) / 2.0 ** f
    top = 1.13 / 64 + 1.5 * 2.0 ** -f  # a constant's half octave, a step of 1.5 y
    assert np.all((y >= 0) & (y <= top))
    assert len(set(y[v >= 65536 << f])) == 1
    if f == 12 and eps > 1e-4:
        off = np.abs(y * np.sqrt(v / 2.0 ** f) - 1)
        assert off[v < 8192 << f].max() <= 0.061 and off[v < 65536 << f].max() <= 0.13
        assert y[-1] == 1 / 256


@pytest.mark.parametrize("eps", [0, 0.0, -1e-5, float("nan"), float("inf"), 1e-8, 2.0 ** -26])
def test_norm_refuses_an_epsilon_that_no_table_takes(eps):
    with pytest.raises(ValueError, match="eps"):
        ff.RMSNorm(1, 8, bytes(range(128)), eps=eps)


def test_norm_refuses_long_tables():
    with pytest.raises(ValueError, match="63"):
        ff.RMSNorm(1, 8, bytes(range(128)), table=(np.arange(64), np.zeros((64, 2))))
    assert len(tables.rsqrt_wide_table(12, 2.0 ** -25)[0]) == 63


@pytest.mark.parametrize("f", [10, 12])
@pytest.mark.parametrize("eps", [1.0 / 1024.0, 1e-5, 1e-6])
def test_norm_of_small_mean_squares(f, eps):
    """What the mean square's and the epsilon's own steps leave of 1/sqrt(ms +
    eps), n steps of them: the floor of ms up to a step, eps half of one, so 1.5
    steps of n, half of it in the root; and the table's 1.5 e^2, e <= 6.25 % (a
    chord of an octave, or of one of the first steps, which are shorter)."""
    table = tables.rsqrt_wide_table(f, eps)
    ms = np.exp2(np.linspace(-f - 3, 0, 20001))
    n = np.floor(ms * 2.0 ** f) + tables.eps_qf(eps, f)
    at = n >= 1
    y = ref.rsqrt(n[at].astype(np.uint64), table, f).view(np.int64) / 2.0 ** f
    off = np.abs(y * np.sqrt(ms[at] + eps) - 1)
    assert np.all(off <= 0.75 / n[at] + 1.5 * 0.0625 ** 2 + 4 * 2.0 ** -f)
