"""The cached-attention calls on the CPU: what they refuse before any device
work, the rotary tables, the cache's bookkeeping."""
import ctypes
import math

import numpy as np
import pytest
import torch

from suf_amd import kv_attention as kv
from suf_amd import native

PTR = 1 << 20  # an address that nothing here reads: 16-byte aligned


def rows(a, ts=64, hs=64):
    a.p[0], a.p[1], a.token_stride, a.head_stride = PTR, PTR, ts, hs


def pool(p, **kw):
    p.e, p.b[0], p.b[1] = PTR, PTR, PTR
    p.pages, p.page_tokens, p.kv_heads, p.dim = 4, 16, 2, 64
    for k, v in kw.items():
        setattr(p, k, v)


def batch(b, **kw):
    b.d_cu_tokens = b.d_kv_lens = b.d_pages = PTR
    b.seqs, b.tokens, b.max_pages, b.max_new, b.max_keys = 1, 1, 2, 1, 32
    for k, v in kw.items():
        setattr(b, k, v)


def refused(name, args, *words):
    lib = native.load()
    rc = getattr(lib, name)(ctypes.byref(args) if args is not None else None, None)
    msg = lib.sufhip_last_error().decode()
    assert rc == -1, (name, rc)
    assert msg.startswith(name) and all(w in msg for w in words), msg


def trunc(**kw):
    e = native.TruncEpilogue()
    e.key[0] = e.key[1] = e.table[0] = e.table[1] = e.y[0] = e.y[1] = PTR
    e.frac_bits, e.work_bytes = 12, 1 << 30
    for k, v in kw.items():
        setattr(e, k, v)
    return ctypes.pointer(e)


def rotary_args(**kw):
    a = native.Rotary2Args()
    rows(a.x)
    a.tokens, a.heads, a.dim = 2, 3, 64
    a.rot.d_table, a.rot.positions, a.rot.rot = PTR, 8, 64
    a.d_positions, a.out[0], a.out[1] = PTR, PTR, PTR
    a.out_token_stride = a.out_head_stride = 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_rotary2_refuses():
    refused("sufhip_rotary2", None, "null args")
    for kw in ({"tokens": -1}, {"heads": -1}, {"dim": -1}):
        refused("sufhip_rotary2", rotary_args(**kw), ">= 0")
    refused("sufhip_rotary2", rotary_args(d_positions=None), "d_positions")
    a = rotary_args()
    a.out[1] = None
    refused("sufhip_rotary2", a, "outputs")
    a = rotary_args()
    a.x.p[0] = None
    refused("sufhip_rotary2", a, "rows")
    for field, v in (("rot", 63), ("rot", 66), ("rot", -2), ("positions", -1),
                     ("d_table", PTR + 4), ("d_table", None)):
        a = rotary_args()
        setattr(a.rot, field, v)
        refused("sufhip_rotary2", a, "rotary table")
    refused("sufhip_rotary2", rotary_args(out_head_stride=-1), "strides")
    a = rotary_args()
    a.x.token_stride = -8
    refused("sufhip_rotary2", a, "strides")
    refused("sufhip_rotary2", rotary_args(trunc=trunc(frac_bits=15)), "frac_bits")
    refused("sufhip_rotary2", rotary_args(trunc=trunc(work_bytes=8)), "work bytes")
    t = trunc()
    t.contents.add[0] = t.contents.add[1] = PTR
    refused("sufhip_rotary2", rotary_args(trunc=t), "addend")
    refused("sufhip_rotary2", rotary_args(heads=1 << 30, dim=256), "too large")
    for kw in ({"tokens": 0}, {"heads": 0}, {"dim": 0}):  # nothing to do
        assert native.load().sufhip_rotary2(ctypes.byref(rotary_args(**kw)), None) == 0


POOLS = [{"page_tokens": 12}, {"page_tokens": 0}, {"dim": 0}, {"dim": 257}, {"kv_heads": 0},
         {"pages": -1}]


def append_args():
    a = native.KvAppend2Args()
    batch(a.batch)
    for p in a.part:
        rows(p.x)
        pool(p.pool)
        p.mask[0] = p.mask[1] = PTR
    return a


def test_append2_refuses():
    refused("sufhip_kv_append2", None, "null args")
    for kw in POOLS:
        a = append_args()
        pool(a.part[1].pool, **kw)
        refused("sufhip_kv_append2", a, "pool")
    a = append_args()
    a.part[0].pool.b[1] = None
    refused("sufhip_kv_append2", a, "null pool")
    a = append_args()
    a.part[0].mask[1] = None
    refused("sufhip_kv_append2", a, "mask")
    a = append_args()
    a.part[1].x.p[1] = None
    refused("sufhip_kv_append2", a, "rows")
    for kw in ({"seqs": -1}, {"tokens": -1}, {"max_pages": -1}, {"max_new": -1}):
        a = append_args()
        batch(a.batch, **kw)
        refused("sufhip_kv_append2", a, ">= 0")
    for field in ("d_cu_tokens", "d_kv_lens", "d_pages"):
        a = append_args()
        setattr(a.batch, field, None)
        refused("sufhip_kv_append2", a, "null")
    a = append_args()
    a.part[0].rot.positions, a.part[0].rot.rot = 4, 8
    refused("sufhip_kv_append2", a, "rotary table")
    a = append_args()
    t = trunc()
    t.contents.y[0] = None  # one party's truncated shares alone
    a.part[0].trunc = t
    refused("sufhip_kv_append2", a, "truncation")
    a = append_args()
    batch(a.batch, tokens=1 << 26)
    refused("sufhip_kv_append2", a, "2^30")
    for kw in ({"seqs": 0}, {"tokens": 0}):
        a = append_args()
        batch(a.batch, **kw)
        assert native.load().sufhip_kv_append2(ctypes.byref(a), None) == 0


def product_args():
    a = native.KvProduct2Args()
    batch(a.batch)
    pool(a.pool)
    rows(a.x)
    for p in (0, 1):
        a.a[p] = a.c[p] = a.out[p] = PTR
    a.heads, a.n, a.d_row_offsets = 4, 100, PTR
    return a


@pytest.mark.parametrize("name", ["sufhip_kv_scores2", "sufhip_kv_values2"])
def test_products_refuse(name):
    refused(name, None, "null args")
    for kw in POOLS + [{"pages": 0}]:
        a = product_args()
        pool(a.pool, **kw)
        refused(name, a, "pool")
    for heads in (0, 3, -2):
        a = product_args()
        a.heads = heads
        refused(name, a, "multiple")
    for i in range(6):
        a = product_args()
        if i < 2:
            a.x.p[i] = None
        elif i < 4:
            a.a[i - 2] = None
        else:
            a.c[i - 4] = None
        refused(name, a, "null operand")
    a = product_args()
    a.d_row_offsets = None
    refused(name, a, "null operand")
    a = product_args()
    a.out[0] = None
    refused(name, a, "outputs")
    a = product_args()
    a.n = 1 << 31
    refused(name, a, "packed elements")
    a = product_args()
    a.heads, a.batch.tokens = 2 << 10, 1 << 20
    refused(name, a, "rows")
    a = product_args()
    a.batch.seqs = (1 << 21) + 1
    refused(name, a, "sequences times")
    a = product_args()
    a.trunc = trunc(frac_bits=0)
    refused(name, a, "frac_bits")
    for kw in ({"seqs": 0}, {"tokens": 0}):
        a = product_args()
        batch(a.batch, **kw)
        assert getattr(native.load(), name)(ctypes.byref(a), None) == 0


@pytest.mark.parametrize("name", ["sufhip_kv_scores2", "sufhip_kv_values2"])
def test_products_number_keys_in_32_bits(name):
    """Two chunks of 64 keys past the last one are numbered too."""
    a = product_args()
    batch(a.batch, tokens=0)
    a.n = (1 << 31) - 256
    assert getattr(native.load(), name)(ctypes.byref(a), None) == 0
    a.n += 1
    refused(name, a, "packed elements")


def test_values2_needs_its_workspace():
    lib = native.load()
    a = product_args()
    batch(a.batch, max_keys=1000)
    need = lib.sufhip_kv_values2_work_bytes(ctypes.byref(a.batch), ctypes.byref(a.pool), a.heads)
    assert need > 0
    for work, nb in ((None, need), (PTR, need - 1), (PTR + 8, need)):
        a.d_work, a.work_bytes = work, nb
        refused("sufhip_kv_values2", a, "d_work")
    assert lib.sufhip_kv_values2_work_bytes(None, ctypes.byref(a.pool), 4) == 0
    assert lib.sufhip_kv_values2_work_bytes(ctypes.byref(a.batch), None, 4) == 0
    assert lib.sufhip_kv_values2_work_bytes(ctypes.byref(a.batch), ctypes.byref(a.pool), 3) == 0


def test_values2_work_bytes_are_bounded():
    """Partial sums are two slots a workgroup, digits at most 2 GiB, also for
    bounds that no cache holds."""
    lib = native.load()
    a = product_args()
    pool(a.pool, pages=1 << 24, page_tokens=64, kv_heads=8, dim=128)

    def need(seqs, new, keys):
        batch(a.batch, seqs=seqs, tokens=seqs * new, max_new=new, max_keys=keys)
        return lib.sufhip_kv_values2_work_bytes(ctypes.byref(a.batch), ctypes.byref(a.pool), 32)

    assert need(1, 4096, 65536) == 8 * 1024 * 8 * 24576  # 24 bytes a value
    assert 0 < need(16, 1, 1 << 20) < 32 << 20
    for seqs, new, keys in ((64, 1024, 1 << 16), (1, 4096, 1 << 30), (1 << 16, 64, 2 ** 31 - 1)):
        assert need(seqs, new, keys) <= 2 << 30
    pool(a.pool, pages=16, page_tokens=64, kv_heads=8, dim=128)
    assert need(1, 4096, 65536) == 0  # more than the pool holds


def test_scores2_refuses_negative_strides():
    a = product_args()
    a.x.token_stride = -1
    refused("sufhip_kv_scores2", a, "strides")


def test_calls_refuse_host_tensors():
    x = torch.zeros(1, 1, 8, dtype=torch.int64)
    for make in (lambda: kv.Rotary(torch.zeros(4, 4, 2, dtype=torch.int32), 8),
                 lambda: kv.Pool(x[None], x[None], x[None]),
                 lambda: kv.Batch(x, x, x, 1, 1, 1)):
        with pytest.raises(ValueError, match="GPU"):
            make()


# ---- rotary tables ----

def angle(table, p, i, one):
    c, s = table[p, i]
    assert abs(math.hypot(c, s) - abs(one)) < 1.5  # two roundings of half a step
    return math.atan2(s, c)


def close(a, b, tol):
    return abs(math.remainder(a - b, 2 * math.pi)) <= tol


@pytest.mark.parametrize("rot,positions,base,frac", [(2, 5, 10000.0, 12), (64, 200, 10000.0, 20),
                                                     (48, 70000, 500000.0, 24)])
def test_table_angles(rot, positions, base, frac):
    t, one = kv.rotary_table(positions, rot, base, frac)
    assert t.dtype == np.int32 and t.shape == (positions, rot // 2, 2) and one == 1 << frac
    # A factor is off by half a step at most, an angle by less than a step's.
    for p in {0, 1, positions // 2, positions - 1}:
        for i in {0, rot // 4, rot // 2 - 1}:
            assert close(angle(t, p, i, one), p * base ** (-2.0 * i / rot), 2.0 / one)
    assert (t[0, :, 0] == one).all() and (t[0, :, 1] == 0).all()


def test_table_scaling():
    frac, rot, p = 24, 32, 3000
    one = 1 << frac
    plain = [10000.0 ** (-2.0 * i / rot) for i in range(rot // 2)]
    t, _ = kv.rotary_table(p + 1, rot, frac_bits=frac, scaling=("linear", 8))
    assert all(close(angle(t, p, i, one), p * plain[i] / 8, 2.0 / one) for i in range(rot // 2))
    t, _ = kv.rotary_table(p + 1, rot, frac_bits=frac, scaling=("base", 8))
    last = rot // 2 - 1
    assert close(angle(t, p, 0, one), p * plain[0], 2.0 / one)          # the fastest: as it was
    assert close(angle(t, p, last, one), p * plain[last] / 8, 2.0 / one)  # the slowest: by 8
    t, got = kv.rotary_table(p + 1, rot, frac_bits=frac, scaling=("parts", 8, 2048, 1, 32))
    scaled = (0.1 * math.log(8) + 1) * one
    assert got == round(scaled)
    for i in range(rot // 2):
        turns = 2048 * plain[i] / (2 * math.pi)
        keep = min(max((turns - 1) / 31, 0), 1)
        assert close(angle(t, p, i, scaled), p * (plain[i] * keep + plain[i] / 8 * (1 - keep)),
                     2.0 / one)
    same, _ = kv.rotary_table(50, rot, scaling=("parts", 1, 2048, 1, 32))
    assert np.array_equal(same, kv.rotary_table(50, rot)[0])


def test_table_scale_and_refusals():
    t, one = kv.rotary_table(9, 8, frac_bits=12, scale=-0.125)
    assert one == -512 and t[0, 0, 0] == -512
    assert kv.rotary_table(0, 8)[0].shape == (0, 4, 2) and kv.rotary_table(3, 0)[0].size == 0
    for args, kw in (((4, 7), {}), ((-1, 8), {}), ((4, 8), {"frac_bits": 0}),
                     ((4, 8), {"frac_bits": 29}), ((4, 8), {"scale": 2.0 ** 19}),
                     ((4, 8), {"scaling": ("linear", 0.5)}), ((4, 8), {"scaling": ("ramp", 2)}),
                     ((4, 8), {"scaling": ("parts", 2, 64, 4, 4)})):
        with pytest.raises(ValueError):
            kv.rotary_table(*args, **kw)


def test_causal_row_offsets():
    off = kv.causal_row_offsets([3, 1], [5, 1], 2)
    assert np.array_equal(np.diff(off), [3, 4, 5, 1] * 2) and off[0] == 0
    assert np.array_equal(np.diff(kv.causal_row_offsets([4], [2], 1)), [0, 0, 1, 2])
    assert np.array_equal(kv.causal_row_offsets([], [], 3), [0])


def test_argument_structures_match_the_header():
    """Sizes of the ctypes structures as the C compiler lays them out."""
    import os
    import subprocess
    import tempfile
    names = {"sufhip_rows2": native.Rows2, "sufhip_rotary": native.RotaryTable,
             "sufhip_rotary2_args": native.Rotary2Args, "sufhip_kv_batch": native.KvBatch,
             "sufhip_kv_pool": native.KvPool, "sufhip_kv_append_part": native.KvAppendPart,
             "sufhip_kv_append2_args": native.KvAppend2Args,
             "sufhip_kv_product2_args": native.KvProduct2Args}
    src = '#include <stdio.h>\n#include "suf_hip.h"\nint main(void) {\n' + "".join(
        '  printf("%%zu\\n", sizeof(%s));\n' % n for n in names) + "  return 0;\n}\n"
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, "s.c")
        with open(path, "w") as f:
            f.write(src)
        subprocess.run(["gcc", "-I", os.path.dirname(native.HEADER), path, "-o",
                        os.path.join(d, "s")], check=True)
        out = subprocess.run([os.path.join(d, "s")], check=True, capture_output=True, text=True)
    assert [int(v) for v in out.stdout.split()] == [ctypes.sizeof(t) for t in names.values()]
