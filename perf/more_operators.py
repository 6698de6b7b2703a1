"""What the parts of a decoder around its attention cost, for both parties on one
GPU: the root-mean-square norm of the residual stream, products with public
weights for any number of tokens, products grouped by expert, and the weighted
sum of the experts' outputs.

Inputs are additive shares mod 2^64 of fixed-point numbers with F fractional
bits.  A truncation gate's output shares depend on its keys, but their sum is the
exact floor of the value, so a pass returns opened sums (what a program that
reveals the result computes) and the kernels and the plain forms agree bit for
bit.  What is local to a party (the residual stream's sum) comes as its shares.

With >> the floor of a division by a power of two, kinds of cases (field
"kind"):
  norm     s = x + residual;  v = ((((sum s s) >> F) inv) >> 26) + eps with inv =
           round(2^26 / cols);  y = 1 / sqrt(v) from a table's chord and one
           Newton step;  out = (s y) >> F, with a weight (out weight) >> F
  linear   out = act((x W + bias) >> F) + residual; "after_norm": x is a norm's
           output, handed over as 8-bit digits
  experts  row i of out = act((x[rows[i]] W[e] + bias[e]) >> F) for the rows i of
           expert e, [offsets[e], offsets[e + 1])
  mix      out[t] = ((sum_k weights[t, k] z[slots[t, k]]) >> F) + residual[t]
act: nothing, "relu", or "gelu" as a table of cubics.
"""
import math

import numpy as np
import torch

own = False

F = 12            # fractional bits of values and factors
LEN_BITS = 26     # of a norm's 1 / cols
EPS = 4           # a norm's epsilon, 2^-10
STATE = bytes(range(1, 129))  # the PRG state that both parties and the dealer share
TOP = -2 ** 63


def listed():
    return [
        # One token's residual stream at GPT-2-small's width: every step of a
        # dialogue, twice a layer.  Latency decides.
        {"name": "norm_token", "kind": "norm", "rows": 1, "cols": 768, "residual": True,
         "weight": False},
        # One token each of 32 dialogues, a wide model with a learned weight.
        {"name": "norm_batch", "kind": "norm", "rows": 32, "cols": 4096, "residual": True,
         "weight": True},
        # Packed prompts.
        {"name": "norm_prompt", "kind": "norm", "rows": 1999, "cols": 2048, "residual": True,
         "weight": True},
        # One token's queries, keys and values at GPT-2-small's sizes.
        {"name": "linear_token", "kind": "linear", "rows": 1, "k": 768, "n": 2304, "bits": 12,
         "bias": True, "act": "", "residual": False, "after_norm": False, "view": False},
        # One token each of 16 dialogues through a square projection back to
        # the residual stream; x is a part of wider rows.
        {"name": "linear_batch", "kind": "linear", "rows": 16, "k": 4096, "n": 4096, "bits": 13,
         "bias": False, "act": "", "residual": True, "after_norm": False, "view": True},
        # One token's logits over a vocabulary.
        {"name": "linear_logits", "kind": "linear", "rows": 1, "k": 2048, "n": 32000, "bits": 13,
         "bias": False, "act": "", "residual": False, "after_norm": False, "view": False},
        # A prompt through the first product of a GELU network.
        {"name": "linear_gelu", "kind": "linear", "rows": 512, "k": 1024, "n": 4096, "bits": 12,
         "bias": True, "act": "gelu", "residual": False, "after_norm": False, "view": False},
        # A prompt's norm and the product that reads it.
        {"name": "linear_prompt", "kind": "linear", "rows": 1000, "k": 2048, "n": 1024,
         "bits": 13, "bias": True, "act": "", "residual": False, "after_norm": True,
         "view": False},
        # One token each of 8 dialogues, two of eight experts each.
        {"name": "experts_tokens", "kind": "experts", "tokens": 8, "each": 2, "experts": 8,
         "k": 1024, "n": 2048, "bits": 12, "bias": False, "act": "relu"},
        # A prompt over 16 experts, some of them far more popular than others.
        {"name": "experts_prompt", "kind": "experts", "tokens": 1000, "each": 2, "experts": 16,
         "k": 1024, "n": 2048, "bits": 12, "bias": True, "act": ""},
        {"name": "mix_tokens", "kind": "mix", "tokens": 8, "each": 2, "cols": 1024,
         "residual": True},
        {"name": "mix_prompt", "kind": "mix", "tokens": 1000, "each": 2, "cols": 2048,
         "residual": True},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "linear", "linear", "experts", "mix"])
    if kind == "norm":
        cols = _spread(rng, 33, 8192)
        return {"kind": kind, "rows": _spread(rng, 1, max(1, min(4096, 3000000 // cols))),
                "cols": cols, "residual": rng.random() < 0.7, "weight": rng.random() < 0.5}
    if kind == "mix":
        cols = _spread(rng, 32, 4096)
        return {"kind": kind, "tokens": _spread(rng, 1, max(1, min(2000, 2000000 // cols))),
                "each": rng.choice([1, 2, 2, 3, 4, 8]), "cols": cols,
                "residual": rng.random() < 0.5}
    k = _spread(rng, 48, 4096)
    if kind == "linear":
        n = _spread(rng, 40, 12000)
        rows = _spread(rng, 1, max(1, min(1200, 1500000000 // (k * n))))
        act = rng.choice(["", "", "relu", "gelu"])
        if act == "gelu":
            rows = max(1, min(rows, 1500000 // n))
        return {"kind": kind, "rows": rows, "k": k, "n": n, "bits": rng.choice([7, 12, 13, 15, 20]),
                "bias": rng.random() < 0.5, "act": act, "residual": rng.random() < 0.5,
                "after_norm": rng.random() < 0.3, "view": rng.random() < 0.3}
    k, n = min(k, 2048), _spread(rng, 40, 3000)
    each, experts = rng.choice([1, 2, 2, 4]), rng.choice([4, 7, 8, 16, 33, 64])
    tokens = _spread(rng, 1, max(1, min(1000, 1500000000 // (each * k * n))))
    return {"kind": kind, "tokens": tokens, "each": each, "experts": experts, "k": k, "n": n,
            "bits": rng.choice([7, 12, 13]), "bias": rng.random() < 0.5,
            "act": rng.choice(["", "relu"])}


# ---- public tables (what a model's program keeps) ----

def _fixed(v):
    return int(math.floor(abs(v) * 2 ** F + 0.5)) * (1 if v >= 0 else -1)


def _rsqrt_table():
    """1 / sqrt on [2^-10, 4096) as words (c0, c1) of c0 + c1 v: chords of an
    octave up to 16, then constants on quarters of one."""
    rows = [(0, _fixed(32.0), 0)]
    lo = 2.0 ** -10
    while lo < 16:
        y0, y1 = lo ** -0.5, (2 * lo) ** -0.5
        c1 = _fixed((y1 - y0) / lo)
        rows.append((_fixed(lo), _fixed(y0) - ((c1 * _fixed(lo)) >> F), c1))
        lo *= 2
    while lo < 4096:
        a, b = lo, lo * 2 ** 0.25
        rows.append((_fixed(a), _fixed(0.5 * (a ** -0.5 + b ** -0.5)), 0))
        lo = b if _fixed(b) < _fixed(4096.0) - 1 else 4096.0
    rows.append((_fixed(4096.0), _fixed(1 / 64), 0))
    return (np.array([r[0] for r in rows], dtype=np.uint64),
            np.array([r[1:] for r in rows], dtype=np.int64))


def _gelu_table():
    """x Phi(x) on pieces of one unit of [-8, 8), cubics in x; 0 below, x above.
    Pieces in the unsigned order of their starts."""
    def value(x):
        return 0.5 * x * (1 + math.erf(x / math.sqrt(2)))

    def slope(x):
        return (0.5 * (1 + math.erf(x / math.sqrt(2))) +
                x * math.exp(-0.5 * x * x) / math.sqrt(2 * math.pi))

    rows = [(8, [0, 1, 0, 0]), (-(1 << (63 - F)), [0, 0, 0, 0])]
    for x0 in range(-8, 8):
        y0, y1, m0, m1 = value(x0), value(x0 + 1), slope(x0), slope(x0 + 1)
        c = [y0, m0, 3 * (y1 - y0) - 2 * m0 - m1, 2 * (y0 - y1) + m0 + m1]
        # in (x - x0) -> in x
        rows.append((x0, [c[0] - c[1] * x0 + c[2] * x0 ** 2 - c[3] * x0 ** 3,
                          c[1] - 2 * c[2] * x0 + 3 * c[3] * x0 ** 2, c[2] - 3 * c[3] * x0, c[3]]))
    rows.sort(key=lambda r: (r[0] << F) % 2 ** 64)
    return (np.array([(r[0] << F) % 2 ** 64 for r in rows], dtype=np.uint64),
            np.array([[_fixed(v) for v in r[1]] for r in rows], dtype=np.int64))


def _on_gpu(table):
    """Starts (their unsigned order as the signed one) and words."""
    return (torch.from_numpy(table[0].view(np.int64)).cuda() ^ TOP,
            torch.from_numpy(table[1]).cuda())


# ---- inputs ----

def _values(gen, *shape, sigma=1.0):
    return torch.round(torch.randn(*shape, device="cuda", generator=gen) *
                       (sigma * 2 ** F)).to(torch.int64)


def _shared(gen, v):
    """Shares of v: a uniform word and the rest."""
    s = torch.randint(TOP, 2 ** 63 - 1, v.shape, dtype=torch.int64, device="cuda", generator=gen)
    return s, v - s


def _empty(*shape):
    return tuple(torch.empty(*shape, dtype=torch.int64, device="cuda") for _ in range(2))


def _matrix(gen, case, *shape):
    """Weights of at most `bits` bits and a sign, and biases in the product's
    scale."""
    w = torch.randn(*shape, device="cuda", generator=gen) * 2.0 ** (case["bits"] - 2)
    lim = 2 ** case["bits"] - 1
    bias = None
    if case["bias"]:
        bias = _values(gen, *shape[:-2], shape[-1]) << F
    return torch.round(w).clamp(-lim, lim).to(torch.int64), bias


def _routing(host, case):
    """Per token its experts (all different), and from them the rows sorted by
    expert: where each expert's begin, the token of each, and each token's
    rows."""
    T, E, each = case["tokens"], case["experts"], min(case["each"], case["experts"])
    likes = host.random((T, E)) ** np.linspace(1.0, 4.0, E)  # the last ones are rare
    chosen = np.argsort(-likes, axis=1)[:, :each]
    flat = chosen.ravel()
    order = np.argsort(flat, kind="stable")
    counts = np.bincount(flat, minlength=E)
    slots = np.empty(T * each, np.int64)
    slots[order] = np.arange(T * each)
    return counts, order // each, slots.reshape(T, each)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    host = np.random.default_rng(seed)
    kind, st = case["kind"], {"case": case}
    if kind == "norm" or case.get("after_norm"):
        rows, cols = case["rows"], case["cols"] if kind == "norm" else case["k"]
        st["x"] = _shared(gen, _values(gen, rows, cols))
        res = case["residual"] if kind == "norm" else True
        st["r"] = _shared(gen, _values(gen, rows, cols)) if res else None
        w = kind == "norm" and case["weight"]
        st["g"] = (1 << F) + _values(gen, cols, sigma=0.2) if w else None
        st["total"], st["out"] = _empty(rows, cols) if res else None, _empty(rows, cols)
        st["rsqrt"] = _rsqrt_table()
        st["rsqrt_table"] = _on_gpu(st["rsqrt"])
    if kind == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        if not case["after_norm"]:
            wide = k + 96 if case["view"] else k
            st["x"] = tuple(t[:, wide - k:] for t in _shared(gen, _values(gen, rows, wide)))
        st["W"], st["bias"] = _matrix(gen, case, k, n)
        st["res"] = _shared(gen, _values(gen, rows, n)) if case["residual"] else None
        st["y"] = _empty(rows, n)
    elif kind == "experts":
        counts, rows, _ = _routing(host, case)
        st["counts"] = [int(c) for c in counts]
        st["rows"], st["offsets"] = _i32(rows), _i32(np.concatenate([[0], np.cumsum(counts)]))
        st["x"] = _shared(gen, _values(gen, case["tokens"], case["k"]))
        st["W"], st["bias"] = _matrix(gen, case, case["experts"], case["k"], case["n"])
        st["y"] = _empty(len(rows), case["n"])
    elif kind == "mix":
        T, each, cols = case["tokens"], case["each"], case["cols"]
        st["z"] = _shared(gen, _values(gen, T * each, cols))
        st["slots"] = _i32(host.permutation(T * each).reshape(T, each))
        w = host.random((T, each))
        st["weights"] = torch.from_numpy(
            np.rint(w / w.sum(1, keepdims=True) * 2 ** F).astype(np.int64)).cuda()
        st["res"] = _shared(gen, _values(gen, T, cols)) if case["residual"] else None
        st["y"] = _empty(T, cols)
    st["act"] = case.get("act") or None
    if st["act"] == "gelu":
        st["act"] = _gelu_table()
        st["act_table"] = _on_gpu(st["act"])
    if own:
        _own_handles(case, st, seed)
    return st


def _own_handles(case, st, seed):
    from suf_amd import feedforward as ff
    if "rsqrt" in st:
        st["norm"] = ff.RMSNorm(*st["x"][0].shape, STATE, weight=st["g"], table=st["rsqrt"],
                                seed=seed)
    if "W" in st:
        weights = ff.PublicWeights(st["W"], st["bias"])
        st["linear"] = ff.Linear(weights, st["y"][0].shape[0], STATE, act=st["act"],
                                 seed=seed + 1)
        if case.get("after_norm"):
            st["digits"] = ff.Digits(*st["x"][0].shape)
    if case["kind"] == "mix":
        st["mix"] = ff.ExpertMix(case["tokens"], case["cols"], STATE, seed=seed)


# ---- a pass ----

def run(st):
    kind, case = st["case"]["kind"], st["case"]
    if kind == "norm":
        if own:
            st["norm"].eval2(st["x"], st["out"], residual=st["r"], total=st["total"])
            out = st["out"][0] + st["out"][1]
        else:
            total, out = _plain_norm(st)
            if st["r"] is not None:
                for t, v in zip(st["total"], total):
                    t.copy_(v)
        return (out,) if st["r"] is None else (out,) + st["total"]
    if kind == "mix":
        if own:
            y = st["mix"].eval2(st["z"], st["slots"], st["weights"], st["y"], residual=st["res"])
            return y[0] + y[1]
        return _plain_mix(st)
    if own:
        x = st["x"]
        if case.get("after_norm"):
            st["norm"].eval2(x, None, residual=st["r"], total=st["total"], digits=st["digits"])
            x = st["digits"]
        if kind == "experts":
            y = st["linear"].eval2(x, st["y"], offsets=st["offsets"], rows=st["rows"])
        else:
            y = st["linear"].eval2(x, st["y"], residual=st["res"])
        out = y[0] + y[1]
        return (out,) + st["total"] if case.get("after_norm") else out
    if kind == "experts":
        return _plain_experts(st)
    if case["after_norm"]:
        total, x = _plain_norm(st)
        for t, v in zip(st["total"], total):
            t.copy_(v)
        return (_plain_linear(st, x),) + st["total"]
    return _plain_linear(st, st["x"][0] + st["x"][1])


# ---- plain forms ----

def _coeffs(v, table):
    """The words of the piece that holds v, in unsigned order."""
    starts, words = table
    return words[torch.bucketize(v ^ TOP, starts, right=True) - 1].unbind(-1)


def _plain_norm(st):
    x, r = st["x"], st["r"]
    s = x if r is None else (x[0] + r[0], x[1] + r[1])
    v = s[0] + s[1]
    inv = (2 ** (LEN_BITS + 1) // v.shape[1] + 1) // 2
    ms = ((((v * v).sum(1) >> F) * inv) >> LEN_BITS) + EPS
    c0, c1 = _coeffs(ms, st["rsqrt_table"])
    y = ((c1 * ms) >> F) + c0
    h = (ms * ((y * y) >> F)) >> (F + 1)
    y = (y * ((3 << (F - 1)) - h)) >> F
    out = (v * y[:, None]) >> F
    return s, out if st["g"] is None else (out * st["g"]) >> F


def _product(x, w):
    """x @ w for int64 (exact mod 2^64)."""
    step = max(1, (1 << 27) // max(1, w.numel()))
    return torch.cat([(x[i:i + step, :, None] * w[None]).sum(1)
                      for i in range(0, x.shape[0], step)]) if x.shape[0] else x @ w


def _activate(y, st):
    if st["act"] is None:
        return y
    if st["act"] == "relu":
        return torch.where(y > 0, y, 0)
    c0, c1, c2, c3 = _coeffs(y, st["act_table"])
    t = ((c3 * y + (c2 << F)) * y) >> F
    t = ((t + (c1 << F)) * y) >> F
    return (t + (c0 << F)) >> F


def _plain_linear(st, x):
    y = _product(x, st["W"])
    if st["bias"] is not None:
        y = y + st["bias"]
    y = _activate(y >> F, st)
    return y if st["res"] is None else y + st["res"][0] + st["res"][1]


def _plain_experts(st):
    x, rows, out, at = st["x"][0] + st["x"][1], st["rows"].long(), [], 0
    for e, n in enumerate(st["counts"]):
        if n:
            y = _product(x[rows[at:at + n]], st["W"][e])
            out.append(y if st["bias"] is None else y + st["bias"][e])
        at += n
    return _activate(torch.cat(out) >> F, st)


def _plain_mix(st):
    z = st["z"][0] + st["z"][1]
    y = (z[st["slots"].long()] * st["weights"][:, :, None]).sum(1) >> F
    return y if st["res"] is None else y + st["res"][0] + st["res"][1]


# ---- what a pass cannot do without ----

def _norm_work(rows, cols, residual, weight):
    """Both parties' words of an element: x, a mask and its product with the
    row's factor, the output; the residual and the sum."""
    n = rows * cols
    return {"bytes": 8 * n * (8 + 4 * residual) + 8 * cols * weight + 8 * rows * 40,
            "flops": 2 * n * (8 + 2 * weight)}


def work(case):
    kind = case["kind"]
    if kind == "norm":
        return _norm_work(case["rows"], case["cols"], case["residual"], case["weight"])
    if kind == "mix":
        n = case["tokens"] * case["cols"]
        return {"bytes": 16 * n * (case["each"] + 1 + case["residual"]) +
                12 * case["tokens"] * case["each"], "flops": 4 * n * case["each"]}
    k, n = case["k"], case["n"]
    each = 16 if case["act"] != "gelu" else 16 + 144  # triples of three products
    weight_bytes = -(-(case["bits"] + 1) // 8)
    if kind == "linear":
        rows, used, x = case["rows"], 1, case["rows"]
        each += 16 * case["residual"]
    else:
        rows = case["tokens"] * min(case["each"], case["experts"])
        used, x = min(case["experts"], rows), case["tokens"]
    got = {"bytes": 16 * x * k + weight_bytes * k * n * used + each * rows * n +
           8 * n * used * case["bias"], "flops": 2 * 2 * rows * k * n}
    if case.get("after_norm"):  # the normalised values are nobody's output
        more = _norm_work(rows, k, True, False)
        got = {"bytes": got["bytes"] + more["bytes"] - 32 * rows * k,
               "flops": got["flops"] + more["flops"]}
    return got


# ---- the definition on the host ----

def _host(t):
    return t.detach().cpu().numpy().view(np.uint64)


def _floor(a, bits):
    return (a.view(np.int64) >> np.int64(bits)).view(np.uint64)


def _matmul(x, w):
    """x w mod 2^64: 16-bit limbs of x against signed weights of at most 2^20 in
    float64 (sums below 2^16 2^20 2^13 < 2^53, whole numbers)."""
    out = np.zeros((x.shape[0], w.shape[1]), np.uint64)
    for i in range(4):
        limb = ((x >> np.uint64(16 * i)) & np.uint64(0xffff)).astype(np.float64)
        out += (limb @ w).astype(np.int64).view(np.uint64) << np.uint64(16 * i)
    return out


def _pieces(v, table):
    at = np.searchsorted(table[0], v, side="right") - 1
    return [c.view(np.uint64) for c in np.moveaxis(table[1][at], -1, 0).copy()]


def _exact_norm(st):
    s = [_host(x) + (0 if st["r"] is None else _host(r))
         for x, r in zip(st["x"], st["r"] or st["x"])]
    v = s[0] + s[1]
    square = np.einsum("ij,ij->i", v, v)
    inv = np.uint64(int(math.floor(2.0 ** LEN_BITS / v.shape[1] + 0.5)))
    ms = _floor(_floor(square, F) * inv, LEN_BITS) + np.uint64(EPS)
    c0, c1 = _pieces(ms, st["rsqrt"])
    y = _floor(c1 * ms, F) + c0
    half = _floor(_floor(ms * _floor(y * y, F), F), 1)
    y = _floor(y * (np.uint64(3 << (F - 1)) - half), F)
    out = _floor(v * y[:, None], F)
    return s, out if st["g"] is None else _floor(out * _host(st["g"]), F)


def _exact_act(y, act):
    if act is None:
        return y
    if act == "relu":
        return np.where(y >> np.uint64(63), np.uint64(0), y)
    c = _pieces(y, act)
    t = _floor((c[3] * y + (c[2] << np.uint64(F))) * y, F)
    t = _floor((t + (c[1] << np.uint64(F))) * y, F)
    return _floor(t + (c[0] << np.uint64(F)), F)


def _signed(a):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int64))


def exact(case, seed):
    st = prepare(case, seed)
    with np.errstate(over="ignore"):
        if case["kind"] == "norm":
            s, out = _exact_norm(st)
            return tuple(_signed(a) for a in ([out] if st["r"] is None else [out] + s))
        res = 0 if st.get("res") is None else _host(st["res"][0]) + _host(st["res"][1])
        if case["kind"] == "mix":
            z, w = _host(st["z"][0]) + _host(st["z"][1]), _host(st["weights"])
            y = np.zeros((case["tokens"], case["cols"]), np.uint64)
            for k, rows in enumerate(st["slots"].cpu().numpy().T):
                y += z[rows] * w[:, k:k + 1]
            return _signed(_floor(y, F) + res)
        s = None
        if case.get("after_norm"):
            s, x = _exact_norm(st)
        else:
            x = _host(st["x"][0]) + _host(st["x"][1])
        w = st["W"].cpu().numpy().astype(np.float64)
        if case["kind"] == "experts":
            rows, off = st["rows"].cpu().numpy(), st["offsets"].cpu().numpy()
            parts = [_matmul(x[rows[off[e]:off[e + 1]]], w[e]) +
                     (0 if st["bias"] is None else _host(st["bias"])[e])
                     for e in range(case["experts"])]
            y = np.concatenate(parts)
        else:
            y = _matmul(x, w) + (0 if st["bias"] is None else _host(st["bias"]))
        y = _exact_act(_floor(np.ascontiguousarray(y), F), st["act"]) + res
        return _signed(y) if s is None else tuple(_signed(a) for a in [y] + s)
