"""What attention over a cache of secret-shared keys and values costs: the
rotary positions, the append to the paged cache and the two products of a
decoder's attention, for both parties on one GPU.

Every value is an integer mod 2^64 (additive shares, masked opens, public
fixed-point factors), so the kernels and the plain forms agree bit for bit.

Shares are uniform words.  So are masks, opens and triple shares, whatever the
values behind them: every input but the angles, lengths and tables is drawn
uniformly.

Kinds of cases (field "kind"):
  rotary   queries or keys of packed tokens, rotated by their positions with a
           public fixed-point table: per pair (u, v) of a head's values
           u' = u c - v s, v' = u s + v c; the values past the rotated part
           times pass_mul
  append   keys (rotated) and values of new tokens into the pages of their
           sequences: the pages keep the opened difference E = value - mask
           and each party's share of the mask
  scores   queries times cached keys, ragged rows: party p's share of
           score(t, h, j) is C_p + sum_i D B_p + (A_p + [p = 0] D) E with
           D = q - A opened on the way
  values   ragged rows of probabilities times cached values: the same form
           summed over the row's keys

Row (h, t) of scores and probabilities (query head h, token t) starts at
offsets[h * tokens + t] and holds the first offsets[h * tokens + t + 1] -
offsets[h * tokens + t] keys of its token's sequence.  Of a case, "new" are the
new tokens of each sequence and "past" the cached ones before them.
"""
import math

import numpy as np
import torch

own = False

FC = 12  # fractional bits of the rotary table
BASE = 10000.0
# A serving batch: 16 dialogues of ragged lengths.
ONE_EACH = "1 1 1 1 1 1 1 1 1 1 1 1 1 1 1 1"
PASTS = "4095 2047 511 3000 1 4000 1777 2500 900 64 3333 2222 1111 128 4001 3500"


def listed():
    return [
        # One token's queries at GPT-2-small's head sizes: the call of every
        # step of a dialogue.  Latency decides.
        {"name": "rotary_token", "kind": "rotary", "tokens": 1, "heads": 12, "dim": 64, "rot": 64,
         "interleaved": False, "far": 2048, "view": False},
        # The queries of packed prompts, read as a view of the rows of a
        # fused query, key and value product.
        {"name": "rotary_prompt", "kind": "rotary", "tokens": 2048, "heads": 32, "dim": 128,
         "rot": 128, "interleaved": False, "far": 8192, "view": True},
        # A part of an odd head rotated, neighbours paired, far positions.
        {"name": "rotary_part_far", "kind": "rotary", "tokens": 1021, "heads": 16, "dim": 80,
         "rot": 32, "interleaved": True, "far": 131072, "view": False},
        # One new token each of eight dialogues.
        {"name": "append_tokens", "kind": "append", "new": "1 1 1 1 1 1 1 1",
         "past": "37 512 0 200 999 63 64 301", "kv_heads": 12, "dim": 64, "page": 16,
         "rot": 64, "interleaved": False},
        # Packed prompts of ragged lengths, one of them continued.
        {"name": "append_prompts", "kind": "append", "new": "1500 777 1 301",
         "past": "0 0 850 40", "kv_heads": 8, "dim": 128, "page": 64, "rot": 128,
         "interleaved": False},
        # One token of one dialogue, as many cached heads as query heads.
        {"name": "scores_token", "kind": "scores", "new": "1", "past": "299", "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 16},
        # A serving batch: one token of each of 16 dialogues of different
        # lengths, four query heads to a cached head.
        {"name": "scores_batch", "kind": "scores", "new": ONE_EACH, "past": PASTS, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64},
        # Packed prompts, one after a cached past, three query heads to a
        # cached head.
        {"name": "scores_prompts", "kind": "scores", "new": "1024 517 33", "past": "0 200 0",
         "heads": 12, "kv_heads": 4, "dim": 64, "page": 32},
        {"name": "values_token", "kind": "values", "new": "1", "past": "299", "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 16},
        {"name": "values_batch", "kind": "values", "new": ONE_EACH, "past": PASTS, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64},
        {"name": "values_prompts", "kind": "values", "new": "1024 517 33", "past": "0 200 0",
         "heads": 12, "kv_heads": 4, "dim": 64, "page": 32},
        # One token of one long document: few rows, a long sum.
        {"name": "values_long", "kind": "values", "new": "1", "past": "65535", "heads": 8,
         "kv_heads": 2, "dim": 128, "page": 64},
    ]


def _counts(text):
    return [int(v) for v in text.split()]


def _text(counts):
    return " ".join(str(v) for v in counts)


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "scores", "values"])
    dim = rng.choice([32, 40, 64, 72, 80, 96, 128])
    if kind == "rotary":
        heads = rng.choice([1, 4, 5, 8, 12, 16, 32])
        tokens = _spread(rng, 1, 2048 * 32 * 128 // (heads * dim) // 2)
        return {"kind": kind, "tokens": min(tokens, 4096), "heads": heads, "dim": dim,
                "rot": 2 * rng.randint(4, dim // 2), "interleaved": rng.random() < 0.5,
                "far": _spread(rng, 512, 131072), "view": rng.random() < 0.5}
    page = rng.choice([1, 8, 16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    if kind == "append":
        new = [_spread(rng, 1, 600) for _ in range(rng.randint(1, 4))]
        return {"kind": kind, "new": _text(new),
                "past": _text([rng.randint(0, 700) for _ in new]), "kv_heads": kv_heads,
                "dim": dim, "page": page, "rot": 2 * rng.randint(0, dim // 2),
                "interleaved": rng.random() < 0.5}
    group = rng.choice([1, 2, 3, 4, 7, 8])
    form = rng.choice(["tokens", "few", "prompts", "long"])
    if form == "tokens":  # one token each
        past = [_spread(rng, 1, 3000) for _ in range(rng.randint(1, 10))]
        new = [1] * len(past)
    elif form == "few":  # a few tokens each: a draft checked at once
        past = [_spread(rng, 1, 2000) for _ in range(rng.randint(1, 5))]
        new = [rng.randint(2, 12) for _ in past]
    elif form == "prompts":
        new = [_spread(rng, 2, 500) for _ in range(rng.randint(1, 3))]
        past = [rng.choice([0, 0, 5, 200]) for _ in new]
        kv_heads, group = min(kv_heads, 3), min(group, 3)
    else:
        new, past = [1], [_spread(rng, 5000, 30000)]
        kv_heads = min(kv_heads, 2)
    return {"kind": kind, "new": _text(new), "past": _text(past), "heads": kv_heads * group,
            "kv_heads": kv_heads, "dim": dim, "page": page}


def _words(gen, *shape):
    return torch.randint(-2 ** 63, 2 ** 63 - 1, shape, dtype=torch.int64, device="cuda",
                         generator=gen)


def _pair(gen, *shape):
    return _words(gen, *shape), _words(gen, *shape)


def _table(far, rot):
    """[far][rot / 2][cos, sin] in Q(FC), int32."""
    freq = BASE ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
    ang = np.arange(far, dtype=np.float64)[:, None] * freq
    t = np.stack([np.cos(ang), np.sin(ang)], -1) * (1 << FC)
    return torch.from_numpy(np.rint(t).astype(np.int32)).cuda()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _prepare_rotary(case, gen, host):
    T, H, dim, rot = (case[k] for k in ("tokens", "heads", "dim", "rot"))
    if case["view"]:  # the queries' part of [tokens][heads + 2 kv_heads][dim] rows
        rows = _pair(gen, T, H + 2 * max(1, H // 4), dim)
        x = tuple(r[:, :H] for r in rows)
    else:
        x = _pair(gen, T, H, dim)
    start = host.integers(0, max(1, case["far"] - T + 1))
    pos = (start + np.arange(T)) % case["far"]
    return {"x": x, "positions": _i32(pos), "table": _table(case["far"], rot),
            "out": tuple(torch.empty(T, H, dim, dtype=torch.int64, device="cuda")
                         for _ in range(2))}


def _prepare_batch(case, host):
    """The packed new tokens, the sequences' whole lengths and their pages: a
    pool with as many pages again as the batch holds, in no order."""
    new = np.array(_counts(case["new"]))
    lens = new + np.array(_counts(case["past"]))
    need = -(-lens // case["page"])
    width = int(need.max())
    pages = int(need.sum()) * 2
    order = host.permutation(pages)
    table = np.full((len(new), width), -1)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return {"new": [int(v) for v in new], "lens": [int(v) for v in lens],
            "cu": _i32(np.concatenate([[0], np.cumsum(new)])), "kv_lens": _i32(lens),
            "pages": _i32(table), "pool_pages": pages, "tokens": int(new.sum())}


def _pool(gen, case, st):
    """An opened difference and both parties' mask shares, [pages][kv_heads]
    [page tokens][dim]."""
    return tuple(_words(gen, st["pool_pages"], case["kv_heads"], case["page"], case["dim"])
                 for _ in range(3))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    host = np.random.default_rng(seed)
    if case["kind"] == "rotary":
        st = _prepare_rotary(case, gen, host)
    else:
        st = _prepare_batch(case, host)
        T, Hk, dim = st["tokens"], case["kv_heads"], case["dim"]
        if case["kind"] == "append":
            st["k_pool"], st["v_pool"] = _pool(gen, case, st), _pool(gen, case, st)
            rows = _pair(gen, T, 3 * Hk, dim)  # the rows of a fused product
            st["k"] = tuple(r[:, Hk:2 * Hk] for r in rows)
            st["v"] = tuple(r[:, 2 * Hk:] for r in rows)
            st["k_mask"], st["v_mask"] = _pair(gen, T, Hk, dim), _pair(gen, T, Hk, dim)
            st["table"] = _table(max(st["lens"]), case["rot"])
        else:
            H = case["heads"]
            rows = np.concatenate([np.arange(L - n + 1, L + 1)
                                   for n, L in zip(st["new"], st["lens"])])
            off = np.concatenate([[0], np.cumsum(np.tile(rows, H))])
            n = int(off[-1])
            st["n"], st["offsets"] = n, _i32(off)
            st["pool"] = _pool(gen, case, st)
            if case["kind"] == "scores":
                st["x"], st["a"], st["c"] = (_pair(gen, T, H, dim), _pair(gen, T, H, dim),
                                             _pair(gen, n))
                st["out"] = tuple(torch.empty(n, dtype=torch.int64, device="cuda")
                                  for _ in range(2))
            else:
                st["x"], st["a"], st["c"] = _pair(gen, n), _pair(gen, n), _pair(gen, T, H, dim)
                st["out"] = tuple(torch.empty(T, H, dim, dtype=torch.int64, device="cuda")
                                  for _ in range(2))
    st["case"] = case
    if own:
        from suf_amd import kv_attention as kv
        if case["kind"] in ("rotary", "append"):
            st["rotary"] = kv.Rotary(st["table"], case["dim"], interleaved=case["interleaved"],
                                     pass_mul=1 << FC)
        if case["kind"] != "rotary":
            st["batch"] = kv.Batch(st["cu"], st["kv_lens"], st["pages"], tokens=st["tokens"],
                                   max_new=max(st["new"]), max_keys=max(st["lens"]))
    return st


def run(st):
    kind = st["case"]["kind"]
    if own:
        from suf_amd import kv_attention as kv
        if kind == "rotary":
            return kv.rotary2(st["x"], st["rotary"], st["positions"], st["out"])
        if kind == "append":
            kv.append2(st["batch"], kv.Pool(*st["k_pool"]), st["k"], st["k_mask"],
                       v_pool=kv.Pool(*st["v_pool"]), v=st["v"], v_mask=st["v_mask"],
                       rotary=st["rotary"])
            return st["k_pool"] + st["v_pool"]
        op = kv.scores2 if kind == "scores" else kv.values2
        return op(st["batch"], kv.Pool(*st["pool"]), st["x"], st["a"], st["c"], st["offsets"],
                  st["out"])
    return {"rotary": _plain_rotary, "append": _plain_append, "scores": _plain_scores,
            "values": _plain_values}[kind](st)


# ---- plain forms ----

def _rotate(x, table, positions, interleaved):
    """x [tokens, heads, dim] int64, rotated by the table's rows."""
    cs = table[positions.long()].long()[:, None]  # [tokens, 1, rot / 2, 2]
    c, s = cs[..., 0], cs[..., 1]
    half = c.shape[-1]
    if interleaved:
        u, v = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([u * c - v * s, u * s + v * c], -1).flatten(-2)
    else:
        u, v = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([u * c - v * s, u * s + v * c], -1)
    return torch.cat([turned, x[..., 2 * half:] * (1 << FC)], -1)


def _plain_rotary(st):
    for p in range(2):
        st["out"][p].copy_(_rotate(st["x"][p], st["table"], st["positions"],
                                   st["case"]["interleaved"]))
    return st["out"]


def _token_places(st):
    """Per new token: its position in its sequence, its page, its place there."""
    new = torch.tensor(st["new"], device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(st["new"]), device="cuda"), new,
                                  output_size=st["tokens"])
    at = torch.arange(st["tokens"], device="cuda")
    pos = st["kv_lens"].long()[seq] - st["cu"].long()[seq + 1] + at
    size = st["case"]["page"]
    return pos, st["pages"].long()[seq, pos // size], pos % size


def _plain_append(st):
    pos, page, slot = _token_places(st)
    k = [_rotate(st["k"][p], st["table"], pos, st["case"]["interleaved"]) for p in range(2)]
    for (e, b0, b1), x, m in ((st["k_pool"], k, st["k_mask"]),
                              (st["v_pool"], st["v"], st["v_mask"])):
        e[page, :, slot] = x[0] + x[1] - m[0] - m[1]
        b0[page, :, slot] = m[0]
        b1[page, :, slot] = m[1]
    return st["k_pool"] + st["v_pool"]


def _cached(st, s, which):
    """Sequence s's part of a pool as [kv_heads, length, dim]."""
    L, size = st["lens"][s], st["case"]["page"]
    ids = st["pages"][s, :-(-L // size)].long()
    pool = st["pool"][which]
    return pool[ids].transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :L]


def _chunks(rows, per_row):
    step = max(1, (1 << 27) // max(1, per_row))
    return [(r, min(rows, r + step)) for r in range(0, rows, step)]


def _row_mask(n, L):
    """[n, L]: token r of n new ones sees the keys up to its own."""
    return (torch.arange(L, device="cuda")[None] <=
            (L - n + torch.arange(n, device="cuda"))[:, None])


def _packed(st, s):
    """Per query head, where sequence s's rows lie in the packed order (they
    are neighbours)."""
    T, off = st["tokens"], st["offsets"].long()
    t0 = sum(st["new"][:s])
    first = off[torch.arange(st["case"]["heads"], device="cuda") * T + t0]
    n, L = st["new"][s], st["lens"][s]
    size = n * L - n * (n - 1) // 2
    return first[:, None] + torch.arange(size, device="cuda")


def _plain_scores(st):
    case = st["case"]
    H, Hk, dim = case["heads"], case["kv_heads"], case["dim"]
    D = st["x"][0] + st["x"][1] - st["a"][0] - st["a"][1]
    left = (st["a"][0] + D, st["a"][1])
    t0 = 0
    for s, n in enumerate(st["new"]):
        L = st["lens"][s]
        E = _cached(st, s, 0)
        mask, place = _row_mask(n, L), _packed(st, s)
        for p in range(2):
            B = _cached(st, s, 1 + p)
            full = torch.empty(H, n, L, dtype=torch.int64, device="cuda")
            for r0, r1 in _chunks(n, H * L * dim):
                rows = slice(t0 + r0, t0 + r1)
                d = D[rows].reshape(r1 - r0, Hk, H // Hk, 1, dim)
                a = left[p][rows].reshape(r1 - r0, Hk, H // Hk, 1, dim)
                z = (d * B[None, :, None]).sum(-1) + (a * E[None, :, None]).sum(-1)
                full[:, r0:r1] = z.reshape(r1 - r0, H, L).transpose(0, 1)
            st["out"][p][place] = full[:, mask] + st["c"][p][place]
        t0 += n
    return st["out"]


def _plain_values(st):
    case = st["case"]
    H, Hk, dim = case["heads"], case["kv_heads"], case["dim"]
    D = st["x"][0] + st["x"][1] - st["a"][0] - st["a"][1]
    left = (st["a"][0] + D, st["a"][1])
    t0 = 0
    for s, n in enumerate(st["new"]):
        L = st["lens"][s]
        E = _cached(st, s, 0)
        mask, place = _row_mask(n, L), _packed(st, s)
        d = torch.zeros(H, n, L, dtype=torch.int64, device="cuda")
        d[:, mask] = D[place]
        d = d.reshape(Hk, H // Hk, n, L, 1)
        for p in range(2):
            B = _cached(st, s, 1 + p)
            a = torch.zeros(H, n, L, dtype=torch.int64, device="cuda")
            a[:, mask] = left[p][place]
            a = a.reshape(Hk, H // Hk, n, L, 1)
            for r0, r1 in _chunks(n, H * L * dim):
                z = (d[:, :, r0:r1] * B[:, None, None]).sum(-2) + \
                    (a[:, :, r0:r1] * E[:, None, None]).sum(-2)
                rows = slice(t0 + r0, t0 + r1)
                st["out"][p][rows] = (z.reshape(H, r1 - r0, dim).transpose(0, 1) +
                                      st["c"][p][rows])
        t0 += n
    return st["out"]


# ---- what a pass cannot do without ----

def work(case):
    dim = case["dim"]
    if case["kind"] == "rotary":
        vals = case["tokens"] * case["heads"] * dim
        return {"bytes": 32 * vals + 4 * case["tokens"] * (1 + case["rot"]),
                "flops": 2 * 3 * vals}
    new = _counts(case["new"])
    lens = [n + p for n, p in zip(new, _counts(case["past"]))]
    if case["kind"] == "append":
        vals = sum(new) * case["kv_heads"] * dim
        return {"bytes": 2 * vals * 8 * (4 + 3) + 4 * sum(new) * (2 + case["rot"]),
                "flops": vals * (2 * 3 + 2 * 3)}
    # Both parties: the cached words of every sequence once (opened
    # difference, two mask shares); per packed element and per query value
    # two shares, two triple shares; the triple product's shares and the
    # outputs.
    cached = sum(lens) * case["kv_heads"] * dim
    packed = case["heads"] * sum(n * L - n * (n - 1) // 2 for n, L in zip(new, lens))
    query = sum(new) * case["heads"] * dim
    return {"bytes": 8 * (3 * cached + 4 * packed + 4 * query) + 4 * case["heads"] * sum(new),
            "flops": 2 * 4 * packed * dim}


# ---- the definition on the host ----

def _host(t):
    return t.detach().cpu().numpy().view(np.uint64)


def _product(x, y):
    """x @ y mod 2^64 for uint64 matrices: 16-bit limbs in float64, whose
    sums of up to 2^20 products stay whole numbers below 2^53."""
    limb = [[((m >> np.uint64(16 * i)) & np.uint64(0xffff)).astype(np.float64) for i in range(4)]
            for m in (x, y)]
    out = np.zeros((x.shape[0], y.shape[1]), np.uint64)
    for i in range(4):
        for j in range(4 - i):
            out += (limb[0][i] @ limb[1][j]).astype(np.uint64) << np.uint64(16 * (i + j))
    return out


def _host_rotate(x, case, positions, far):
    half = case["rot"] // 2
    out = x * np.uint64(1 << FC)
    freq = BASE ** (-2.0 * np.arange(half) / max(1, 2 * half))
    ang = positions.astype(np.float64)[:, None] * freq
    scale = float(1 << FC)
    c = np.rint(np.cos(ang) * scale).astype(np.int64).view(np.uint64)[:, None]
    s = np.rint(np.sin(ang) * scale).astype(np.int64).view(np.uint64)[:, None]
    first = 2 * np.arange(half) if case["interleaved"] else np.arange(half)
    second = first + 1 if case["interleaved"] else first + half
    out[..., first] = x[..., first] * c - x[..., second] * s
    out[..., second] = x[..., first] * s + x[..., second] * c
    return out


def exact(case, seed):
    st = prepare(case, seed)
    with np.errstate(over="ignore"):
        return {"rotary": _exact_rotary, "append": _exact_append, "scores": _exact_product,
                "values": _exact_product}[case["kind"]](case, st)


def _signed(a):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int64))


def _exact_rotary(case, st):
    pos = st["positions"].cpu().numpy()
    return tuple(_signed(_host_rotate(_host(x), case, pos, case["far"])) for x in st["x"])


def _exact_append(case, st):
    table = st["pages"].cpu().numpy()
    pools = [[_host(t).copy() for t in st[k]] for k in ("k_pool", "v_pool")]
    t = 0
    for s, n in enumerate(st["new"]):
        pos = np.arange(st["lens"][s] - n, st["lens"][s])
        rows = slice(t, t + n)
        k = [_host_rotate(_host(x[rows]), case, pos, 0) for x in st["k"]]
        v = [_host(x[rows]) for x in st["v"]]
        for pool, x, m in zip(pools, (k, v), (st["k_mask"], st["v_mask"])):
            m = [_host(w[rows]) for w in m]
            for i, q in enumerate(pos):
                page, slot = table[s, q // case["page"]], q % case["page"]
                pool[0][page, :, slot] = (x[0][i] - m[0][i]) + (x[1][i] - m[1][i])
                pool[1][page, :, slot], pool[2][page, :, slot] = m[0][i], m[1][i]
        t += n
    return tuple(_signed(a) for pool in pools for a in pool)


def _exact_product(case, st):
    H, Hk, size = case["heads"], case["kv_heads"], case["page"]
    T, off, table = st["tokens"], st["offsets"].cpu().numpy(), st["pages"].cpu().numpy()
    x, a, c = ([_host(w) for w in st[k]] for k in ("x", "a", "c"))
    pool = [_host(w) for w in st["pool"]]
    opened = (x[0] - a[0]) + (x[1] - a[1])
    out = [w.copy() for w in c]
    t0 = 0
    for s, n in enumerate(st["new"]):
        L = st["lens"][s]
        ids = table[s, np.arange(L) // size]
        for g in range(Hk):
            E, B0, B1 = (w[ids, g, np.arange(L) % size] for w in pool)
            for h in range(g * (H // Hk), (g + 1) * (H // Hk)):
                spans = [slice(off[h * T + t], off[h * T + t + 1]) for t in range(t0, t0 + n)]
                if case["kind"] == "scores":
                    d, a0, a1 = (w[t0:t0 + n, h] for w in (opened, a[0], a[1]))
                    z = (_product(d, B0.T) + _product(a0 + d, E.T),
                         _product(d, B1.T) + _product(a1, E.T))
                    for p in range(2):
                        for i, sp in enumerate(spans):
                            out[p][sp] += z[p][i, :sp.stop - sp.start]
                else:
                    d, a0, a1 = (np.zeros((n, L), np.uint64) for _ in range(3))
                    for i, sp in enumerate(spans):
                        w = sp.stop - sp.start
                        d[i, :w], a0[i, :w], a1[i, :w] = opened[sp], a[0][sp], a[1][sp]
                    out[0][t0:t0 + n, h] += _product(d, B0) + _product(a0 + d, E)
                    out[1][t0:t0 + n, h] += _product(d, B1) + _product(a1, E)
        t0 += n
    return tuple(_signed(w) for w in out)
