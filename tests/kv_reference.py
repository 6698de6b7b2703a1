"""Plain numpy forms (uint64, wrapping) of the operators of attention over a
paged cache, written from their formulas token by token."""
import numpy as np

U = np.uint64


def words(rng, *shape):
    return rng.integers(0, 1 << 64, shape, dtype=U)


def rotate_row(x, factors, interleaved, pass_mul):
    """One head's values x [dim] by factors int [rot / 2][2]."""
    f = np.asarray(factors, dtype=np.int64).astype(U)
    half = len(f)
    out = x * U(pass_mul & (2 ** 64 - 1))
    u = np.arange(half) * (2 if interleaved else 1)
    v = u + (1 if interleaved else half)
    out[u] = x[u] * f[:, 0] - x[v] * f[:, 1]
    out[v] = x[u] * f[:, 1] + x[v] * f[:, 0]
    return out


def rotary(x, table, positions, interleaved, pass_mul, before):
    """x, before [tokens, heads, dim]; rows outside the table keep `before`."""
    out = before.copy()
    for t, pos in enumerate(positions):
        if 0 <= pos < len(table):
            for h in range(x.shape[1]):
                out[t, h] = rotate_row(x[t, h], table[pos], interleaved, pass_mul)
    return out


class Case:
    """A batch: new and kv lengths of each sequence, page numbers and pools."""

    def __init__(self, rng, new, lens, page, kv_heads, dim, pad=0, spare=3, width=None):
        self.new, self.lens, self.page = list(new), list(lens), page
        self.kv_heads, self.dim = kv_heads, dim
        need = [-(-n // page) for n in lens]
        self.width = max(need + [1]) if width is None else width
        pages = sum(need) + spare
        order = rng.permutation(pages)
        self.table = np.full((len(new), self.width), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.tokens = int(self.cu[-1]) + pad
        self.pages = pages
        self.pool = [words(rng, pages, kv_heads, page, dim) for _ in range(3)]

    def spot(self, s, j):
        """(page, place) of key j of sequence s, or None."""
        if j < 0 or j // self.page >= self.width:
            return None
        pg = self.table[s, j // self.page]
        return (pg, j % self.page) if 0 <= pg < self.pages else None

    def cached(self, s, g, which, most):
        """[length, dim] words of a pool array (no more keys than the longest
        row's); zeros without a page."""
        out = np.zeros((min(max(0, self.lens[s]), most), self.dim), U)
        for j in range(len(out)):
            at = self.spot(s, j)
            if at is not None:
                out[j] = self.pool[which][at[0], g, at[1]]
        return out

    def causal(self, heads):
        """Offsets of causal rows, padding rows empty."""
        rows = np.zeros(self.tokens, np.int64)
        for s, n in enumerate(self.new):
            rows[self.cu[s]:self.cu[s] + n] = np.maximum(
                0, np.arange(self.lens[s] - n + 1, self.lens[s] + 1))
        return np.concatenate([[0], np.cumsum(np.tile(rows, heads))]).astype(np.int32)


def append(case, x, mask, table=None, interleaved=False, pass_mul=1, positions=None, shift=None):
    """The pool's three arrays after the append of x, mask (pairs [tokens,
    kv_heads, dim]).  shift: the rows truncated by that many bits first."""
    e, b0, b1 = (a.copy() for a in case.pool)
    for s, n in enumerate(case.new):
        for r in range(n):
            t, at = case.cu[s] + r, case.lens[s] - n + r
            spot = case.spot(s, at)
            pos = at if positions is None else positions[t]
            if spot is None or (table is not None and not 0 <= pos < len(table)):
                continue
            for h in range(case.kv_heads):
                v = [w[t, h] for w in x]
                if table is not None:
                    v = [rotate_row(w, table[pos], interleaved, pass_mul) for w in v]
                whole = v[0] + v[1]
                if shift is not None:
                    whole = (whole.view(np.int64) >> shift).view(U)
                e[spot[0], h, spot[1]] = whole - mask[0][t, h] - mask[1][t, h]
                b0[spot[0], h, spot[1]], b1[spot[0], h, spot[1]] = mask[0][t, h], mask[1][t, h]
    return e, b0, b1


def _span(off, i, n, kv):
    f, l = int(off[i]), int(off[i + 1]) - int(off[i])
    return (0, 0) if f < 0 or l <= 0 or f + l > n else (f, min(l, max(kv, 0)))


def scores(case, heads, off, x, a, c, before):
    out = [b.copy() for b in before]
    d = (x[0] - a[0]) + (x[1] - a[1])
    left = (a[0] + d, a[1])
    most = int(max(0, np.diff(off.astype(np.int64)).max(initial=0)))
    for s, n in enumerate(case.new):
        for h in range(heads):
            g = h // (heads // case.kv_heads)
            E, *B = (case.cached(s, g, i, most) for i in range(3))
            for t in range(case.cu[s], case.cu[s] + n):
                f, l = _span(off, h * case.tokens + t, len(out[0]), case.lens[s])
                for p in range(2):
                    out[p][f:f + l] = (c[p][f:f + l] + (B[p][:l] * d[t, h]).sum(1, dtype=U) +
                                       (E[:l] * left[p][t, h]).sum(1, dtype=U))
    return out


def values(case, heads, off, x, a, c, before):
    out = [b.copy() for b in before]
    d = (x[0] - a[0]) + (x[1] - a[1])
    left = (a[0] + d, a[1])
    most = int(max(0, np.diff(off.astype(np.int64)).max(initial=0)))
    for s, n in enumerate(case.new):
        for h in range(heads):
            g = h // (heads // case.kv_heads)
            E, *B = (case.cached(s, g, i, most) for i in range(3))
            for t in range(case.cu[s], case.cu[s] + n):
                f, l = _span(off, h * case.tokens + t, len(d), case.lens[s])
                for p in range(2):
                    out[p][t, h] = (c[p][t, h] + (B[p][:l] * d[f:f + l, None]).sum(0, dtype=U) +
                                    (E[:l] * left[p][f:f + l, None]).sum(0, dtype=U))
    return out
