"""The feed-forward operators' definitions in whole numbers mod 2^64 (numpy
uint64; >> is the floor of a division of the signed value)."""
import numpy as np

M64 = (1 << 64) - 1


def floor_shift(v, bits):
    return (np.asarray(v).view(np.int64) >> np.int64(bits)).view(np.uint64)


def matmul(x, w):
    """x w mod 2^64 for uint64 x and int64 w."""
    with np.errstate(over="ignore"):
        return np.matmul(x, w.view(np.uint64))


def piece(v, table):
    """The words of the pieces that hold v (unsigned order), uint64."""
    alpha, words = table
    at = np.searchsorted(alpha, v, side="right") - 1
    return [np.ascontiguousarray(words[:, k]).view(np.uint64)[at] for k in range(words.shape[1])]


def rsqrt(ms, table, f):
    with np.errstate(over="ignore"):
        c0, c1 = piece(ms, table)
        y = floor_shift(c1 * ms, f) + c0
        h = floor_shift(ms * floor_shift(y * y, f), f + 1)
        return floor_shift(y * (np.uint64(3 << (f - 1)) - h), f)


def rmsnorm(x, residual, inv_len, eps, table, f, weight=None, len_bits=26):
    """(s, out) of opened uint64 [rows, cols]."""
    with np.errstate(over="ignore"):
        s = x if residual is None else x + residual
        sq = (s * s).sum(1, dtype=np.uint64)
        ms = floor_shift(floor_shift(sq, f) * np.uint64(inv_len & M64), len_bits)
        y = rsqrt(ms + np.uint64(eps & M64), table, f)
        out = floor_shift(s * y[:, None], f)
        if weight is not None:
            out = floor_shift(out * weight.view(np.uint64), f)
    return s, out


def activate(y, act, f):
    if act is None:
        return y
    if isinstance(act, str):
        return np.where(y >> np.uint64(63), np.uint64(0), y)
    with np.errstate(over="ignore"):
        c0, c1, c2, c3 = piece(y, act)
        f64 = np.uint64(f)
        t = floor_shift((c3 * y + (c2 << f64)) * y, f)
        t = floor_shift((t + (c1 << f64)) * y, f)
        return floor_shift(t + (c0 << f64), f)


def linear(x, W, bias, f, act=None, residual=None, offsets=None, rows=None, n_rows=None,
           trunc=True):
    """(out, written): opened uint64 [rows, N] and which rows have an expert."""
    W = W if W.ndim == 3 else W[None]
    n_rows = (len(rows) if rows is not None else x.shape[0]) if n_rows is None else n_rows
    src = np.arange(n_rows) if rows is None else np.asarray(rows)
    offsets = [0, n_rows] if offsets is None else offsets
    out = np.zeros((n_rows, W.shape[2]), np.uint64)
    written = np.zeros(n_rows, bool)
    with np.errstate(over="ignore"):
        for e in range(W.shape[0]):
            for i in range(max(0, int(offsets[e])), min(n_rows, int(offsets[e + 1]))):
                v = x[src[i]] if 0 <= src[i] < x.shape[0] else np.zeros(x.shape[1], np.uint64)
                z = matmul(v[None], W[e])[0]
                if bias is not None:
                    z = z + bias.reshape(W.shape[0], -1)[e].view(np.uint64)
                out[i], written[i] = z, True
        if trunc:
            out = activate(floor_shift(out, f), act, f)
        if residual is not None:
            out = out + residual
    return out, written


def mix(z, slots, weights, f, residual=None):
    with np.errstate(over="ignore"):
        out = np.zeros((slots.shape[0], z.shape[1]), np.uint64)
        for t in range(slots.shape[0]):
            for s, w in zip(slots[t], weights[t]):
                if 0 <= s < z.shape[0]:
                    out[t] += z[s] * np.uint64(int(w) & M64)
        out = floor_shift(out, f)
        return out if residual is None else out + residual


def routing(rng, tokens, each, experts, rare=True):
    """(offsets, rows, slots): rows sorted by expert, the x row of each, and
    each token's rows; the last experts are rare."""
    likes = rng.random((tokens, experts)) ** (np.linspace(1, 4, experts) if rare else 1)
    chosen = np.argsort(-likes, axis=1)[:, :each].ravel()
    order = np.argsort(chosen, kind="stable")
    slots = np.empty(chosen.size, np.int64)
    slots[order] = np.arange(chosen.size)
    counts = np.bincount(chosen, minlength=experts)
    return (np.concatenate([[0], np.cumsum(counts)]), order // max(each, 1),
            slots.reshape(tokens, each))
