"""The closed form of the softmax of long rows (exact products and shifts), and
how far it may be from real numbers."""
import numpy as np

import fixed_point as fp
from suf_amd import softmax, tables

HALF, WEIGHT, INV = softmax.HALF_BITS, softmax.WEIGHT_BITS, softmax.INV_BITS


def weights(scores, offsets, f):
    """Q(f) scores of packed rows -> (weights, their sums, reciprocals)."""
    lens = np.diff(offsets)
    g = fp.cubic_task(*tables.nexp_fine_table(HALF),
                      fp.row_max_diff(scores, offsets) << (HALF - 1 - f), HALF)
    w = fp.mul_shift(g, g, 2 * HALF - WEIGHT)
    s = fp.row_sums(w, offsets)
    nmax = 2.0 ** max(1, int(lens.max()).bit_length())
    y = fp.recip_task(*tables.recip_wide_table(INV, nmax), s << (INV - WEIGHT), INV, 3)
    return w, s, y


def quotient(z, y):
    """z: sums of weights times Q(f) values -> Q(f)."""
    return fp.mul_shift(z >> WEIGHT, y, INV)


def bound(real):
    """Most that a row's shares can be from real / sum(real) in all (real: the
    exact exponentials, 1 the largest).  g = exp(-t / 2) is within 2.7e-4 of
    itself (h^4 / 384 at a piece's start) and 3 steps; its square adds a step
    of 2^-24; t past 32 counts as 0; the reciprocal three floors of up to its
    sum's steps of 2^-28 and its guess's error to the eighth power."""
    g = np.sqrt(real)
    d = 0.5 ** 4 / 384 * np.exp(0.5) * g + 3 * 2.0 ** -HALF
    err = np.where(g < np.exp(-16.0), real, 2 * g * d + d * d + 2.0 ** -WEIGHT)
    s, e = real.sum(), err.sum()
    return 2 * e / (s - e) + 3 * (s + e + 1) * 2.0 ** -INV + 0.125 ** 8
