"""Inputs of 4-bit projections that show a lost or misplaced low piece at any width, and the bound that sums of them obey.

The kernels hold x as two f16 pieces of a scaled value. Against random vectors the error of dropped low pieces falls, relative
to the sum of the magnitudes, as the root of the width, while a bound for that many roundings grows: at 16,000 columns it
would pass. Here only TERMS elements of a vector are not 0, each of 22 significant bits, which two pieces hold exactly."""
import numpy as np

TERMS = 4


def vectors(rng, n, cols, first=0):
    """n vectors: columns first, first + 1, ... in turn (every width is walked through by enough vectors), the last column, and
    two drawn ones; magnitudes from 1/4 to 4. The lowest of the 22 bits is set, so no low piece is 0."""
    x = np.zeros((n, cols))
    for i in range(n):
        at = np.unique(np.concatenate([[(first + i) % cols, cols - 1], rng.integers(0, cols, 8)]))
        at = np.concatenate([[(first + i) % cols], rng.permutation(at[at != (first + i) % cols])[:TERMS - 1]])
        m = 1.0 + (rng.integers(0, 1 << 20, len(at)) * 2 + 1) * 2.0 ** -21
        x[i, at] = m * 2.0 ** rng.integers(-2, 2, len(at)) * rng.choice([-1.0, 1.0], len(at))
    return x.astype(np.float32)


def bound(x, wd, wm):
    """Of |y - exact|, per output. x's pieces are exact and so is every product; what rounds is an addition whose operands are
    both not 0 and a scaling. An output has 2 * TERMS products not 0 (a high and a low piece each) and, where the format has
    minima, 2 * TERMS more with the sums of x by groups (a sum of up to TERMS elements rounded to f32 and to two pieces of 22
    bits: 2^-22 of it): 4 * TERMS - 1 additions and 2 * TERMS scalings at most, half a step (2^-24) of at most the sum of
    the magnitudes each, and a whole one where the matrix unit truncates instead."""
    size = np.abs(x.astype(np.float64)) @ (np.abs(wd) + wm).T
    minima = np.abs(x.astype(np.float64)) @ wm.T
    return size * (6 * TERMS) * 2.0 ** -23 + minima * 2.0 ** -22


def holds(got, x, wd, wm):
    want = x.astype(np.float64) @ (wd - wm).T
    return bool(np.all(np.abs(got.astype(np.float64) - want) <= bound(x, wd, wm)))


def in_pieces(x, wd, wm, mistake=None):
    """The product as the kernels hold x, in 64 bits: what the test has to tell from a product with a mistake in it. `mistake`:
    "lost", no low pieces; "shifted", low pieces 8 columns on; "tail", no low pieces from column 16,384 on."""
    x = x.astype(np.float64)
    top = np.abs(x).max(1, keepdims=True)
    scale = 2.0 ** (13 - np.floor(np.log2(np.where(top > 0, top, 1.0))))
    hi = (x * scale).astype(np.float16).astype(np.float64)
    lo = (x * scale - hi).astype(np.float16).astype(np.float64)
    if mistake == "lost":
        lo[:] = 0
    elif mistake == "shifted":
        lo = np.roll(lo, 8, 1)
    elif mistake == "tail":
        lo[:, 16384:] = 0
    # the minima take the sums of x, not of its pieces: they hide no mistake and show none
    return ((hi + lo) @ wd.T - (x * scale) @ wm.T) / scale
