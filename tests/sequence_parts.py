"""f32 numbers as three bf16 parts: inputs whose third parts show in a result, and
the sum of the six products by which the cross entropy takes them."""
import numpy as np

import sequence_ref as ref

U = ref.U
SIX = [(2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0)]  # part of a, part of b


def parts(x):
    """x = x0 + x1 + x2, each a bf16 number (as f64)."""
    out, rest = [], np.asarray(x, np.float64)
    for _ in range(3):
        out.append(ref.rounded(rest, "bf16"))
        rest = rest - out[-1]
    return out


def product(a, b, without=()):
    """a b^T of f32 matrices by the products of their parts."""
    pa, pb = parts(a), parts(b)
    return sum(pa[i] @ pb[j].T for i, j in SIX if (i, j) not in without)


def pattern(rows, cols, seed, low=32):
    """Numbers of 24 bits whose parts are 1, 2^-9 and c 2^-23 with c of `low` to 63,
    all positive: a lost third part takes at least low / 64 of 2^-17 away, in the
    same direction everywhere."""
    c = np.random.default_rng(seed).integers(low, 64, (rows, cols))
    return 1 + 2.0 ** -9 + c * 2.0 ** -23


# What a logit of 64 such terms may be off, relative to it.  Left out are A1 B2, A2 B1
# and A2 B2, below 2^-24.  In units of 2^-23 every sum before A0 B0 is a whole number
# of at most 22 bits, so exact; the four steps of 16 terms of A0 B0 cut the running
# sum and their own terms to 24 bits, twice 2^-23 of the sum each: 8 * 2 U.  The
# epilogue's addition: U.
LOGIT = 24 * U


def logit_inputs(n, v, seed):
    """64 columns; rows of w at three sizes."""
    size = 2.0 ** -np.random.default_rng(seed).integers(0, 3, (v, 1))
    return pattern(n, 64, seed), pattern(v, 64, seed + 1) * size


def gradient_inputs(n, d, seed):
    """Two entries, the targets' all zeros: dx = dz_1 w_1 and dw_1 = dz_1^T x are
    single products where one token counts; dloss has 24 bits."""
    r = np.random.default_rng(seed)
    x = pattern(n, d, seed, 63) * 2.0 ** -6
    w = np.concatenate([np.zeros((1, d)), pattern(1, d, seed, 63)])
    return x, w, np.zeros(n, np.int64), (0.5 + r.random(n) / 2).astype(np.float32)
