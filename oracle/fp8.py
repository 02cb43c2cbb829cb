"""Rows in 8 bits from their definition, in 64-bit arithmetic on the CPU (no reference counterpart).

A block of 128 elements of a row (the last may be short) with largest finite magnitude a has the
scale 2^e, e the smallest integer >= -127 with a <= 448 * 2^e (a = 0: -127); an element's code stands for
the nearest multiple of 2^(max(floor(log2 |u|), -6) - 3) to u = element / 2^e, ties to the even multiple.
"""

import numpy as np

BLOCK = 128
CODES = np.array([(-1.0) ** (c >> 7) * (np.nan if c & 127 == 127 else
                                        (c & 7) / 512 if c & 120 == 0 else (8 + (c & 7)) * 2.0 ** ((c >> 3 & 15) - 10))
                  for c in range(256)])


def exponent(a):
    """The scale's exponent for a largest magnitude a, by search from the definition."""
    if a == 0:
        return -127
    e = int(np.ceil(np.log2(a / 448)))
    while a <= 448 * 2.0 ** (e - 1):
        e -= 1
    while a > 448 * 2.0 ** e:
        e += 1
    return max(e, -127)


def quantize(v):
    """float [R, d] -> (values that the codes stand for, before scaling [R, d], scale bytes [R, ceil(d / 128)])."""
    v = np.asarray(v, dtype=np.float64)
    R, d = v.shape
    nb = -(-d // BLOCK)
    codes, scale = np.zeros((R, d)), np.zeros((R, nb), dtype=np.uint8)
    for r in range(R):
        for b in range(nb):
            u = v[r, b * BLOCK:(b + 1) * BLOCK]
            fine = np.isfinite(u)
            e = exponent(np.abs(u[fine]).max() if fine.any() else 0.0)
            scale[r, b] = e + 127
            u = np.where(fine, u, 0.0) / 2.0 ** e
            mantissa, power = np.frexp(u)  # |mantissa| in [1/2, 1)
            step = 2.0 ** (np.maximum(power - 1, -6) - 3)
            codes[r, b * BLOCK:(b + 1) * BLOCK] = np.where(fine, np.rint(u / step) * step, np.nan)
    return codes, scale


def values(codes, scale):
    """Code bytes (uint8 [R, d]) and scale bytes -> the elements they stand for."""
    two = np.repeat(2.0 ** (scale.astype(np.float64) - 127), BLOCK, axis=1)[:, :codes.shape[1]]
    return CODES[codes] * two
