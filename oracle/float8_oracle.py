"""Plain numpy statements of the float8 operators with a scale for each block of 128, in 64 bits; used by the tests only."""

from __future__ import annotations

import numpy as np

BLOCK, LARGEST, LEAST = 128, 448.0, 2.0 ** -80


def e4m3(x):
    """The nearest e4m3fn number, ties to even: three bits behind the leading one down to 2^-6, multiples of 2^-9 below."""
    x = np.asarray(x, np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6))) - 3)
    return np.clip(np.round(x / step) * step, -LARGEST, LARGEST)


def scales_of(largest, pow2):
    s = (np.maximum(largest, LEAST).astype(np.float32) / np.float32(LARGEST)).astype(np.float64)
    if pow2:
        mantissa, exponent = np.frexp(s)
        s = np.ldexp(1.0, exponent - (mantissa == 0.5))
    return np.where(np.isfinite(largest), s, np.nan)


def quantize(x, height=1, pow2=False):
    """(codes, scales) of blocks ``height`` x 128 of x [rows, cols], codes as the e4m3fn numbers that they are."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    down, across = -(-rows // height), -(-cols // BLOCK)
    whole = np.zeros((down * height, across * BLOCK))
    whole[:rows, :cols] = x
    blocks = whole.reshape(down, height, across, BLOCK)
    with np.errstate(invalid="ignore"):
        s = scales_of(np.abs(blocks).max((1, 3)), pow2)
        q = e4m3((blocks / s[:, None, :, None]).astype(np.float32))
    return q.reshape(whole.shape)[:rows, :cols], s


def values(q, s, height=1):
    return q * np.repeat(np.repeat(s, height, 0)[:q.shape[0]], BLOCK, 1)[:, :q.shape[1]]


def held(x, height=1, pow2=False):
    return values(*quantize(x, height, pow2), height)


def ragged_dot(x, A, sizes, trans_rhs=False):
    """Rows past the groups are zero; groups end at the last row; negative sizes are empty groups."""
    m, n = x.shape[0], A.shape[1 if trans_rhs else 2]
    y, row = np.zeros((m, n)), 0
    for e, size in enumerate(sizes):
        end = min(m, row + max(int(size), 0))
        y[row:end] = x[row:end] @ (A[e].T if trans_rhs else A[e])
        row = end
    return y
