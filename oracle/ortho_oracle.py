"""Plain numpy statement of the Newton-Schulz iteration, in 64 bits; used by the tests only."""

from __future__ import annotations

import numpy as np


def orthogonalize(G, coefficients, eps=1e-7, scale=1.0):
    """One matrix; ``coefficients``: a triple for each step."""
    X = np.asarray(G, np.float64)
    X = X / (np.sqrt((X * X).sum()) + eps)
    wide = X.shape[0] <= X.shape[1]
    for a, b, c in coefficients:
        A = X @ X.T if wide else X.T @ X
        P = a * np.eye(len(A)) + b * A + c * (A @ A)
        X = P @ X if wide else X @ P
    return scale * X


def by_singular_values(G, coefficients, eps=1e-7):
    """The same through the singular value decomposition: every step maps a value s to a s + b s^3 + c s^5."""
    U, s, V = np.linalg.svd(np.asarray(G, np.float64), full_matrices=False)
    s = s / (np.sqrt((s * s).sum()) + eps)
    for a, b, c in coefficients:
        s = a * s + b * s ** 3 + c * s ** 5
    return (U * s) @ V


def rounded(G, coefficients, two, eps=1e-7, rng=None):
    """The iteration with the roundings of the kernels' design and no others: X in a float16 number and, but before the last step, the
    next four bits of what that leaves, A and B in one float16 number, products of X's first number; with ``two`` all in two float16
    numbers and products hi hi + hi lo + lo hi.  Numbers are scaled so that float16's range plays no part.  With ``rng`` every rounding is
    a random one of up to half a step instead."""
    def leading(x, bits):
        unit = 2.0 ** (np.frexp(np.where(x == 0, 1.0, x))[1] - bits)
        return x * (1 + 2.0 ** -bits * rng.uniform(-1, 1, x.shape)) if rng is not None else np.round(x / unit) * unit

    def split(x, bits):
        hi = leading(x, 11)
        return hi, leading(x - hi, bits) if bits else 0 * hi

    def product(p, q):
        return p[0] @ q[0] + (p[0] @ q[1] + p[1] @ q[0] if two else 0)

    G = np.asarray(G, np.float64)
    X = G if G.shape[0] <= G.shape[1] else G.T
    X = split(X / (np.sqrt((X * X).sum()) + eps), 11 if two else 4 if len(coefficients) > 1 else 0)
    for i, (a, b, c) in enumerate(coefficients):
        A = split(product(X, (X[0].T, X[1].T)), 11 if two else 0)
        B = split(b * (A[0] + A[1]) + c * product(A, A), 11 if two else 0)
        Y = a * (X[0] + X[1]) + product(B, X)
        left = len(coefficients) - 1 - i
        X = split(Y, 11 if two else 4 if left > 1 else 0) if left else (Y, 0 * Y)
    X = X[0] + X[1]
    return X if G.shape[0] <= G.shape[1] else X.T
