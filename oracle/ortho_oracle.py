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
    """The iteration with the roundings of the kernels' design and no others: X in two float16 numbers, hi + lo, A and B in one, products
    of hi alone; with ``two`` all in two numbers and products hi hi + hi lo + lo hi.  Numbers are scaled so that float16's range plays
    no part.  With ``rng`` every rounding is a random one of up to half a step instead."""
    def split(x, planes):
        if rng is not None:
            fine = x * (1 + 2.0 ** -22 * rng.uniform(-1, 1, x.shape)) if planes else x
            hi = fine * (1 + 2.0 ** -11 * rng.uniform(-1, 1, x.shape))
            return (hi, fine - hi) if planes else (hi, 0 * hi)
        top = np.abs(x).max()
        unit = 2.0 ** (14 - np.frexp(top)[1]) if top else 1.0
        hi = (x * unit).astype(np.float16).astype(np.float64)
        lo = (x * unit - hi).astype(np.float16).astype(np.float64) if planes else 0 * hi
        return hi / unit, lo / unit

    def product(p, q):
        return p[0] @ q[0] + (p[0] @ q[1] + p[1] @ q[0] if two else 0)

    G = np.asarray(G, np.float64)
    X = G if G.shape[0] <= G.shape[1] else G.T
    X = split(X / (np.sqrt((X * X).sum()) + eps), True)
    for i, (a, b, c) in enumerate(coefficients):
        A = split(product(X, (X[0].T, X[1].T)), two)
        B = split(b * (A[0] + A[1]) + c * product(A, A), two)
        Y = a * (X[0] + X[1]) + product(B, X)
        X = split(Y, True) if i + 1 < len(coefficients) else (Y, 0 * Y)
    X = X[0] + X[1]
    return X if G.shape[0] <= G.shape[1] else X.T
