"""Updates of experts' weights with singular values near one, by Newton-Schulz products: what the Muon optimiser makes of a momentum.

    dA = torch.autograd.grad(ragged_dot(x, A, group_sizes), A, dout)     # [g, k, n]
    momentum.lerp_(dA, 0.05)
    A -= lr * orthogonalize(momentum)

The reference has no counterpart; the kernels are behind ``rd_orthogonalize`` of the C ABI (``include/ragged_dot_hip.h``), the host
side in ``csrc/rd_torch.cpp``.
"""

from __future__ import annotations

from typing import Sequence, Union

import torch

from . import _tracing
from ._native import lib as _native

__all__ = ["orthogonalize"]

COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # steep at 0, and within 0.7 .. 1.2 once there


def orthogonalize(G: torch.Tensor, *, steps: int = 5, coefficients: Union[Sequence[float], Sequence[Sequence[float]]] = COEFFICIENTS,
                  eps: float = 1e-7, scale: float = 1.0) -> torch.Tensor:
    """``scale * X`` for every matrix of ``G`` ``[g, k, n]`` or ``[k, n]`` (bfloat16, float16 or float32, and so the result): ``X = G /
    (|G|_F + eps)``, then ``steps`` times ``A = X X'; X = a X + (b A + c A A) X``, on the transpose where ``k > n``.
    ``coefficients``: ``(a, b, c)``, or one such triple for each of the steps.  Products of bfloat16 matrices are of float16 numbers, with
    ``X`` held in 15 bits, off by 1e-3 to 3e-3 of the result's norm (up to 1e-2 where there are few rows, columns or directions), or, with
    coefficients that multiply roundings by more than 2048 (seven steps of the default ones), as those of float32 and
    float16 matrices; these are as accurate as float32 products, for 2.4 times the time.  No gradient."""
    triples = [tuple(map(float, t)) for t in coefficients] if len(coefficients) and hasattr(coefficients[0], "__len__") else None
    if triples is None:
        triples = [tuple(map(float, coefficients))] * steps
    if any(len(t) != 3 for t in triples):
        raise ValueError("coefficients are a triple (a, b, c), or one for each step")
    if steps < 0 or len(triples) != steps:
        raise ValueError(f"{steps=} but {len(triples)} triples of coefficients")
    flat = [v for t in triples for v in t]
    if _tracing.active():
        return _tracing.record(lambda G: _native.orthogonalize(G.detach(), flat, eps, scale), G)
    return _native.orthogonalize(G, flat, eps, scale)
