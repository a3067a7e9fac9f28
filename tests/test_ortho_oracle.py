"""The numpy statement of the Newton-Schulz iteration against the singular value decomposition."""

import numpy as np
import pytest

from oracle import ortho_oracle as oracle

TRIPLE = (3.4445, -4.7750, 2.0315)


@pytest.mark.parametrize("k,n", [(5, 5), (8, 40), (40, 8), (1, 7), (7, 1)])
def test_singular_values(k, n):
    G = np.random.default_rng(k * n).standard_normal((k, n))
    for steps in (0, 1, 5):
        got, want = oracle.orthogonalize(G, [TRIPLE] * steps), oracle.by_singular_values(G, [TRIPLE] * steps)
        assert np.max(np.abs(got - want)) < 1e-9
    assert np.all(np.abs(np.linalg.svd(oracle.orthogonalize(G, [TRIPLE] * 5), compute_uv=False) - 0.95) < 0.3) or min(k, n) > 1


def test_zeros_stay_zeros():
    assert not oracle.orthogonalize(np.zeros((3, 4)), [TRIPLE] * 5).any()
