"""The numpy statements of the float8 operators, against torch's own conversion and by hand."""

import numpy as np
import pytest
import torch

from oracle import float8_oracle as oracle


def test_e4m3_is_torchs_conversion():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    numbers = codes[~codes.isnan()].numpy()
    assert np.array_equal(oracle.e4m3(numbers), numbers)
    x = (torch.randn(20000, generator=torch.Generator().manual_seed(0)) * torch.linspace(-20, 8.5, 20000).exp2()).clamp(-448, 448)
    middles = torch.from_numpy((np.sort(numbers)[1:] + np.sort(numbers)[:-1]).astype(np.float32) / 2)
    for t in (x, middles):
        assert np.array_equal(oracle.e4m3(t.numpy()), t.to(torch.float8_e4m3fn).double().numpy())


def test_blocks_by_hand():
    x = np.zeros((3, 130))
    x[0, :3], x[0, 128:] = [448, 1, -0.5], [3, -1.5]
    x[1, 5] = np.inf
    q, s = oracle.quantize(x)
    assert np.array_equal(s[0], [1.0, float(np.float32(3) / np.float32(448))]) and np.array_equal(q[0, [0, 1, 2, 128, 129]], [448, 1, -0.5, 448, -224])
    assert np.isnan(s[1, 0]) and s[1, 1] == s[2, 0] == float(np.float32(2.0 ** -80) / np.float32(448))
    assert np.all(q[2] == 0) and np.isnan(oracle.held(x)[1, :128]).all() and not np.isnan(oracle.held(x)[1, 128:]).any()
    assert np.array_equal(oracle.quantize(x, pow2=True)[1][0], [1.0, 2.0 ** -7])
    q, s = oracle.quantize(np.outer(np.arange(1, 131), np.ones(4)), height=128)
    assert np.array_equal(s[:, 0], np.float32([128, 130]) / np.float32(448)) and q[63, 0] == 224 and q[129, 0] == 448


@pytest.mark.parametrize("pow2", [False, True])
def test_values_are_within_half_a_step(pow2):
    x = np.random.default_rng(0).standard_normal((50, 300))
    q, s = oracle.quantize(x, pow2=pow2)
    wide = np.repeat(s, 128, 1)[:, :300]
    assert np.all(np.abs(oracle.held(x, pow2=pow2) - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * wide) * (1 + 2.0 ** -20))


def test_ragged_dot_by_hand():
    x, A = np.arange(8.0).reshape(4, 2), np.stack([np.eye(2), 2 * np.eye(2), 3 * np.eye(2)])
    assert np.array_equal(oracle.ragged_dot(x, A, [1, 0, 2]), np.stack([x[0], 3 * x[1], 3 * x[2], 0 * x[3]]))
    assert np.array_equal(oracle.ragged_dot(x, A, [-3, 9, 1], trans_rhs=True), 2 * x)
