"""Products on 4-bit weights that are not rounded, whatever the number of rows."""

import numpy as np
import pytest
import torch

import gpu_ragged_dot_amd as rd
from oracle import expert_ops_oracle as oracle

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("k,n,sizes,block,zeros", [(1024, 640, [1500, 900, 40], 128, False), (1000, 515, [700, 0, 1301], 32, True), (4096, 512, [2048], 64, True)])
def test_the_result_is_the_only_rounding(k, n, sizes, block, zeros, dtype):
    print(f"int4 exact weights k {k} n {n} {sizes} block {block} {dtype}", flush=True)
    rng = np.random.default_rng(k)
    g, blocks, m = len(sizes), -(-k // block), sum(sizes)
    q = rng.integers(0, 16, (g, k, n)).astype(np.uint8)
    s = torch.from_numpy(rng.uniform(0.5, 1.5, (g, blocks, n)) * k ** -0.5).to(dtype)
    z = rng.integers(0, 16, (g, blocks, n)).astype(np.uint8) if zeros else None
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(k)).to(dtype)
    dense = oracle.int4_dense(q, s.double().numpy(), z, block)
    at = np.arange(k) // block
    reach = np.abs(s.double().numpy())[:, at] * (32.0 if z is None else 32.0 + z[:, at].astype(float))
    want, sums, row = np.zeros((m, n)), np.zeros((m, n)), 0
    for e, size in enumerate(sizes):
        part = slice(row, row + size)
        want[part], sums[part] = x[part].double().numpy() @ dense[e], x[part].double().abs().numpy() @ reach[e]
        row += size
    to = lambda a: None if a is None else torch.as_tensor(a).cuda()
    w = rd.pack_int4(to(q), to(s), to(z), block=block)
    error = {}
    for exact in (False, True):
        got = rd.ragged_dot_int4(x.cuda(), w, torch.tensor(sizes), exact_weights=exact).double().cpu().numpy()
        error[exact] = np.abs(got - want)
    # one rounding of the result; fp32 sums of k terms, of x and of x times codes, lose at most 2^-23 per term of what they add up
    assert np.all(error[True] <= HALF_ULP[dtype] * np.abs(want) + (k + 16) * 2.0 ** -23 * sums + 2.0 ** -25)
    assert np.linalg.norm(error[True]) <= np.linalg.norm(error[False])
    # (results are spread over a binade: a rounding to nearest is off by 0.42 of the half step, root mean square, at most 0.58)
    assert np.linalg.norm(error[True]) <= 0.6 * HALF_ULP[dtype] * np.linalg.norm(want)
