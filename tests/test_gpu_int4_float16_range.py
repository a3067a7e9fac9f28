"""Weights and padding at the end of float16's range in the tiles of the product on 4-bit weights: a weight that rounds to infinity makes
the results that it goes into infinite, and what stands past the last contraction index - codes of 8 on the last block's scale - goes
into none.  All sums here are exact in fp32."""

import pytest
import torch

import gpu_ragged_dot_amd as rd
from gpu_ragged_dot_amd import _capi
from gpu_ragged_dot_amd.int4 import _ragged_dot_int4

pytestmark = pytest.mark.gpu

LENGTHS = [8, 63, 64, 65, 72, 100, 128, 129, 191, 200, 256, 257, 320, 448, 641]


@pytest.mark.parametrize("k", LENGTHS)
@pytest.mark.parametrize("sizes", [[300], [70, 130]], ids=["one", "two"])
def test_an_infinite_weight_makes_its_results_infinite(k, sizes):
    print(f"int4 float16 infinite weight k {k} {sizes}", flush=True)
    n, g, m = 80, len(sizes), sum(sizes)
    q = torch.full((g, k, n), 8, dtype=torch.uint8)
    q[:, :, :40] = torch.randint(7, 10, (g, k, 40), generator=torch.Generator().manual_seed(k), dtype=torch.uint8)
    q[:, k - 1, 5], q[:, 0, 44], q[:, k // 2, 70] = 15, 15, 1  # 7 and -7 times 16384
    scales = torch.full((g, -(-k // 128), n), 16384.0).half()
    x = torch.full((m, k), 2.0 ** -8).half()
    x[::2] = 2.0 ** -9
    y = _ragged_dot_int4(x.cuda(), rd.pack_int4(q.cuda(), scales.cuda()), torch.tensor(sizes), kernel=_capi.RD_INT4_TILES).cpu()
    dense = (q.double() - 8) * 16384
    dense[dense.abs() > 65504] *= torch.inf
    want, row = torch.empty((m, n), dtype=torch.float64), 0
    for e, size in enumerate(sizes):
        # (every x is above 0: an infinite weight's column is of its sign)
        want[row:row + size] = x[row:row + size].double() @ dense[e].where(dense[e].isfinite(), 0) + dense[e].where(~dense[e].isfinite(), 0).sum(0)
        row += size
    assert torch.equal(y, want.half())


@pytest.mark.parametrize("k", LENGTHS + [4104, 8200])
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("sizes", [[300], [70, 130]], ids=["one", "two"])
def test_what_lies_past_the_contraction_is_not_multiplied(k, block, sizes):
    print(f"int4 float16 tail k {k} block {block} {sizes}", flush=True)
    n, g, m = 80, len(sizes), sum(sizes)
    gen = torch.Generator().manual_seed(k)
    q = torch.randint(5, 8, (g, k, n), generator=gen, dtype=torch.uint8)
    scales = torch.full((g, -(-k // block), n), 60000.0).half()  # weights of -1, 0 and 1 times that; a code of 8 would be infinite
    zeros = torch.full(scales.shape, 6, dtype=torch.uint8)
    x = (torch.randint(-1, 2, (m, k), generator=gen) * 2.0 ** -12).half()
    w = rd.pack_int4(q.cuda(), scales.cuda(), zeros.cuda(), block=block)
    y = _ragged_dot_int4(x.cuda(), w, torch.tensor(sizes), kernel=_capi.RD_INT4_TILES).cpu()
    want, row = torch.empty((m, n), dtype=torch.float64), 0
    for e, size in enumerate(sizes):
        want[row:row + size] = x[row:row + size].double() @ ((q[e].double() - 6) * 60000)
        row += size
    assert torch.equal(y, want.half())
