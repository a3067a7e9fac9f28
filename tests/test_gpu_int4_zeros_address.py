"""Zeros of the product on 4-bit weights at every address: they are bytes, of which the kernels load one, two or four at a time."""

import pytest
import torch

import gpu_ragged_dot_amd as rd
from gpu_ragged_dot_amd import _capi
from gpu_ragged_dot_amd.int4 import _ragged_dot_int4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("m", [20, 300])
@pytest.mark.parametrize("kernel", [_capi.RD_INT4_STREAM, _capi.RD_INT4_TILES], ids=["stream", "tiles"])
def test_zeros_at_odd_addresses(m, block, dtype, kernel):
    print(f"int4 zeros m {m} block {block} {dtype} kernel {kernel}", flush=True)
    k, n, g = 300, 83, 2
    gen = torch.Generator().manual_seed(block)
    codes = lambda *s: torch.randint(0, 16, s, generator=gen, dtype=torch.uint8).cuda()
    blocks = -(-k // block)
    w = rd.pack_int4(codes(g, k, n), (0.1 * torch.rand((g, blocks, n), generator=gen)).to(dtype).cuda(), codes(g, blocks, n), block=block)
    x = torch.randn((m, k), generator=gen).to(dtype).cuda()
    gs = torch.tensor([m // 2, m - m // 2], dtype=torch.int32, device="cuda")
    want = _ragged_dot_int4(x, w, gs, kernel=kernel)
    for by in (1, 2, 3):
        zeros = torch.empty(w.zeros.numel() + by, dtype=torch.uint8, device="cuda")[by:].view(w.zeros.shape).copy_(w.zeros)
        assert zeros.data_ptr() % 4 == by
        assert torch.equal(_ragged_dot_int4(x, w._replace(zeros=zeros), gs, kernel=kernel), want)
