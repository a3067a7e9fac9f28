"""Which kernel multiplies a slice of the groups: by what the slice is, not by what all groups would be."""

import pytest
import torch

import gpu_ragged_dot_amd as rd
from gpu_ragged_dot_amd import _capi
from gpu_ragged_dot_amd.int4 import _ragged_dot_int4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("g,rows,first,held,kernel", [(64, 64, 16, 8, _capi.RD_INT4_STREAM), (64, 64, 0, 64, _capi.RD_INT4_TILES),
                                                      (16, 300, 8, 8, _capi.RD_INT4_TILES), (32, 5, 30, 2, _capi.RD_INT4_STREAM)])
def test_a_slice_is_multiplied_by_the_kernel_for_its_size(g, rows, first, held, kernel):
    k, n = 2048, 4096
    gen = torch.Generator(device="cuda").manual_seed(g + held)
    codes = torch.randint(-2 ** 31, 2 ** 31 - 1, (held, n // 16, k // 128, 64, 4), generator=gen, dtype=torch.int32, device="cuda")
    scales = (torch.rand((held, k // 128, n, 1), generator=gen, device="cuda") * 0.01).bfloat16()
    w = rd.Int4Weights(codes, scales, None, k, n, 128)
    x = torch.randn((g * rows, k), generator=gen, device="cuda").bfloat16()
    gs = torch.full((g,), rows, dtype=torch.int32, device="cuda")
    offset = None if held == g else first
    by = {q: _ragged_dot_int4(x, w, gs, group_offset=offset, kernel=q) for q in (_capi.RD_INT4_AUTO, _capi.RD_INT4_STREAM, _capi.RD_INT4_TILES)}
    assert torch.equal(by[_capi.RD_INT4_AUTO], by[kernel])
    if rows > 48:  # (up to there both are the streaming kernel)
        assert not torch.equal(by[_capi.RD_INT4_STREAM], by[_capi.RD_INT4_TILES])
    for y in by.values():
        assert not y[:first * rows].any() and not y[(first + held) * rows:].any()
    part = slice(first * rows, (first + held) * rows)
    alone = _ragged_dot_int4(x[part].contiguous(), w, gs[first:first + held].contiguous(), kernel=_capi.RD_INT4_TILES)
    # the same product, but for the order of fp32 sums and, by the other kernel, a rounding of every weight
    assert (by[kernel][part].double() - alone.double()).norm() <= 2.0 ** -7 * alone.double().norm()
