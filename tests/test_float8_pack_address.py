"""Codes of a checkpoint at any address, on the host alone: the products take them from 16-byte addresses on."""

import torch

import gpu_ragged_dot_amd as rd


def test_codes_at_odd_addresses_are_copied():
    flat = torch.arange(2 * 128 * 256 + 32, dtype=torch.int64).remainder(127).to(torch.uint8)
    for first in (0, 1, 8, 16, 24):
        codes = flat[first:first + 2 * 128 * 256].view(2, 128, 256).view(torch.float8_e4m3fn)
        assert codes.is_contiguous()
        packed = rd.pack_float8(codes, torch.ones(2, 1, 2))
        assert packed.codes.data_ptr() % 16 == 0 and torch.equal(packed.codes.view(torch.uint8), codes.view(torch.uint8))
        assert (packed.codes.data_ptr() == codes.data_ptr()) == (first % 16 == 0)
