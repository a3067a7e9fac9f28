"""The largest numbers of float8 blocks that a launch is given, on the host alone: no more than 2^32 - 1 threads."""

import ctypes

from gpu_ragged_dot_amd import _capi

lib = _capi.lib
UNSUPPORTED = -2
BF16 = _capi.RD_DTYPE_BF16
HERE = ctypes.addressof(ctypes.create_string_buffer(4096)) // 256 * 256 + 256  # an address that is never read


def test_rows():
    """A row of up to 512 numbers is four blocks, of sixteen lanes each, in work-groups of sixteen blocks."""
    p = HERE
    for rows in ((1 << 26) - 1, (1 << 26) - 3, 1 << 26):
        assert lib.rd_float8_rows(None, p, p, p, rows, 100, 0, BF16) == UNSUPPORTED, rows
        assert lib.rd_moe_swiglu_float8(None, p, p, p, rows, 512, 0, BF16) == UNSUPPORTED, rows
