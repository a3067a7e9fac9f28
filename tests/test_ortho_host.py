"""What the orthogonalised update refuses, on the host alone."""

import ctypes

from gpu_ragged_dot_amd import _capi

lib = _capi.lib
INVALID = -1
F32 = _capi.RD_DTYPE_F32
HERE = ctypes.addressof(ctypes.create_string_buffer(4096)) // 256 * 256 + 256  # an address that is never read


def _call(triples, dtype=F32, g=1, k=4, n=4, scale=1.0, ws_bytes=1 << 40):
    flat = (ctypes.c_double * (3 * len(triples)))(*(v for t in triples for v in t))
    s = _capi.OrthoSpec(len(triples), flat, 1e-7, scale)
    return lib.rd_orthogonalize(None, HERE, HERE, g, k, n, ctypes.byref(s), dtype, HERE, ws_bytes)


def test_growth_of_nearly_cubic_steps():
    """The largest value of a x + b x^3 + c x^5 is found whatever c is: 0.385 a for b = -a."""
    for c in (0.0, 1e-20, -1e-20, 1e-300, 5e-324, 1e-9):
        assert _call([(1e5, -1e5, c)]) == INVALID and b"converge" in lib.rd_last_error(), c
        assert _call([(2700.0, -2700.0, c)]) == INVALID and b"converge" in lib.rd_last_error(), c
        assert _call([(2600.0, -2600.0, c)], g=0) == 0, c
        assert _call([(1e200, -1e200, c)]) == INVALID and b"converge" in lib.rd_last_error(), c
    assert _call([(0.0, 0.0, 2000.0)]) == INVALID and _call([(0.0, 0.0, 1000.0)], g=0) == 0
    assert _call([(0.0, -2000.0, 0.0)]) == INVALID and _call([(0.0, 0.0, 0.0)], g=0) == 0


def test_scale_is_a_float32():
    assert _call([(1.0, 0.0, 0.0)], scale=1e39) == INVALID and b"scale" in lib.rd_last_error()
    assert _call([(1.0, 0.0, 0.0)], scale=-3e38, g=0) == 0
