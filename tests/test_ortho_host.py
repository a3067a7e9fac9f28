"""What the orthogonalised update refuses and how much memory it asks for, on the host alone."""

import ctypes

from gpu_ragged_dot_amd import _capi

lib = _capi.lib
INVALID, WORKSPACE = -1, -3
BF16, F32, F16 = _capi.RD_DTYPE_BF16, _capi.RD_DTYPE_F32, _capi.RD_DTYPE_F16
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


def _bytes(triples, dtype, g=3, k=200, n=150):
    flat = (ctypes.c_double * (3 * len(triples)))(*(v for t in triples for v in t))
    s = _capi.OrthoSpec(len(triples), flat, 1e-7, 1.0)
    return lib.rd_orthogonalize_spec_workspace_bytes(g, k, n, ctypes.byref(s), dtype)


def test_workspace_follows_from_the_growth_of_roundings():
    """bfloat16 matrices in 15 bits up to 2048 times, and in two numbers beyond; the others in two always."""
    steep, slow, flat = (3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0), (0.5, 0.0, 0.0)
    assert _bytes([steep] * 5, F16) == _bytes([steep] * 5, F32) == lib.rd_orthogonalize_workspace_bytes(3, 200, 150, F16)
    few, most = _bytes([steep] * 5, BF16), lib.rd_orthogonalize_workspace_bytes(3, 200, 150, BF16)
    assert 0 < few < most == _bytes([steep] * 5, F32) == lib.rd_orthogonalize_workspace_bytes(3, 200, 150, F32)
    for triples, want in (([steep] * 6, few), ([steep] * 7, most), ([slow] * 18, few), ([slow] * 19, most), ([flat] * 10 + [steep] * 6, few),
                          ([steep] * 6 + [flat] * 10, few), ([flat] + [steep] * 8, most),
                          ([flat] * 10 + [steep] * 7, few), ([], few)):  # (before the last: 2^-10 of X is what is rounded, and grows 5752 times)
        assert _bytes(triples, BF16) == want, triples
        assert _call(triples, BF16, g=3, k=200, n=150, ws_bytes=want - 256) == WORKSPACE
    assert _bytes([(30.0, 0.0, 0.0)] * 3, BF16) == 0 and b"converge" in lib.rd_last_error()
    assert lib.rd_orthogonalize_spec_workspace_bytes(3, 200, 150, None, BF16) == 0
    assert _bytes([steep], BF16, k=1 << 30) == 0 and _bytes([steep], BF16, g=0) == 0
