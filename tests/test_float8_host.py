"""What the float8 and Newton-Schulz entry points refuse, and the product's loaders, on the host alone."""

import ctypes
import os
import subprocess

import pytest
import torch

import gpu_ragged_dot_amd as rd
from gpu_ragged_dot_amd import _capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "gpu_ragged_dot_amd", "csrc")
EXE = os.path.join(ROOT, "tests", "host_checks", "float8_loader")
lib = _capi.lib
INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3
BF16, F32, F8 = _capi.RD_DTYPE_BF16, _capi.RD_DTYPE_F32, _capi.RD_DTYPE_F8E4M3_BF16
HERE = ctypes.addressof(ctypes.create_string_buffer(4096)) // 256 * 256 + 256  # an address that is never read
NOW = None  # stream


def test_loaders_stay_inside_their_windows():
    r = subprocess.run(["make", "-C", CSRC, os.path.relpath(EXE, CSRC)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([EXE], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.startswith("float8_loader ok ") and int(r.stdout.split()[2]) > 1_000_000


def test_rows():
    p = HERE
    assert lib.rd_float8_rows(NOW, p, p, p, 0, 5, 0, BF16) == 0 and lib.rd_float8_rows(NOW, None, None, None, 5, 0, 0, BF16) == 0
    assert lib.rd_float8_rows(NOW, p, p, p, 2, 5, 0, F8) == INVALID
    assert lib.rd_float8_rows(NOW, p, p, p, -1, 5, 0, BF16) == INVALID
    assert lib.rd_float8_rows(NOW, p, p, p, 1, (1 << 22) + 1, 0, BF16) == INVALID
    assert lib.rd_float8_rows(NOW, None, p, p, 2, 5, 0, BF16) == INVALID
    assert lib.rd_float8_rows(NOW, p, p + 8, p, 2, 5, 0, BF16) == INVALID
    assert lib.rd_float8_rows(NOW, p, p, p + 4, 2, 5, 0, BF16) == INVALID
    assert lib.rd_float8_rows(NOW, p, p, p, (1 << 31) - 1, 1024, 0, BF16) == UNSUPPORTED
    assert lib.rd_moe_swiglu_float8(NOW, None, p, p, 2, 5, 0, BF16) == INVALID
    assert lib.rd_moe_swiglu_float8(NOW, p, None, p, 2, 5, 0, BF16) == INVALID
    i32 = ctypes.cast(p, ctypes.POINTER(ctypes.c_int32))
    assert lib.rd_moe_dispatch_float8(NOW, p, i32, i32, p, p, 4, 65, 128, 0, BF16) == INVALID
    assert lib.rd_moe_dispatch_float8(NOW, p, None, i32, p, p, 4, 2, 128, 0, BF16) == INVALID
    assert lib.rd_moe_dispatch_float8(NOW, p, None, None, None, None, 0, 2, 128, 0, BF16) == 0


def test_weights():
    p = HERE
    assert lib.rd_float8_weights(NOW, None, None, None, 3, 0, 4, 0, BF16) == 0
    assert lib.rd_float8_weights(NOW, p, p, p, 0, 4, 4, 0, BF16) == INVALID
    assert lib.rd_float8_weights(NOW, p, p, p, 1, 4, 4, 0, F8) == INVALID
    assert lib.rd_float8_weights(NOW, p, p + 4, p, 1, 4, 4, 0, BF16) == INVALID
    assert lib.rd_float8_weights(NOW, None, p, p, 1, 4, 4, 0, BF16) == INVALID
    assert lib.rd_float8_weights(NOW, p, p, p, 1 << 23, 128, 256, 0, BF16) == UNSUPPORTED
    assert lib.rd_float8_values(NOW, p, p, p, 2, 4, 4, 1, BF16) == INVALID   # rows come as one matrix
    assert lib.rd_float8_values(NOW, p, p, p, 1, 4, 4, 64, BF16) == INVALID
    assert lib.rd_float8_values(NOW, p, p, None, 1, 4, 4, 128, BF16) == INVALID
    assert lib.rd_float8_values(NOW, p, p, p, 1 << 11, 1 << 20, 128, 128, BF16) == UNSUPPORTED


def test_product():
    p = HERE
    i32 = ctypes.cast(p, ctypes.POINTER(ctypes.c_int32))

    def call(m=4, k=128, n=128, total=4, first=0, local=4, trans=0, dtype=BF16, x=p, xs=p, a=p, s=p, gs=i32, y=p):
        return lib.rd_gmm_float8(NOW, x, xs, a, s, gs, y, m, k, n, total, first, local, trans, dtype)

    assert call(m=0) == 0 and call(n=0) == 0
    for bad in (dict(m=-1), dict(m=1 << 25), dict(k=-1), dict(n=(1 << 22) + 1), dict(local=0), dict(first=1), dict(first=-1), dict(total=0), dict(dtype=F8),
                dict(x=None), dict(xs=None), dict(a=None), dict(s=None), dict(gs=None), dict(y=None), dict(x=p + 8), dict(xs=p + 8), dict(a=p + 8)):
        assert call(**bad) == INVALID, bad
    assert call(k=1 << 16, n=1 << 15, local=1, total=1) == UNSUPPORTED and b"2 GiB" in lib.rd_last_error()
    assert call(m=(1 << 25) - 1, n=1 << 22, k=128, total=1, local=1, trans=1) == UNSUPPORTED


def test_orthogonalize():
    p = HERE
    one = (ctypes.c_double * 3)(3.4445, -4.775, 2.0315)

    def call(g=1, k=4, n=4, dtype=F32, G=p, out=p, ws=p, ws_bytes=None, steps=1, c=one, eps=1e-7, scale=1.0, spec=True):
        s = _capi.OrthoSpec(steps, c, eps, scale)
        have = lib.rd_orthogonalize_workspace_bytes(g, k, n, dtype) if ws_bytes is None else ws_bytes
        return lib.rd_orthogonalize(NOW, G, out, g, k, n, ctypes.byref(s) if spec else None, dtype, ws, have)

    assert call(g=0) == 0 and call(k=0) == 0 and call(n=0) == 0
    none = (ctypes.c_double * 3)(float("inf"), 0.0, 0.0)
    for bad in (dict(g=-1), dict(dtype=F8), dict(G=None), dict(out=None), dict(spec=False), dict(steps=-1), dict(steps=33), dict(c=None), dict(eps=-1.0),
                dict(eps=float("nan")), dict(scale=float("inf")), dict(c=none)):
        assert call(**bad) == INVALID, bad
    two = (ctypes.c_double * 9)(*([30.0, 0.0, 0.0] * 3))
    assert call(steps=3, c=two) == INVALID and b"converge" in lib.rd_last_error()
    assert call(ws=None) == WORKSPACE and call(ws=p + 16) == WORKSPACE and call(ws_bytes=64) == WORKSPACE
    assert call(k=1 << 16, n=1 << 15) == UNSUPPORTED and call(k=1 << 30, n=1 << 30) == UNSUPPORTED
    assert lib.rd_orthogonalize_workspace_bytes(1, 1 << 30, 4, F32) == 0


def test_python_arguments():
    codes = torch.zeros(2, 130, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    packed = rd.pack_float8(codes, torch.ones(2, 2, 1))
    assert packed.codes.shape == (2, 256, 128) and packed.scales.shape == (2, 2, 1) and packed[2:] == (130, 64)
    whole = torch.zeros(1, 128, 256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert rd.pack_float8(whole, torch.ones(1, 1, 2)).codes.data_ptr() == whole.data_ptr()
    with pytest.raises(ValueError):
        rd.pack_float8(codes, torch.ones(2, 1, 1))
    with pytest.raises(TypeError):
        rd.pack_float8(codes.view(torch.uint8), torch.ones(2, 2, 1))
    with pytest.raises(TypeError):
        rd.pack_float8(codes, torch.ones(2, 2, 1, dtype=torch.int32))
    with pytest.raises(AssertionError):
        rd.pack_float8(codes[0], torch.ones(2, 1))
    with pytest.raises(RuntimeError):
        rd.quantize_rows(torch.ones(2, 2))
    with pytest.raises(TypeError):
        rd.dequantize(packed, torch.float64)
    with pytest.raises(RuntimeError):
        rd.dequantize(packed)
    with pytest.raises(RuntimeError):
        rd.orthogonalize(torch.ones(2, 2))
    with pytest.raises(ValueError):
        rd.orthogonalize(torch.ones(2, 2), coefficients=())
