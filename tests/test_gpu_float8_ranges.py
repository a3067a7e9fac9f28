"""The product on float8 with scales anywhere in float32's range, and contractions of more than 64 blocks, against 64 bits."""

import numpy as np
import pytest
import torch

import gpu_ragged_dot_amd as rd

pytestmark = pytest.mark.gpu

# m, n, groups: launches of tiles of 64 x 64, 64 x 128, 128 x 128 and 256 x 256, the last with tiles of every height
LAUNCHES = [(5, 256, [2, 3]), (160, 512, [4] * 40), (1500, 2500, [257, 31, 200, 640, 128, 96, 140]), (2600, 4100, [900, 300, 1, 0, 256, 64, 700])]
launches = pytest.mark.parametrize("m,n,sizes", LAUNCHES, ids=["64x64", "64x128", "128x128", "256x256"])
layouts = pytest.mark.parametrize("trans", [False, True], ids=["nn", "nt"])


def _float8(t):
    return t.to(torch.float8_e4m3fn)


def _products(x, w, sizes, trans):
    """Of float64 numbers, and of their magnitudes."""
    n, row = w.shape[1 if trans else 2], 0
    ref, mag = torch.zeros(2, len(x), n, dtype=torch.float64, device="cuda")
    for e, size in enumerate(sizes):
        at = slice(row, row + size)
        wk = w[e].t().contiguous() if trans else w[e]
        ref[at], mag[at] = x[at] @ wk, x[at].abs() @ wk.abs()
        row += size
    return ref, mag


@layouts
@launches
@pytest.mark.parametrize("extreme", [True, False], ids=["far", "near"])
def test_scales_of_any_size(m, n, sizes, trans, extreme):
    """Pairs of scales whose product is beyond float32, less than its least normal number, or 0 in it, beside ordinary ones, where the codes
    keep what comes out a float32: codes of 256 for small scales and of 2^-9 for large ones, all those of a block in a row the same or 0,
    so that the sums of a block are exact.  A row whose codes are 0 in a block gets nothing from it, whatever its scale."""
    print(f"scales {m} x {n} {len(sizes)} groups trans={trans}", flush=True)
    k, g = 384, len(sizes)
    kb, nb = k // 128, -(-n // 128)
    rng = np.random.default_rng(m + trans)
    rows = rng.choice([-90, -70, 0, 65] if extreme else [0], m)
    cols = rng.choice([-70, 0, 65] if extreme else [0], (g, nb))
    steps = rng.integers(-20, 21, kb)
    sx = np.ldexp(rng.uniform(1, 2, (m, kb)), rows[:, None] + steps).astype(np.float32)
    sw = np.ldexp(rng.uniform(1, 2, (g, kb, nb)), cols[:, None, :] - steps[:, None]).astype(np.float32)
    cx = rng.integers(-1, 2, (m, k)) * np.where(rows > 0, 2.0 ** -9, 256.0)[:, None]
    cx[rng.random((m, kb)).repeat(128, 1) < 0.2] = 0
    cw = rng.integers(-1, 2, (g, k, n)) * np.where(cols > 0, 2.0 ** -9, 256.0).repeat(128, 1)[:, None, :n]
    sx, sw, cx, cw = (torch.from_numpy(t).cuda() for t in (sx, sw, cx, cw))
    x64 = cx * sx.double().repeat_interleave(128, 1)
    w64 = cw * sw.double().repeat_interleave(128, 1).repeat_interleave(128, 2)[:, :, :n]
    if trans:
        cw, sw, w64 = (t.transpose(1, 2).contiguous() for t in (cw, sw, w64))
    held = rd.Float8Rows(_float8(cx.float()), torch.nn.functional.pad(sx, (0, -kb % 4)).contiguous(), k)
    weights = rd.pack_float8(_float8(cw.float()), sw)
    y = rd.ragged_dot_float8(held, weights, torch.tensor(sizes, dtype=torch.int32, device="cuda"), trans_rhs=trans, out_dtype=torch.float32)
    ref, mag = _products(x64, w64, sizes, trans)
    # per block three roundings of factors and products and one of the sum; what is below the normal numbers is rounded to 2^-149
    off = (y.double() - ref).abs() - (4 * kb * 2.0 ** -24 * mag + 4 * kb * 2.0 ** -149)
    assert not y.isnan().any() and (off <= 0).all(), (int((off > 0).sum()), float(off.max()))


@layouts
def test_scales_that_are_no_numbers_or_zero(trans):
    """A block's scale is NaN, infinite or 0: its row or its columns are what products with it are."""
    k, n = 384, 300
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, A = torch.randn(70, k, generator=gen, device="cuda"), torch.randn((2, n, k) if trans else (2, k, n), generator=gen, device="cuda")
    gs = torch.tensor([30, 35], dtype=torch.int32, device="cuda")
    q, w = rd.quantize_rows(x), rd.quantize_weights(A)
    want = rd.ragged_dot_float8(q, w, gs, trans_rhs=trans, out_dtype=torch.float32)
    sx, sw = q.scales.clone(), w.scales.clone()
    sx[3, 1], sx[40, 2], sx[50] = torch.nan, torch.inf, 0
    sw[0, 0, 0] = torch.nan
    y = rd.ragged_dot_float8(q._replace(scales=sx), w._replace(scales=sw), gs, trans_rhs=trans, out_dtype=torch.float32)
    assert y[3].isnan().all() and not y[40].isfinite().any() and not y[50].any() and y[:30, :128].isnan().all()
    same = torch.ones(70, n, dtype=torch.bool, device="cuda")
    same[[3, 40, 50]] = False
    same[:30, :128] = False
    assert torch.equal(y[same], want[same])


def _uneven(shape, axis, exponents, seed):
    """Normal numbers whose blocks of 128 along ``axis`` differ by powers of two."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    by = torch.from_numpy(np.exp2(exponents)).cuda().float().repeat_interleave(128)[:shape[axis]]
    return torch.randn(shape, generator=gen, device="cuda") * by.view([-1 if i == axis else 1 for i in range(len(shape))])


@launches
@pytest.mark.parametrize("k", [8193, 8320, 14336])
def test_contractions_of_more_than_64_blocks(m, n, sizes, k):
    """Weights [k, n], whose columns' scales are held 64 blocks at a time.  The scales differ from block to block by powers of two, the rows'
    the other way round, so that every block counts alike and the scale of another one would show."""
    print(f"long {m} x {k} x {n} {len(sizes)} groups", flush=True)
    exponents = np.random.default_rng(k).integers(-12, 13, -(-k // 128)).astype(np.float64)
    x, A = _uneven((m, k), 1, -exponents, 1), _uneven((len(sizes), k, n), 1, exponents, 2)
    q, w = rd.quantize_rows(x), rd.quantize_weights(A)
    y = rd.ragged_dot_float8(q, w, torch.tensor(sizes, dtype=torch.int32, device="cuda"), out_dtype=torch.float32)
    ref, mag = _products(rd.dequantize(q, torch.float32).double(), rd.dequantize(w, torch.float32).double(), sizes, False)
    # of eight products at most seven lose 2^-13 of the largest of them: less than 2^-10 of their sum; then fp32 sums
    assert ((y.double() - ref).abs() <= (2.0 ** -10 + k * 2.0 ** -24) * mag).all()


@pytest.mark.parametrize("m,sizes", [(6, [2, 4]), (300, [100, 200]), (1500, [1500])])
def test_gradient_of_rows_over_more_than_64_blocks(m, sizes):
    """Weights [n, k] of n beyond 8192: the rows' gradient is a product on them as [k, n]."""
    k, n = 300, 9000
    print(f"long gradient {m}", flush=True)
    exponents = np.random.default_rng(n).integers(-12, 13, -(-n // 128)).astype(np.float64)
    x = torch.randn(m, k, device="cuda").requires_grad_()
    A, dy = _uneven((len(sizes), n, k), 1, exponents, 3), _uneven((m, n), 1, -exponents, 4)
    w, gs = rd.quantize_weights(A), torch.tensor(sizes, dtype=torch.int32, device="cuda")
    dx, = torch.autograd.grad(rd.ragged_dot_float8(x, w, gs, trans_rhs=True), x, dy)
    ref, mag = _products(rd.dequantize(rd.quantize_rows(dy), torch.float32).double(), rd.dequantize(w, torch.float32).double(), sizes, False)
    assert ((dx.double() - ref).abs() <= (2.0 ** -10 + n * 2.0 ** -24) * mag).all()
