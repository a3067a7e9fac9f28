"""Ragged products on 4-bit weights against float64."""

import numpy as np
import pytest
import torch

import gpu_ragged_dot_amd as rd
from gpu_ragged_dot_amd import _capi
from gpu_ragged_dot_amd.int4 import _ragged_dot_int4
from oracle import expert_ops_oracle as oracle

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.bfloat16, torch.float16]
KERNELS = [_capi.RD_INT4_STREAM, _capi.RD_INT4_TILES]
KERNEL_IDS = ["stream", "tiles"]


def _weights(seed, g, k, n, block, zeros, scale_dtype):
    rng = np.random.default_rng(seed)
    blocks = -(-k // block)
    q = rng.integers(0, 16, (g, k, n)).astype(np.uint8)
    s = torch.from_numpy((rng.uniform(0.5, 1.5, (g, blocks, n)) * rng.choice([-1.0, 1.0], (g, blocks, n)) * max(k, 1) ** -0.5)).to(scale_dtype)
    z = rng.integers(0, 16, (g, blocks, n)).astype(np.uint8) if zeros else None
    return q, s, z


def _pack(q, s, z, block, trans_rhs=False):
    dev = lambda a: None if a is None else torch.as_tensor(a).cuda()
    if trans_rhs:
        turn = lambda a: None if a is None else torch.as_tensor(a).transpose(1, 2).contiguous().cuda()
        return rd.pack_int4(turn(q), turn(s), turn(z), block=block, trans_rhs=True)
    return rd.pack_int4(dev(q), dev(s), dev(z), block=block)


def _product(x, q, s, z, sizes, block):
    """y, and for its error: the sum of |x| |A|, and of |x| |scale| (16 + zero), what the sums of codes and of x amount to."""
    x = x.double().cpu().numpy()
    A = oracle.int4_dense(q, s.double().numpy(), z, block)
    at = np.arange(q.shape[1]) // block
    reach = np.abs(s.double().numpy())[:, at] * (32.0 if z is None else 32.0 + z[:, at].astype(float))
    m, n = x.shape[0], q.shape[2]
    y, absolute, sums = np.zeros((m, n)), np.zeros((m, n)), np.zeros((m, n))
    row = 0
    for e, size in enumerate(sizes):
        end = min(row + max(size, 0), m)
        y[row:end], absolute[row:end], sums[row:end] = x[row:end] @ A[e], np.abs(x[row:end]) @ np.abs(A[e]), np.abs(x[row:end]) @ reach[e]
        row = end
    return y, absolute, sums


def _check(seed, m, k, n, sizes, block=128, zeros=False, dtype=torch.bfloat16, scale_dtype=None, trans_rhs=False, kernel=0):
    print(f"int4 m {m} k {k} n {n} g {len(sizes)} block {block} zeros {zeros} {dtype} kernel {kernel}", flush=True)
    q, s, z = _weights(seed, len(sizes), k, n, block, zeros, scale_dtype or dtype)
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()
    w = _pack(q, s, z, block, trans_rhs)
    y = _ragged_dot_int4(x, w, torch.tensor(sizes, dtype=torch.int32, device="cuda"), kernel=kernel)
    assert y.dtype == dtype and y.shape == (m, n)
    got = y.double().cpu().numpy()
    ref, absolute, sums = _product(x, q, s, z, sizes, block)
    total = min(sum(max(v, 0) for v in sizes), m)
    assert not got[total:].any()
    # The result is rounded once; a weight may be rounded to the rows' type before its product; fp32 sums of k terms, of x and of
    # x times codes, lose at most a rounding of 2^-23 (matrix cores) per term of what they add up.
    half = HALF_ULP[dtype]
    bound = half * np.abs(ref) + 1.01 * half * absolute + (k + 16) * 2.0 ** -23 * sums + 2.0 ** -25
    assert np.all(np.abs(got - ref) <= bound)
    # and all in all: a rounding of the result and independent ones of the weights
    if ref.size >= 1000 and np.any(ref):
        assert np.linalg.norm(got - ref) <= half * np.linalg.norm(ref)
    return w, x, y


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f16"])
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,k,n,sizes", [
    (1, 1, 1, [1]), (1, 128, 64, [1]), (5, 31, 7, [2, 0, 3]), (17, 129, 65, [16, 1]), (3, 7, 100, [1, 1, 1]), (40, 256, 200, [0, 33, 0, 7]),
    (64, 512, 128, [8] * 8), (130, 1001, 333, [1, 64, 15, 17, 33]), (90, 384, 48, [90]), (300, 640, 96, [299, 1])])
def test_shapes(m, k, n, sizes, block, zeros, dtype):
    _check(m + k, m, k, n, sizes, block, zeros, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f16"])
@pytest.mark.parametrize("m,k,n,sizes", [(2000, 512, 384, [700, 0, 1, 129, 1100]), (1025, 1000, 515, [1025]), (700, 2048, 256, [128, 256, 127, 129, 60]),
                                         (513, 136, 1030, [255, 257]), (4096, 256, 256, [1024, 2972])])
@pytest.mark.parametrize("block,zeros", [(128, False), (64, True), (32, False), (128, True), (32, True)])
@pytest.mark.parametrize("kernel", KERNELS, ids=KERNEL_IDS)
def test_many_rows(m, k, n, sizes, block, zeros, dtype, kernel):
    _check(m * 3 + k, m, k, n, sizes, block, zeros, dtype, kernel=kernel)


@pytest.mark.parametrize("k", [8, 9, 63, 64, 65, 127, 128, 129, 191, 255, 256, 257, 385, 640])
@pytest.mark.parametrize("rows", [49, 65, 130, 193, 256, 257])
def test_tile_heights_and_slabs(rows, k):
    """Every height of a tile, the last row and the last contraction index at either side of what a slab holds; n on either side of
    a strip and a tile's columns."""
    n = {49: 256, 65: 255, 130: 17, 193: 300, 256: 513, 257: 16}[rows]
    _check(rows + k, rows + 3, k, n, [rows, 3], 64, True, kernel=_capi.RD_INT4_TILES)


@pytest.mark.parametrize("sizes,k,n", [([600, 300], 2048, 512), ([256] * 3, 4096, 256), ([100], 8192, 700), ([3000, 50, 1], 1024, 2048)])
def test_tiles_cut_along_k(sizes, k, n):
    """Launches that do not fill a round, whose tiles are cut: the same for every call, and without the workspace but for the order
    of the sums."""
    w, x, y = _check(k, sum(sizes), k, n, sizes, kernel=_capi.RD_INT4_TILES)
    gs = torch.tensor(sizes, dtype=torch.int32, device="cuda")
    for _ in range(3):
        assert torch.equal(_ragged_dot_int4(x, w, gs, kernel=_capi.RD_INT4_TILES), y)
    uncut = torch.empty_like(y)
    _capi.check(_capi.lib.rd_gmm_int4(torch.cuda.current_stream().cuda_stream, x.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), None, gs.data_ptr(),
                                      uncut.data_ptr(), sum(sizes), k, n, len(sizes), 0, len(sizes), 128, 0, 0, _capi.RD_INT4_TILES, None, 0))
    assert (uncut.double() - y.double()).norm() <= 2.0 ** -9 * y.double().norm()


def test_float16_rows_with_bfloat16_scales():
    """Scales that float16 does not hold: the weights are not rounded to it, whatever the number of rows."""
    rng = np.random.default_rng(0)
    q, z = rng.integers(0, 16, (1, 256, 64)).astype(np.uint8), None
    s = torch.full((1, 2, 64), 2.0 ** -30).bfloat16()
    x = (torch.randn(300, 256) * 1024).half().cuda()
    for kernel in (0, *KERNELS):
        y = _ragged_dot_int4(x, _pack(q, s, z, 128), torch.tensor([300]), kernel=kernel).double().cpu().numpy()
        ref, _, sums = _product(x, q, s, z, [300], 128)
        assert np.all(np.abs(y - ref) <= 2.0 ** -11 * np.abs(ref) + 272 * 2.0 ** -23 * sums + 2.0 ** -25)


@pytest.mark.parametrize("sizes,m", [([0, 0, 0], 20), ([3, 4, 5], 40), ([30, 30, 30], 50), ([0, 0, 9], 9), ([-5, 4, 2], 10), ([7, 1000000, 3], 33)])
@pytest.mark.parametrize("kernel", KERNELS, ids=KERNEL_IDS)
def test_tails_and_sums_beyond_the_rows(sizes, m, kernel):
    """Rows behind the last group are zero whatever was there, groups end at row m, negative sizes count as none."""
    _check(1, m, 200, 72, sizes, 64, True, kernel=kernel)
    _check(1, 60 * m, 200, 72, [60 * v for v in sizes], 64, True, kernel=kernel)


@pytest.mark.parametrize("g", [255, 256, 257, 300, 600])
def test_many_groups(g):
    rng = np.random.default_rng(g)
    sizes = (rng.random(g) < 0.4).astype(int) * rng.integers(1, 4, g)
    _check(g, int(sizes.sum()) + 5, 128, 40, sizes.tolist())


@pytest.mark.parametrize("k,n", [(1, 16), (127, 33), (128, 64), (129, 20), (300, 65), (1000, 17)])
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("trans_rhs", [False, True])
def test_every_code_is_where_it_belongs(k, n, block, trans_rhs):
    """Rows of the unit matrix times scales that are powers of two: the weights themselves, to the last bit."""
    print(f"unit rows k {k} n {n} block {block}", flush=True)
    rng = np.random.default_rng(k + n)
    blocks = -(-k // block)
    q, z = rng.integers(0, 16, (2, k, n)).astype(np.uint8), rng.integers(0, 16, (2, blocks, n)).astype(np.uint8)
    s = torch.from_numpy(2.0 ** rng.integers(-3, 3, (2, blocks, n))).bfloat16()
    x = torch.eye(k, dtype=torch.bfloat16).repeat(2, 1).cuda()
    y = rd.ragged_dot_int4(x, _pack(q, s, z, block, trans_rhs), torch.tensor([k, k]))
    assert np.array_equal(y.double().cpu().numpy().reshape(2, k, n), oracle.int4_dense(q, s.double().numpy(), z, block))


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f16"])
@pytest.mark.parametrize("scale_dtype", TYPES, ids=["sbf16", "sf16"])
@pytest.mark.parametrize("m", [9, 600])
@pytest.mark.parametrize("kernel", KERNELS, ids=KERNEL_IDS)
def test_scale_types(m, scale_dtype, dtype, kernel):
    _check(4, m, 320, 130, [m // 2, m - m // 2], 32, True, dtype, scale_dtype, kernel=kernel)


@pytest.mark.parametrize("m", [12, 700])
@pytest.mark.parametrize("kernel", KERNELS, ids=KERNEL_IDS)
def test_a_slice_of_the_groups(m, kernel):
    sizes = [m // 4, 0, m // 4, m // 8, m // 8]
    w, x, y = _check(6, m, 256, 80, sizes, 64, True, kernel=kernel)
    gs = torch.tensor(sizes, dtype=torch.int32, device="cuda")
    part = w._replace(codes=w.codes[1:4], scales=w.scales[1:4], zeros=w.zeros[1:4])
    got = _ragged_dot_int4(x, part, gs, group_offset=1, kernel=kernel)
    want = y.clone()
    want[:sizes[0]] = 0
    want[sum(sizes[:4]):] = 0
    assert torch.equal(got, want)


@pytest.mark.parametrize("m", [20, 520])
@pytest.mark.parametrize("kernel", KERNELS, ids=KERNEL_IDS)
def test_a_row_does_not_see_its_neighbours(m, kernel):
    w, x, y = _check(9, m, 256, 96, [m - 5, 3, 2], kernel=kernel)
    spoilt = x.clone()
    spoilt[3], spoilt[7, 11] = torch.nan, torch.inf
    got = _ragged_dot_int4(spoilt, w, torch.tensor([m - 5, 3, 2]), kernel=kernel)
    assert not got[3].isfinite().any() and not got[7].isfinite().any()
    rest = [i for i in range(m) if i not in (3, 7)]
    assert torch.equal(got[rest], y[rest])


@pytest.mark.parametrize("m", [16, 400])
@pytest.mark.parametrize("kernel", KERNELS, ids=KERNEL_IDS)
def test_strides_addresses_and_empty_calls(m, kernel):
    w, x, y = _check(13, m, 136, 48, [m // 2, m - m // 2], kernel=kernel)
    gs = torch.tensor([m // 2, m - m // 2])
    wide = torch.randn(m, 272, device="cuda").bfloat16()
    wide[:, ::2] = x
    assert torch.equal(_ragged_dot_int4(wide[:, ::2], w, gs, kernel=kernel), y)
    odd = torch.empty(m * 136 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(m, 136).copy_(x)
    assert torch.equal(_ragged_dot_int4(odd, w, gs.long().cuda(), kernel=kernel), y)
    shifted = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)
    w_odd = w._replace(scales=shifted(w.scales), zeros=shifted(torch.full_like(w.scales, 8, dtype=torch.uint8)))
    assert torch.equal(_ragged_dot_int4(x, w_odd, gs, kernel=kernel), y)
    assert rd.ragged_dot_int4(x[:0], w, torch.tensor([0, 0])).shape == (0, 48)
    none = rd.pack_int4(torch.empty((2, 0, 48), dtype=torch.uint8, device="cuda"), torch.empty((2, 0, 48), device="cuda").half())
    assert not rd.ragged_dot_int4(x[:, :0], none, gs).any()


@pytest.mark.parametrize("kernel", KERNELS, ids=KERNEL_IDS)
def test_replayed_on_new_sizes_and_on_another_stream(kernel):
    w, x, _ = _check(17, 300, 512, 192, [100, 100, 100], kernel=kernel)
    product = lambda: _ragged_dot_int4(x, w, gs, kernel=kernel)
    gs = torch.tensor([100, 100, 100], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = product()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, product())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = product()
    for sizes in ([0, 300, 0], [1, 2, 3], [299, 0, 1], [0, 0, 0]):
        gs.copy_(torch.tensor(sizes))
        x.copy_(torch.randn(300, 512, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, product())


def test_codes_beyond_32_bit_offsets():
    """More than 2^31 codes and 2^32 bytes of them in one tensor: the last groups, as weights of their own."""
    g, k, n = 36, 4096, 65600
    codes = torch.randint(-2 ** 31, 2 ** 31 - 1, (g, n // 16, k // 128, 64, 4), dtype=torch.int32, device="cuda")
    scales = torch.rand((g, k // 128, n, 1), device="cuda").bfloat16()
    assert codes.numel() * 4 > 2 ** 32
    w = rd.Int4Weights(codes, scales, None, k, n, 128)
    for m, kernel in ((8, 0), (300, KERNELS[0]), (300, KERNELS[1])):
        x = torch.randn(m, k, device="cuda").bfloat16()
        gs = torch.zeros(g, dtype=torch.int32, device="cuda")
        gs[g - 1] = m
        y = _ragged_dot_int4(x, w, gs, kernel=kernel)
        last = rd.Int4Weights(codes[g - 1:].contiguous(), scales[g - 1:].contiguous(), None, k, n, 128)
        assert torch.equal(y, _ragged_dot_int4(x, last, gs[g - 1:].contiguous(), kernel=kernel))
