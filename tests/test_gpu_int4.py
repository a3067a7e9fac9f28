"""Ragged products on 4-bit weights against float64."""

import numpy as np
import pytest
import torch

import gpu_ragged_dot_amd as rd
from oracle import expert_ops_oracle as oracle

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.bfloat16, torch.float16]


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


def _check(seed, m, k, n, sizes, block=128, zeros=False, dtype=torch.bfloat16, scale_dtype=None, trans_rhs=False):
    print(f"int4 m {m} k {k} n {n} g {len(sizes)} block {block} zeros {zeros} {dtype}", flush=True)
    q, s, z = _weights(seed, len(sizes), k, n, block, zeros, scale_dtype or dtype)
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()
    w = _pack(q, s, z, block, trans_rhs)
    y = rd.ragged_dot_int4(x, w, torch.tensor(sizes, dtype=torch.int32, device="cuda"))
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
@pytest.mark.parametrize("block,zeros", [(128, False), (64, True), (32, False)])
def test_many_rows(m, k, n, sizes, block, zeros, dtype):
    _check(m * 3 + k, m, k, n, sizes, block, zeros, dtype)


@pytest.mark.parametrize("sizes,m", [([0, 0, 0], 20), ([3, 4, 5], 40), ([30, 30, 30], 50), ([0, 0, 9], 9), ([-5, 4, 2], 10), ([7, 1000000, 3], 33)])
def test_tails_and_sums_beyond_the_rows(sizes, m):
    """Rows behind the last group are zero whatever was there, groups end at row m, negative sizes count as none."""
    _check(1, m, 200, 72, sizes, 64, True)


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
def test_scale_types(m, scale_dtype, dtype):
    _check(4, m, 320, 130, [m // 2, m - m // 2], 32, True, dtype, scale_dtype)


@pytest.mark.parametrize("m", [12, 700])
def test_a_slice_of_the_groups(m):
    sizes = [m // 4, 0, m // 4, m // 8, m // 8]
    w, x, y = _check(6, m, 256, 80, sizes, 64, True)
    gs = torch.tensor(sizes, dtype=torch.int32, device="cuda")
    part = w._replace(codes=w.codes[1:4].contiguous(), scales=w.scales[1:4].contiguous(), zeros=w.zeros[1:4].contiguous())
    got = rd.ragged_dot_int4(x, part, gs, group_offset=1)
    want = y.clone()
    want[:sizes[0]] = 0
    want[sum(sizes[:4]):] = 0
    assert torch.equal(got, want)


@pytest.mark.parametrize("m", [20, 520])
def test_a_row_does_not_see_its_neighbours(m):
    w, x, y = _check(9, m, 256, 96, [m - 5, 3, 2])
    spoilt = x.clone()
    spoilt[3], spoilt[7, 11] = torch.nan, torch.inf
    got = rd.ragged_dot_int4(spoilt, w, torch.tensor([m - 5, 3, 2]))
    assert not got[3].isfinite().any() and not got[7].isfinite().any()
    rest = [i for i in range(m) if i not in (3, 7)]
    assert torch.equal(got[rest], y[rest])


@pytest.mark.parametrize("m", [16, 400])
def test_strides_addresses_and_empty_calls(m):
    w, x, y = _check(13, m, 136, 48, [m // 2, m - m // 2])
    gs = torch.tensor([m // 2, m - m // 2])
    wide = torch.randn(m, 272, device="cuda").bfloat16()
    wide[:, ::2] = x
    assert torch.equal(rd.ragged_dot_int4(wide[:, ::2], w, gs), y)
    odd = torch.empty(m * 136 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(m, 136).copy_(x)
    assert torch.equal(rd.ragged_dot_int4(odd, w, gs.long().cuda()), y)
    assert rd.ragged_dot_int4(x[:0], w, torch.tensor([0, 0])).shape == (0, 48)
    none = rd.pack_int4(torch.empty((2, 0, 48), dtype=torch.uint8, device="cuda"), torch.empty((2, 0, 48), device="cuda").half())
    assert not rd.ragged_dot_int4(x[:, :0], none, gs).any()


def test_replayed_on_new_sizes_and_on_another_stream():
    w, x, _ = _check(17, 300, 512, 192, [100, 100, 100])
    gs = torch.tensor([100, 100, 100], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = rd.ragged_dot_int4(x, w, gs)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, rd.ragged_dot_int4(x, w, gs))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = rd.ragged_dot_int4(x, w, gs)
    for sizes in ([0, 300, 0], [1, 2, 3], [299, 0, 1], [0, 0, 0]):
        gs.copy_(torch.tensor(sizes))
        x.copy_(torch.randn(300, 512, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, rd.ragged_dot_int4(x, w, gs))


def test_codes_beyond_32_bit_offsets():
    """More than 2^31 codes and 2^32 bytes of them in one tensor: the last groups, as weights of their own."""
    g, k, n = 36, 4096, 65600
    codes = torch.randint(-2 ** 31, 2 ** 31 - 1, (g, n // 16, k // 128, 64, 4), dtype=torch.int32, device="cuda")
    scales = torch.rand((g, k // 128, n, 1), device="cuda").bfloat16()
    assert codes.numel() * 4 > 2 ** 32
    w = rd.Int4Weights(codes, scales, None, k, n, 128)
    for m in (8, 300):
        x = torch.randn(m, k, device="cuda").bfloat16()
        gs = torch.zeros(g, dtype=torch.int32, device="cuda")
        gs[g - 1] = m
        y = rd.ragged_dot_int4(x, w, gs)
        last = rd.Int4Weights(codes[g - 1:].contiguous(), scales[g - 1:].contiguous(), None, k, n, 128)
        assert torch.equal(y, rd.ragged_dot_int4(x, last, gs[g - 1:].contiguous()))
