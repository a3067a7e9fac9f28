"""Numbers held as float8 with a scale for each block of 128, and the ragged product on them, against 64 bits."""

import numpy as np
import pytest
import torch

import gpu_ragged_dot_amd as rd
from gpu_ragged_dot_amd import moe
from oracle import float8_oracle as oracle
from oracle import moe_glue_oracle

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LEAST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
types = pytest.mark.parametrize("dtype", list(TYPES.values()), ids=list(TYPES))


def _np(t):
    return t.detach().double().cpu().numpy()


def _within(got, ref, bound):
    off = np.abs(got - ref) / bound
    over = np.isinf(got) & (np.sign(got) == np.sign(ref)) & (np.abs(ref) + bound >= 65520)  # what float16 rounds to infinity
    off[over] = 0
    worst = np.unravel_index(np.argmax(np.where(np.isnan(off), np.inf, off)), off.shape)
    assert off[worst] <= 1, f"{(off > 1).sum()} of {off.size} off, at {worst} {got[worst]} for {ref[worst]}, {off[worst]:.3} times what it may be"


def _rows(m, k, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=gen) * (2 * torch.randn((m, 1), generator=gen)).exp()
    return x.to(dtype).cuda()


def _expect_rows(held, x64, pow2):
    """Codes and scales, the padding included, bit for bit."""
    m, k = x64.shape
    q, s = oracle.quantize(x64, pow2=pow2)
    assert held.k == k and held.codes.shape == (m, -(-k // 128) * 128) and held.scales.shape == (m, -(-k // 512) * 4)
    codes, scales = _np(held.codes.float()), _np(held.scales)
    assert np.array_equal(scales[:, :s.shape[1]], s, equal_nan=True) and not scales[:, s.shape[1]:].any()
    assert np.array_equal(codes[:, :k], q, equal_nan=True)
    assert not held.codes.view(torch.uint8)[:, k:].any() or np.isnan(s).any()


@types
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 7), (5, 129), (64, 2048), (33, 1515), (2, 8192), (257, 500), (1000, 64)])
def test_rows(m, k, pow2, dtype):
    print(f"rows {m} x {k} {dtype} {pow2}", flush=True)
    x = _rows(m, k, dtype, m + k)
    held = rd.quantize_rows(x, pow2=pow2)
    _expect_rows(held, _np(x), pow2)
    for out in TYPES.values():
        got, ref = _np(rd.dequantize(held, out)), oracle.held(_np(x), pow2=pow2)
        ref = np.where(np.abs(ref) > torch.finfo(out).max, np.copysign(np.inf, ref), ref)
        with np.errstate(invalid="ignore"):
            assert np.all((got == ref) | (np.abs(got - ref) <= HALF_ULP[out] * np.abs(ref) * (1 + 2.0 ** -20) + 2.0 ** -24 * np.abs(ref) + LEAST[out]))


@pytest.mark.parametrize("pow2", [False, True])
def test_rows_at_the_edges_of_the_types(pow2):
    """Zeros, subnormals, the largest numbers, ties between codes, infinities and NaN; rows at odd addresses."""
    top = torch.finfo(torch.float32).max
    x = torch.zeros(12, 300)
    x[1, :5] = torch.tensor([1e-45, -1e-40, 1e-38, 1e-30, -0.0])
    x[2, 128:131] = torch.tensor([top, -top, 1.0])
    x[3] = torch.arange(300) * 2.0 ** -83
    x[4, :256] = torch.arange(256) * 0.5     # halves of steps of the codes
    x[4, 255] = 448.0
    x[5, 7], x[6, 200], x[7, 299] = torch.inf, torch.nan, -torch.inf
    x[8] = 2.0 ** -80
    x[9] = torch.linspace(-448, 448, 300)
    x[10, :17] = 1 + torch.arange(17) / 16
    x[11] = 3.0
    _expect_rows(rd.quantize_rows(x.cuda(), pow2=pow2), x.double().numpy(), pow2)
    flat = torch.zeros(12 * 300 + 1, device="cuda")
    flat[1:] = x.flatten().cuda()
    _expect_rows(rd.quantize_rows(flat[1:].view(12, 300), pow2=pow2), x.double().numpy(), pow2)
    _expect_rows(rd.quantize_rows(x.cuda()[::2, 1::3], pow2=pow2), x.double().numpy()[::2, 1::3], pow2)


def test_quotients_next_to_borders_of_codes():
    """Float32 rows whose quotients lie a few units of 2^-24 around the middles between two codes, for many scales."""
    rng = np.random.default_rng(3)
    top = np.float32(1) + np.arange(4096, dtype=np.float32) / np.float32(4096)
    s = top / np.float32(448)
    t = np.float32(1 + (2 * rng.integers(0, 8, (4096, 127)) + 1) / 16.0)
    x = (s[:, None] * t * 2.0 ** rng.integers(0, 8, (4096, 127))).astype(np.float32)
    x = (x.view(np.int32) + rng.integers(-2, 3, x.shape).astype(np.int32)).view(np.float32)
    x = np.concatenate([x, top[:, None]], 1)
    x = np.minimum(x, top[:, None])
    _expect_rows(rd.quantize_rows(torch.from_numpy(x).cuda()), x.astype(np.float64), False)


@types
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("g,a,b", [(1, 1, 1), (2, 128, 256), (3, 130, 100), (5, 257, 1515), (1, 1000, 8)])
def test_weights(g, a, b, pow2, dtype):
    print(f"weights {g} x {a} x {b} {dtype} {pow2}", flush=True)
    A = _rows(g * a, b, dtype, a).view(g, a, b)
    held = rd.quantize_weights(A, pow2=pow2)
    assert held.rows == a and held.cols == b
    back = _np(rd.dequantize(held, torch.float32))
    for e in range(g):
        q, s = oracle.quantize(_np(A[e]), 128, pow2)
        assert np.array_equal(_np(held.scales[e]), s)
        assert np.array_equal(_np(held.codes[e].float())[:a, :b], q)
        assert np.array_equal(back[e], oracle.values(q, s, 128).astype(np.float32))
    pad = held.codes.view(torch.uint8)
    assert not pad[:, a:].any() and not pad[:, :, b:].any()
    packed = rd.pack_float8(held.codes[:, :a, :b], held.scales)
    assert torch.equal(packed.codes.view(torch.uint8), pad) and torch.equal(packed.scales, held.scales) and packed[2:] == (a, b)


@types
@pytest.mark.parametrize("tokens,top_k,d,g", [(1, 1, 5, 1), (8, 8, 2048, 128), (33, 3, 130, 5), (257, 2, 1001, 7)])
def test_dispatch(tokens, top_k, d, g, dtype):
    print(f"dispatch {tokens} x {top_k} {d} {g} {dtype}", flush=True)
    ids = torch.from_numpy(np.random.default_rng(tokens).integers(-1, g, (tokens, top_k)).astype(np.int32)).cuda()
    h, r = _rows(tokens, d, dtype), moe.route(ids, g)
    want = moe_glue_oracle.dispatch(_np(h), r.slot_of_row.cpu().numpy(), top_k)
    for pow2 in (False, True):
        _expect_rows(moe.dispatch(h, r, float8=True, pow2=pow2), want, pow2)


@types
@pytest.mark.parametrize("rows,f", [(1, 1), (64, 768), (5, 1515), (257, 130)])
def test_swiglu(rows, f, dtype):
    """Against the quantised activation in 64 bits: an activation next to a border of two codes may fall to either side, and a scale
    of 24 bits differ in its last ones."""
    print(f"swiglu {rows} x {f} {dtype}", flush=True)
    y = _rows(rows, 2 * f, dtype, f).clamp(-60, 60)
    yn = _np(y)
    ref = yn[:, :f] / (1 + np.exp(-yn[:, :f])) * yn[:, f:]
    for pow2 in (False, True):
        held = moe.swiglu(y, float8=True, pow2=pow2)
        got, s = _np(rd.dequantize(held, torch.float32)), _np(held.scales)[:, :-(-f // 128)]
        unit = (8 + 2 * np.abs(yn[:, :f]).max()) * 2.0 ** -23  # of the activation, relative (the exponential's argument first)
        q, s_ref = oracle.quantize(ref, pow2=pow2)
        if not pow2:
            assert np.all(np.abs(s - s_ref) <= (unit + 2.0 ** -23) * s_ref)
        wide = np.repeat(s, 128, 1)[:, :f]
        # half a step of the codes: 2^-4 of a number, 2^-10 of a scale for the least ones
        assert np.all(np.abs(got - ref) <= np.maximum(2.0 ** -4 * np.abs(ref), 2.0 ** -10 * wide) * (1 + 32 * unit))
        assert held.k == f and not held.codes.view(torch.uint8)[:, f:].any()


def _largest_of_eight(x, axis):
    """Of every eight neighbours' magnitudes along the contraction."""
    pad = [(0, 0)] * x.ndim
    pad[axis] = (0, -x.shape[axis] % 8)
    x = np.abs(np.pad(x, pad))
    return x.reshape(*x.shape[:axis], x.shape[axis] // 8, 8, *x.shape[axis + 1:]).max(axis + 1)


def _bound(x8, A8, sizes, trans, ref, dtype):
    """The matrix-core instruction cuts the products of eight neighbouring indices at 2^-13 of the exponent of the largest of them,
    which is no more than that product, before it adds them: seven lose less than a unit each.  What they make is summed in fp32,
    in blocks of 128 and over the blocks, behind factors rounded twice."""
    k = x8.shape[1]
    magnitude = oracle.ragged_dot(np.abs(x8), np.abs(A8), sizes, trans)
    eights = oracle.ragged_dot(_largest_of_eight(x8, 1), _largest_of_eight(A8, 2 if trans else 1), sizes, trans)
    return 7 * 2.0 ** -13 * eights + (k / 8 + 24) * 2.0 ** -23 * magnitude + HALF_ULP[dtype] * np.abs(ref) + LEAST[dtype]


def _check_product(m, k, n, sizes, trans, dtype, pow2=False, held=True, seed=0):
    g = len(sizes)
    gen = torch.Generator().manual_seed(seed)
    x = _rows(m, k, dtype, seed)
    A = torch.randn((g, n, k) if trans else (g, k, n), generator=gen).to(dtype).cuda()
    sizes_t = torch.tensor(sizes, dtype=torch.int32, device="cuda")
    rows, weights = (rd.quantize_rows(x, pow2=pow2), rd.quantize_weights(A, pow2=pow2)) if held else (x, A)
    y = rd.ragged_dot_float8(rows, weights, sizes_t, trans_rhs=trans, out_dtype=dtype, pow2=pow2)
    assert y.dtype == dtype and y.shape == (m, n)
    x8, A8 = oracle.held(_np(x), 1, pow2), np.stack([oracle.held(_np(a), 128, pow2) for a in A])
    ref = oracle.ragged_dot(x8, A8, sizes, trans)
    _within(_np(y), ref, _bound(x8, A8, sizes, trans, ref, dtype))
    return y


SHAPES = [(1, 1, 1, [1]), (5, 128, 128, [5]), (64, 2048, 768, [0, 3, 1, 0, 60]), (515, 1001, 1515, [100, 0, 200, 7, 150]), (33, 257, 129, [32, 1]),
          (300, 130, 300, [1, 255, 40]), (1024, 512, 520, [256, 513, 100, 155]), (700, 64, 1000, [700]), (40, 1280, 256, [10, 10, 20]),
          (200, 300, 200, [-5, 120, 0, 500]), (129, 640, 384, [129] + [0] * 300), (800, 384, 640, [1] * 400 + [0, 7])]


@pytest.mark.parametrize("trans", [False, True], ids=["nn", "nt"])
@pytest.mark.parametrize("m,k,n,sizes", SHAPES)
def test_product(m, k, n, sizes, trans):
    print(f"product {m} {k} {n} {len(sizes)} groups trans={trans}", flush=True)
    for i, dtype in enumerate(TYPES.values()):
        _check_product(m, k, n, sizes, trans, dtype, pow2=i == 1, held=i != 2, seed=i)


# Launches large enough for tiles of 128 x 128 (the first three) and of 256 x 256, with tiles of every height left over, contractions
# of one block, of few and of more than the rings of slabs and scales hold.
FILLED = [(2500, 1300, 2304, [700, 129, 0, 65, 33, 1, 1000, 500]), (1500, 130, 2500, [257, 31, 200, 640, 128, 96, 140]),
          (3900, 700, 1100, [130] * 10 + [0, 1, 400, 63] * 5), (2600, 700, 4100, [900, 300, 1, 0, 256, 64, 700]),
          (2600, 1156, 2100, [130, 127, 128, 0, 257, 1, 64, 65, 500, 17] * 2), (5000, 100, 2100, [513, 300, 200, 1000, 40, 700, 0, 1500, 129, 255])]


@pytest.mark.parametrize("trans", [False, True], ids=["nn", "nt"])
@pytest.mark.parametrize("m,k,n,sizes", FILLED)
def test_product_that_fills_the_device(m, k, n, sizes, trans):
    print(f"product {m} {k} {n} {len(sizes)} groups trans={trans}", flush=True)
    for i, dtype in enumerate(TYPES.values()):
        _check_product(m, k, n, sizes, trans, dtype, pow2=i == 1, held=i != 2, seed=i)


def test_no_rows_no_columns_no_contraction():
    gs = torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    for m, k, n in ((0, 64, 32), (4, 0, 32), (4, 64, 0)):
        y = rd.ragged_dot_float8(torch.ones(m, k, device="cuda"), torch.ones(2, k, n, device="cuda"), gs)
        assert y.shape == (m, n) and not y.any()
        assert rd.dequantize(rd.quantize_rows(torch.ones(m, k, device="cuda"))).shape == (m, k)


def test_a_slice_of_the_groups():
    sizes = [3, 70, 0, 5, 90, 2]
    x, A, gs = _rows(180, 256, torch.bfloat16), torch.randn(6, 256, 384, device="cuda").bfloat16(), torch.tensor(sizes, device="cuda", dtype=torch.int32)
    whole = rd.ragged_dot_float8(x, A, gs)
    w = rd.quantize_weights(A)
    for first, count in ((0, 6), (1, 3), (3, 3), (2, 1), (0, 1)):
        part = rd.Float8Weights(w.codes[first:first + count], w.scales[first:first + count], w.rows, w.cols)
        lo, hi = sum(sizes[:first]), sum(sizes[:first + count])
        want = torch.zeros_like(whole)
        want[lo:hi] = whole[lo:hi]
        assert torch.equal(rd.ragged_dot_float8(x, part, gs, group_offset=first), want)
        xg, Ag = x.clone().requires_grad_(), A[first:first + count].clone().requires_grad_()
        dx, dA = torch.autograd.grad(rd.ragged_dot_float8(xg, Ag, gs, group_offset=first), (xg, Ag), torch.ones_like(whole))
        assert not dx[:lo].any() and not dx[hi:].any() and dA.shape == Ag.shape and (lo == hi or dx[lo:hi].any())


@pytest.mark.parametrize("trans", [False, True], ids=["nn", "nt"])
@pytest.mark.parametrize("m,k,n,sizes", [(40, 256, 384, [10, 0, 25]), (515, 1001, 130, [100, 0, 200, 7, 150]), (1500, 300, 520, [700, 1, 799])])
def test_gradients(m, k, n, sizes, trans):
    """dx: of the quantised cotangent with the quantised weights; dA: of the rows and the cotangent as they are."""
    print(f"gradients {m} {k} {n} trans={trans}", flush=True)
    for pow2, dtype in ((False, torch.bfloat16), (True, torch.float16), (False, torch.float32)):
        x, dy = _rows(m, k, dtype, 1).clamp(-100, 100).requires_grad_(), _rows(m, n, dtype, 2).clamp(-100, 100)
        A = torch.randn((len(sizes), n, k) if trans else (len(sizes), k, n), generator=torch.Generator().manual_seed(3)).to(dtype).cuda().requires_grad_()
        gs = torch.tensor(sizes, dtype=torch.int32, device="cuda")
        y = rd.ragged_dot_float8(x, A, gs, trans_rhs=trans, pow2=pow2)
        dx, dA = torch.autograd.grad(y, (x, A), dy, retain_graph=True)
        assert dx.dtype == dtype and dA.dtype == dtype
        only_x, = torch.autograd.grad(rd.ragged_dot_float8(x, rd.quantize_weights(A.detach(), pow2=pow2), gs, trans_rhs=trans, pow2=pow2), x, dy)
        assert torch.equal(only_x, dx)
        d8, A8 = oracle.held(_np(dy), 1, pow2), np.stack([oracle.held(_np(a), 128, pow2) for a in A])
        ref = oracle.ragged_dot(d8, A8, sizes, not trans)
        _within(_np(dx), ref, _bound(d8, A8, sizes, not trans, ref, dtype))
        row = 0
        for e, size in enumerate(sizes):
            xs, ds = _np(x)[row:row + size], _np(dy)[row:row + size]
            ref, mag = ((f(ds).T @ f(xs) if trans else f(xs).T @ f(ds)) for f in (lambda t: t, np.abs))
            _within(_np(dA[e]), ref, (size + 8) * 2.0 ** -23 * mag + HALF_ULP[dtype] * np.abs(ref) + LEAST[dtype])
            row += size


def test_infinities_and_nan_stay_in_their_rows_and_columns():
    x, A = _rows(6, 300, torch.float32).clamp(-9, 9), torch.randn(2, 300, 300, device="cuda")
    x[1, 5], x[4, 299], A[1, 140, 7] = torch.inf, torch.nan, torch.nan
    y = rd.ragged_dot_float8(x, A, torch.tensor([2, 3], dtype=torch.int32, device="cuda"))
    want = torch.zeros(6, 300, dtype=torch.bool, device="cuda")
    want[[1, 4]] = True
    want[2:5, :128] = True  # the block of 128 x 128 that holds the NaN
    assert torch.equal(y.isnan(), want) and not y[5].any()


def test_rows_past_the_groups_are_not_read():
    x, A = _rows(50, 256, torch.bfloat16), torch.randn(2, 256, 128, device="cuda").bfloat16()
    x[30:] = torch.nan
    y = rd.ragged_dot_float8(x, A, torch.tensor([20, 10], dtype=torch.int32, device="cuda"))
    assert not y[30:].any() and not y.isnan().any()


def test_refusals():
    x, A = torch.randn(4, 128, device="cuda"), torch.randn(2, 128, 256, device="cuda")
    gs = torch.tensor([2, 2], dtype=torch.int32, device="cuda")
    w, q = rd.quantize_weights(A), rd.quantize_rows(x)
    with pytest.raises(AssertionError, match="contraction"):
        rd.ragged_dot_float8(x, A, gs, trans_rhs=True)
    with pytest.raises(AssertionError, match="contraction"):
        rd.ragged_dot_float8(q, w, gs, trans_rhs=True)
    with pytest.raises(TypeError):
        rd.ragged_dot_float8(x.bfloat16(), A, gs)
    with pytest.raises(TypeError):
        rd.ragged_dot_float8(x, A, gs, out_dtype=torch.float64)
    with pytest.raises(TypeError):
        rd.quantize_rows(x.double())
    with pytest.raises(ValueError):
        rd.quantize_rows(A)
    with pytest.raises(ValueError):
        rd.quantize_weights(x)
    with pytest.raises(RuntimeError):
        rd.quantize_rows(x.cpu())
    with pytest.raises(RuntimeError):
        rd.ragged_dot_float8(x.cpu(), w, gs)
    with pytest.raises(AssertionError, match="groups"):
        rd.ragged_dot_float8(x, A, gs[:1])
    with pytest.raises(AssertionError, match="quantize_rows"):
        rd.ragged_dot_float8(q._replace(scales=q.scales[:, :1]), w, gs)
    with pytest.raises(AssertionError, match="quantize_weights"):
        rd.ragged_dot_float8(q, w._replace(codes=w.codes[:, :64]), gs)
    with pytest.raises(NotImplementedError):
        rd.quantize_rows(x.clone().requires_grad_())
    with pytest.raises(NotImplementedError):
        rd.ragged_dot_float8(q, A.clone().requires_grad_(), gs)
    with torch.no_grad():
        rd.quantize_rows(x.clone().requires_grad_())
        rd.ragged_dot_float8(q, A.clone().requires_grad_(), gs)
    with pytest.raises(NotImplementedError):
        moe.swiglu(torch.randn(4, 8, device="cuda", requires_grad=True), float8=True)


def test_captured_and_replayed():
    x, A = _rows(300, 512, torch.bfloat16).requires_grad_(), torch.randn(4, 512, 256, device="cuda").bfloat16().requires_grad_()
    gs, dy = torch.tensor([100, 0, 150, 50], dtype=torch.int32, device="cuda"), _rows(300, 256, torch.bfloat16, 9)

    def step():
        y = rd.ragged_dot_float8(x, A, gs)
        return (y.detach(), *torch.autograd.grad(y, (x, A), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        with torch.no_grad():
            x.copy_(_rows(300, 512, torch.bfloat16, 20 + seed))
            gs.copy_(torch.tensor([[100, 0, 150, 50], [1, 2, 3, 4], [0, 0, 300, 0]][seed], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)
