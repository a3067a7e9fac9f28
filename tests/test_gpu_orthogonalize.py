"""Updates orthogonalised by Newton-Schulz products, against 64 bits."""

import numpy as np
import pytest
import torch

import gpu_ragged_dot_amd as rd
from gpu_ragged_dot_amd.ortho import COEFFICIENTS
from oracle import ortho_oracle as oracle

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
types = pytest.mark.parametrize("dtype", list(TYPES.values()), ids=list(TYPES))


def _np(t):
    return t.double().cpu().numpy()


def _matrix(k, n, kind, seed=0):
    rng = np.random.default_rng(seed + 7 * k + n)
    if kind == "low rank":  # the gradient of an expert that saw few tokens
        q = max(1, min(k, n) // 8)
        return rng.standard_normal((k, q)) @ rng.standard_normal((q, n))
    if kind == "uneven":  # rows and columns of very different sizes
        return np.exp(1.5 * rng.standard_normal((k, 1))) * rng.standard_normal((k, n)) * np.exp(1.5 * rng.standard_normal((1, n)))
    return 1e-3 * rng.standard_normal((k, n))


def _single(G, triples):
    """The iteration in float32."""
    X = G.astype(np.float32)
    X = X if X.shape[0] <= X.shape[1] else X.T.copy()
    X = X * np.float32(1 / (np.sqrt((G * G).sum()) + 1e-7))
    for a, b, c in np.float32(triples):
        A = X @ X.T
        X = a * X + (b * A + c * (A @ A)) @ X
    return X if G.shape[0] <= G.shape[1] else X.T


def _check(got, G, triples, scale=1.0):
    """The norm of what is off is that of the roundings which the kernels are meant to make, computed in 64 bits between them, a quarter
    more for sums in another order; for float32 the larger of that and of the iteration in float32, twice; and the last rounding."""
    dtype, g64 = got.dtype, _np(G)
    ref = scale * oracle.orthogonalize(g64, triples)
    of = lambda y: np.linalg.norm(scale * y - ref)
    two = dtype == torch.float32
    rounding = of(oracle.rounded(g64, triples, two))
    if min(g64.shape) < 16:  # too few numbers for their roundings to average: the worst of a hundred draws of them
        rounding = max(rounding, *(of(oracle.rounded(g64, triples, two, rng=np.random.default_rng(i))) for i in range(100)))
    if two:
        rounding = 2 * max(rounding, of(_single(g64, triples)))
    off = np.linalg.norm(_np(got) - ref)
    norm = np.linalg.norm(ref)
    assert off <= 1.25 * rounding + HALF_ULP[dtype] * norm + 2.0 ** -25 * np.sqrt(ref.size), f"off by {off / norm:.2e}, the roundings by {rounding / norm:.2e}"
    return off / norm if norm else 0.0


@types
@pytest.mark.parametrize("kind", ["gaussian", "low rank", "uneven"])
@pytest.mark.parametrize("k,n", [(1, 1), (1, 300), (300, 1), (64, 64), (63, 65), (128, 130), (200, 129), (256, 512), (515, 100), (257, 1000)])
def test_against_float64(k, n, kind, dtype):
    print(f"orthogonalize {k} x {n} {kind} {dtype}", flush=True)
    G = torch.from_numpy(np.stack([_matrix(k, n, kind, s) for s in range(2)])).to(dtype).cuda()
    out = rd.orthogonalize(G)
    assert out.dtype == dtype and out.shape == G.shape
    for e in range(2):
        rel = _check(out[e], G[e], [COEFFICIENTS] * 5)
        assert dtype == torch.float32 or rel <= (2e-3 if min(k, n) >= 63 else 8e-3) + HALF_ULP[dtype]  # what the header promises, and the last rounding


@types
def test_singular_values_near_one(dtype):
    G = torch.from_numpy(_matrix(96, 400, "gaussian")).to(dtype).cuda()
    s = np.linalg.svd(_np(rd.orthogonalize(G)), compute_uv=False)
    assert s.min() > 0.65 and s.max() < 1.25 and rd.orthogonalize(G).shape == (96, 400)


@types
@pytest.mark.parametrize("steps", [0, 1, 2, 8])
def test_steps_and_coefficients(steps, dtype):
    G = torch.from_numpy(_matrix(130, 90, "gaussian")).to(dtype).cuda()
    for triples in ([COEFFICIENTS] * steps, [(1.5, -0.5, 0.0)] * steps, [(1.875, -1.25, 0.375), (3.0, -4.0, 1.75)] * (steps // 2) + [(2.0, 0.0, 0.0)] * (steps % 2),
                    [(0.01, 0.0, 0.0)] * steps):
        _check(rd.orthogonalize(G, steps=steps, coefficients=triples, scale=-0.2) if steps else rd.orthogonalize(G, steps=0, scale=-0.2), G, triples, -0.2)


def test_sizes_of_the_numbers():
    """Norms that squares in 32 bits would lose, and ones that eps swallows."""
    for size in (1e-30, 1e-12, 1.0, 1e15, 1e30):
        G = torch.from_numpy(_matrix(70, 80, "gaussian") * size).float().cuda()
        _check(rd.orthogonalize(G), G, [COEFFICIENTS] * 5)
    zeros = torch.zeros(2, 40, 30, device="cuda")
    assert torch.equal(rd.orthogonalize(zeros), zeros)


def test_infinities_and_nan_stay_in_their_matrix():
    G = torch.randn(4, 70, 200, device="cuda")
    want = rd.orthogonalize(G)
    G[1, 3, 5], G[2, 69, 199] = torch.nan, torch.inf
    got = rd.orthogonalize(G)
    assert torch.equal(got[[0, 3]], want[[0, 3]]) and got[1:3].isnan().all() and rd.orthogonalize(G, steps=0)[1:3].isnan().all()


def test_matrices_do_not_depend_on_their_neighbours():
    for shape in ((300, 40, 96), (5, 300, 700)):
        G = torch.randn(shape, device="cuda").bfloat16()
        whole = rd.orthogonalize(G)
        for e in (0, shape[0] // 2, shape[0] - 1):
            assert torch.equal(rd.orthogonalize(G[e]), whole[e])


def test_strides_and_addresses():
    base = torch.randn(3, 200, 141, device="cuda")
    want = rd.orthogonalize(base[:, ::2, 1:].contiguous())
    assert torch.equal(rd.orthogonalize(base[:, ::2, 1:]), want)
    flat = torch.randn(100 * 77 + 1, device="cuda").half()
    assert torch.equal(rd.orthogonalize(flat[1:].view(100, 77)), rd.orthogonalize(flat[1:].clone().view(100, 77)))
    assert torch.equal(rd.orthogonalize(base.transpose(1, 2)), rd.orthogonalize(base.transpose(1, 2).contiguous()))
    for shape in ((0, 5, 6), (2, 0, 6), (2, 5, 0)):
        assert rd.orthogonalize(torch.empty(shape, device="cuda")).shape == shape


def test_refusals():
    G = torch.randn(20, 30, device="cuda")
    with pytest.raises(ValueError):
        rd.orthogonalize(G[0])
    with pytest.raises(TypeError):
        rd.orthogonalize(G.double())
    with pytest.raises(RuntimeError):
        rd.orthogonalize(G.cpu())
    with pytest.raises(ValueError):
        rd.orthogonalize(G, coefficients=(1.0, 2.0))
    with pytest.raises(ValueError):
        rd.orthogonalize(G, steps=3, coefficients=[COEFFICIENTS] * 2)
    with pytest.raises(RuntimeError, match="converge"):
        rd.orthogonalize(G, coefficients=(30.0, 0.0, 0.0))
    with pytest.raises(RuntimeError, match="finite"):
        rd.orthogonalize(G, coefficients=(float("nan"), 0.0, 0.0))
    with pytest.raises(RuntimeError, match="eps"):
        rd.orthogonalize(G, eps=-1.0)
    with pytest.raises(RuntimeError, match="steps"):
        rd.orthogonalize(G, steps=33)
    with pytest.raises(NotImplementedError):
        rd.orthogonalize(G.clone().requires_grad_())
    with torch.no_grad():
        rd.orthogonalize(G.clone().requires_grad_())


@pytest.mark.parametrize("g,k,n", [(1, 32, 4000), (30, 40, 100), (2, 2048, 128), (1, 100, 8000), (1, 1024, 1500), (64, 512, 1280)])
def test_float32_is_as_accurate_as_float32_products(g, k, n):
    """Long contractions of few rows, one of more than a piece of the sums, and tiles of each size; float32 products of the vendor's
    library in the formulas, whose roundings are others of the same size: three times what they are off by."""
    print(f"accuracy {g} x {k} x {n}", flush=True)
    G = torch.randn(g, k, n, generator=torch.Generator().manual_seed(k)).cuda()

    def iterate(X):
        X = X if k <= n else X.transpose(1, 2).contiguous()
        X = X / (X.flatten(1).norm(dim=1)[:, None, None] + 1e-7)
        for a, b, c in [COEFFICIENTS] * 5:
            A = torch.bmm(X, X.transpose(1, 2).contiguous())
            X = a * X + torch.bmm(b * A + c * torch.bmm(A, A), X)
        return X if k <= n else X.transpose(1, 2)

    ref = iterate(G.double())
    off, plain = (float((y.double() - ref).norm() / ref.norm()) for y in (rd.orthogonalize(G), iterate(G)))
    assert off <= 3 * plain, f"off by {off:.2e}, float32 products by {plain:.2e}"


def test_captured_and_replayed():
    G = torch.randn(3, 200, 150, device="cuda").bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rd.orthogonalize(G)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rd.orthogonalize(G)
    for _ in range(3):
        G.copy_(torch.randn(3, 200, 150, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, rd.orthogonalize(G))
