"""Orthogonalised updates of any size of numbers, rank and coefficients, against 64 bits and relative to the result."""

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
wide_types = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])  # with eight bits of exponent


def _np(t):
    return t.double().cpu().numpy()


def _randn(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def _relative(got, ref):
    return np.linalg.norm(_np(got) - ref) / np.linalg.norm(ref)


# One rounding of X to what it is held in, relative: 22 bits for float32; 15 for bfloat16, 11 before the last step.  Where the
# iteration is linear, all directions grow alike and the roundings of up to eight steps add up as they are.
LINEAR = {torch.float32: 8 * 2.0 ** -22, torch.bfloat16: 8 * 2.0 ** -15 + 2.0 ** -11}


@types
@pytest.mark.parametrize("steps", [0, 1, 5])
def test_zeros_stay_zeros_without_eps(steps, dtype):
    """Such as the gradient of an expert that saw no token, among others."""
    G = _randn(3, 70, 200).to(dtype).cuda()
    G[1] = 0
    out = rd.orthogonalize(G, steps=steps, eps=0.0)
    assert not out[1].any()
    for e in (0, 2):
        assert torch.equal(out[e], rd.orthogonalize(G[e], steps=steps, eps=0.0)) and out[e].isfinite().all()


@wide_types
@pytest.mark.parametrize("power", [-120, -100, 100])
def test_without_eps_a_power_of_two_changes_nothing(power, dtype):
    for shape in ((70, 200), (200, 70)):
        G = _randn(*shape, seed=1).to(dtype).cuda()
        G[G.abs() < 2.0 ** -5] = 0  # (what stays a normal number)
        for steps in (0, 1, 5):
            assert torch.equal(rd.orthogonalize(G * 2.0 ** power, steps=steps, eps=0.0), rd.orthogonalize(G, steps=steps, eps=0.0))


@wide_types
@pytest.mark.parametrize("size", [1e-11, 1e-13, 1e-15, 1e-18, 1e-25])
def test_norms_far_below_eps(size, dtype):
    """X starts at |G| / eps and every step multiplies it by a."""
    G = _randn(70, 80, seed=2)
    G = (G * (size / G.norm())).to(dtype).cuda()
    ref = oracle.orthogonalize(_np(G), [COEFFICIENTS] * 5)
    assert _relative(rd.orthogonalize(G), ref) <= LINEAR[dtype] + HALF_ULP[dtype]


@wide_types
@pytest.mark.parametrize("a,steps", [(0.01, 8), (2.0 ** -9, 5), (0.25, 8)])
def test_coefficients_that_shrink(a, steps, dtype):
    G = _randn(130, 90, seed=3).to(dtype).cuda()
    for triple in ((a, 0.0, 0.0), (a, -0.1 * a, 0.0)):
        ref = oracle.orthogonalize(_np(G), [triple] * steps)
        assert _relative(rd.orthogonalize(G, steps=steps, coefficients=triple), ref) <= LINEAR[dtype] + HALF_ULP[dtype]


def test_norms_of_every_size_in_one_stack():
    G = _randn(6, 100, 140, seed=4)
    G *= torch.tensor([1.0, 1e-9, 1e-20, 0.0, 1e12, 1e-6])[:, None, None]
    for dtype in (torch.float32, torch.bfloat16):
        H = G.to(dtype).cuda()
        out = rd.orthogonalize(H)
        for e in range(len(G)):
            assert torch.equal(rd.orthogonalize(H[e]), out[e])


@types
def test_a_nearly_cubic_step(dtype):
    """c so small that the largest value lies where the cubic's does, at 3^-1/2, where all singular values are; what the next step's numbers
    are multiplied with follows from it."""
    G = torch.eye(3, 5)[None].repeat(2, 1, 1).to(dtype).cuda()
    for c in (1e-20, -1e-20, 1e-300, 0.0):
        out = rd.orthogonalize(G, steps=2, coefficients=[(3.0, -3.0, c), (1.0, 0.0, 0.0)], eps=0.0)
        # 2 / 3^1/2 on the diagonal.  Two steps: roundings of X, A and B, each of 22 or 11 bits, times 3 at most
        assert ((out.double() - G.double() * 2 / 3 ** 0.5).abs() <= (2.0 ** -18 if dtype == torch.float32 else 2.0 ** -7) + 2 * HALF_ULP[dtype]).all()


def test_scales_of_any_size():
    for shape, steps in (((60, 100), 5), ((100, 60), 5), ((60, 100), 1), ((60, 100), 0)):
        G = _randn(*shape, seed=6).cuda()
        base = rd.orthogonalize(G, steps=steps)
        base[base.abs() < 2.0 ** -8] = 0
        for power in (-116, -60, 60, 116):
            got = rd.orthogonalize(G, steps=steps, scale=2.0 ** power)
            got[base == 0] = 0
            assert torch.equal(got, base * 2.0 ** power)
    with pytest.raises(RuntimeError, match="scale"):
        rd.orthogonalize(G, scale=1e39)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("k,n,rank", [(256, 512, 4), (512, 256, 1), (64, 64, 2)])
@pytest.mark.parametrize("steps", [8, 10])
def test_many_steps_on_low_rank(steps, k, n, rank, dtype):
    """The gradient of an expert that saw few tokens, exact in 16 bits.  What a step rounds in directions that it leaves empty is multiplied by
    a = 3.4445 in every later one.  Numbers of 22 bits: X is off by 2^-22 of its norm at the start, and by less than three times that in all
    steps together, weighted with what is left to grow; the norm is at least 0.7: 2^-20 a^steps of the result.  (Numbers of 11 and 15 bits
    leave 0.04 to 0.09 of noise at eight steps, 0.4 to 1 at ten.)"""
    rng = np.random.default_rng(rank)
    G = rng.integers(-2, 3, (k, rank)) @ rng.integers(-2, 3, (rank, n)) if rank > 1 else np.outer(rng.integers(1, 8, k), rng.integers(-7, 8, n))
    t = torch.from_numpy(G).to(dtype).cuda()
    assert np.array_equal(_np(t), G)
    ref = oracle.orthogonalize(G, [COEFFICIENTS] * steps)
    assert _relative(rd.orthogonalize(t, steps=steps), ref) <= 2.0 ** -20 * COEFFICIENTS[0] ** steps + HALF_ULP[dtype]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("steps,most", [(5, 8e-3), (6, 1e-2)])
def test_few_steps_on_low_rank(steps, most, dtype):
    """What the header promises for matrices of few rows, columns or directions."""
    for k, n, rank in ((256, 512, 1), (64, 64, 1), (512, 100, 2), (256, 512, 4)):
        rng = np.random.default_rng(rank)
        G = rng.integers(-2, 3, (k, rank)) @ rng.integers(-2, 3, (rank, n)) if rank > 1 else np.outer(rng.integers(1, 8, k), rng.integers(-7, 8, n))
        t = torch.from_numpy(G).to(dtype).cuda()
        assert _relative(rd.orthogonalize(t, steps=steps), oracle.orthogonalize(G, [COEFFICIENTS] * steps)) <= most + HALF_ULP[dtype]


def test_a_workspace_of_one_spec_does():
    """Stacks of 16-bit matrices, few steps and many, in the bytes that the C entry asks for and no more."""
    import ctypes

    from gpu_ragged_dot_amd import _capi

    G = _randn(3, 200, 150, seed=8).bfloat16().cuda()
    for steps in (5, 8):
        flat = (ctypes.c_double * (3 * steps))(*(COEFFICIENTS * steps))
        spec = _capi.OrthoSpec(steps, flat, 1e-7, 1.0)
        need = _capi.lib.rd_orthogonalize_spec_workspace_bytes(3, 200, 150, ctypes.byref(spec), _capi.RD_DTYPE_BF16)
        whole = torch.full((need + 512,), 77, dtype=torch.uint8, device="cuda")
        out = torch.empty_like(G)
        at = -whole.data_ptr() % 256
        status = _capi.lib.rd_orthogonalize(torch.cuda.current_stream().cuda_stream, G.data_ptr(), out.data_ptr(), 3, 200, 150, ctypes.byref(spec),
                                            _capi.RD_DTYPE_BF16, whole.data_ptr() + at, need)
        assert status == 0 and torch.equal(out, rd.orthogonalize(G, steps=steps))
        assert (whole[:at] == 77).all() and (whole[at + need:] == 77).all()


@pytest.mark.parametrize("k,n", [(8, 300), (64, 64), (256, 512), (515, 100), (1024, 768)])
@pytest.mark.parametrize("rank", [None, 5])
def test_float16_results_are_off_by_their_own_rounding(rank, k, n):
    """Eleven bits of a result are not to be had from products of eleven: 2^-20 of the result for each time that the coefficients multiply
    roundings, which numbers of 22 bits leave at most, and half a step of float16."""
    G = _randn(k, n, seed=9) if rank is None else _randn(k, rank, seed=9) @ _randn(rank, n, seed=10)
    G = G.half().cuda()
    ref = oracle.orthogonalize(_np(G), [COEFFICIENTS] * 5)
    got = rd.orthogonalize(G)
    assert _relative(got, ref) <= 2.0 ** -20 * COEFFICIENTS[0] ** 5 + HALF_ULP[torch.float16]
