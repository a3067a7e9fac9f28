"""Gradients of the product on float8 where the output's type is not the rows', against 64 bits."""

import numpy as np
import pytest
import torch

import gpu_ragged_dot_amd as rd

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LEAST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
PAIRS = [(a, b) for a in HALF_ULP for b in HALF_ULP if a != b]
pairs = pytest.mark.parametrize("dtype,out_dtype", PAIRS, ids=lambda t: str(t).split(".")[1])


def _np(t):
    return t.detach().double().cpu().numpy()


@pairs
@pytest.mark.parametrize("trans", [False, True], ids=["nn", "nt"])
def test_weights_gradient_takes_the_cotangent_as_it_is(trans, dtype, out_dtype):
    """float32 sums of the rows' and the cotangent's own products, one rounding to the weights' type: no cotangent becomes infinite, 0 or
    shorter on its way to a narrower type."""
    sizes, k, n = [90, 0, 150, 50], 136, 200
    gen = torch.Generator().manual_seed(k + n)
    x = (torch.randn(300, k, generator=gen) * 2.0 ** -8).to(dtype).cuda().requires_grad_()
    A = torch.randn((4, n, k) if trans else (4, k, n), generator=gen).to(dtype).cuda().requires_grad_()
    dy = torch.randn(300, n, generator=gen)
    dy[:, :40] *= 2e5 if out_dtype != torch.float16 else 1e4   # beyond float16
    dy[:, 40:80] *= 1e-4
    dy = dy.to(out_dtype).cuda()
    print(f"types {dtype} {out_dtype} trans={trans}", flush=True)
    y = rd.ragged_dot_float8(x, A, torch.tensor(sizes, dtype=torch.int32, device="cuda"), trans_rhs=trans, out_dtype=out_dtype)
    assert y.dtype == out_dtype
    dx, dA = torch.autograd.grad(y, (x, A), dy)
    assert dx.dtype == dtype and dA.dtype == dtype
    row = 0
    for e, size in enumerate(sizes):
        xs, ds = _np(x)[row:row + size], _np(dy)[row:row + size]
        ref, mag = ((f(ds).T @ f(xs) if trans else f(xs).T @ f(ds)) for f in (lambda t: t, np.abs))
        bound = (size + 8) * 2.0 ** -23 * mag + HALF_ULP[dtype] * np.abs(ref) * (1 + 2.0 ** -10) + LEAST[dtype]
        assert np.all(np.abs(_np(dA[e]) - ref) <= bound), (e, np.abs(_np(dA[e]) - ref).max())
        row += size


def test_small_cotangents_add_up():
    """10000 cotangents below what float16 holds, against ones: 2e-4, a float16 number."""
    m = 10000
    x, A = torch.ones(m, 128, device="cuda").half(), torch.ones(1, 128, 128, device="cuda").half().requires_grad_()
    y = rd.ragged_dot_float8(x, A, torch.tensor([m], dtype=torch.int32, device="cuda"), out_dtype=torch.float32)
    dA, = torch.autograd.grad(y, A, torch.full((m, 128), 2e-8, device="cuda"))
    # float32 sums of 10^4 equal numbers, in any order within 10^4 roundings of 2^-24; half a step of float16
    assert ((dA.double() - 2e-4).abs() <= 2e-4 * (m * 2.0 ** -24 + 2.0 ** -11)).all()
