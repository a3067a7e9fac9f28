"""The gated activation and its gradient against float64."""

import numpy as np
import pytest
import torch

from gpu_ragged_dot_amd import moe
from oracle import expert_ops_oracle as oracle

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LEAST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check(y, dout):
    leaf = y.detach().requires_grad_()
    out = moe.swiglu(leaf)
    dy = torch.autograd.grad(out, leaf, dout)[0]
    assert out.dtype == y.dtype and dy.dtype == y.dtype and dy.shape == y.shape
    yn, dn = y.double().cpu().numpy(), dout.double().cpu().numpy()
    f = y.shape[1] // 2
    g, u = yn[:, :f], yn[:, f:]
    sig = 1 / (1 + np.exp(-g))
    # an exponential of |g|: 2^-24 |g| for each rounding of its argument, 2 units of its own; a quotient and products behind it
    unit = (8 + 2 * np.abs(g)) * 2.0 ** -23
    # a sigmoid below 2^-126 is subnormal in 32 bits and may count as 0: that much of what it is multiplied with
    flush = 2.0 ** -126
    ref = oracle.swiglu(yn)
    assert np.all(np.abs(out.detach().double().cpu().numpy() - ref) <= (unit + HALF_ULP[y.dtype]) * np.abs(ref) + flush * np.abs(g * u) + LEAST[y.dtype])
    ref = oracle.swiglu_grad(yn, dn)
    magnitude = np.concatenate([np.abs(dn * u) * sig * (1 + np.abs(g) * (1 - sig)), np.abs(dn * g) * sig], 1)
    magnitude += flush / (2 * np.concatenate([unit, unit], 1)) * np.concatenate([np.abs(dn * u) * (1 + np.abs(g)), np.abs(dn * g)], 1)
    unit = np.concatenate([unit, unit], 1)
    assert np.all(np.abs(dy.double().cpu().numpy() - ref) <= 2 * unit * magnitude + HALF_ULP[y.dtype] * np.abs(ref) + LEAST[y.dtype])


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,f", [(1, 1), (1, 8), (3, 7), (64, 768), (5, 1515), (33, 24), (257, 1000), (2, 4096), (1000, 12), (1, 20001)])
def test_against_float64(rows, f, dtype):
    print(f"swiglu {rows} x {f} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(rows * f)
    y = 2 * torch.randn((rows, 2 * f), generator=gen)
    _check(y.to(dtype).cuda(), torch.randn((rows, f), generator=gen).to(dtype).cuda())


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f16", "f32"])
def test_large_gates(dtype):
    """Where exponentials overflow and a sigmoid is one less a difference."""
    g = torch.tensor([-1000.0, -104.0, -89.0, -88.0, -30.0, -17.0, -1.2785, -1e-3, 0.0, 1e-6, 1.0, 17.0, 30.0, 88.0, 89.0, 1000.0])
    y = torch.cat([g, torch.full((16,), 3.0)])[None].to(dtype).cuda()
    _check(y, torch.full((1, 16), 2.0, dtype=dtype, device="cuda"))


def test_infinity_and_nan_stay_in_their_cells():
    y = torch.randn(4, 64, device="cuda")
    want = moe.swiglu(y)
    y[1, 3], y[2, 32 + 5] = torch.nan, torch.inf
    got = moe.swiglu(y)
    assert got[1, 3].isnan() and not got[2, 5].isfinite()
    got[1, 3], got[2, 5] = want[1, 3], want[2, 5]
    assert torch.equal(got, want)


def test_strides_addresses_and_empty_rows():
    y = torch.randn(9, 2 * 40, device="cuda").bfloat16()
    want = moe.swiglu(y)
    wide = torch.randn(9, 4 * 40, device="cuda").bfloat16()
    wide[:, ::2] = y
    assert torch.equal(moe.swiglu(wide[:, ::2]), want)
    odd = torch.empty(9 * 80 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(9, 80).copy_(y)  # at an odd address
    assert torch.equal(moe.swiglu(odd), want)
    odd.requires_grad_()
    dout = torch.randn(9, 40, device="cuda").bfloat16()
    leaf = y.clone().requires_grad_()
    a = torch.autograd.grad(moe.swiglu(odd), odd, dout)[0]
    b = torch.autograd.grad(moe.swiglu(leaf), leaf, dout)[0]
    assert torch.equal(a, b)
    c = torch.autograd.grad(moe.swiglu(leaf), leaf, torch.ones(1, 1, device="cuda").bfloat16().expand(9, 40))[0]  # a broadcast cotangent
    assert torch.equal(c, torch.autograd.grad(moe.swiglu(leaf), leaf, torch.ones(9, 40, device="cuda").bfloat16())[0])
    for shape in ((0, 8), (3, 0)):
        empty = torch.empty(shape, device="cuda", requires_grad=True)
        out = moe.swiglu(empty)
        assert out.shape == (shape[0], shape[1] // 2)
        assert torch.autograd.grad(out.sum(), empty)[0].shape == shape


def test_more_cells_than_32_bits_index():
    """2^31 input elements and some: the last rows, and some in the middle, as a call on them alone."""
    rows, f = 262145, 4096
    y = torch.empty((rows, 2 * f), dtype=torch.bfloat16, device="cuda")
    part = torch.randn((1024, 2 * f), device="cuda").bfloat16()
    for at in range(0, rows, 1024):
        y[at:at + 1024] = part[:min(1024, rows - at)] * (1 + at / rows)
    out = moe.swiglu(y)
    for at in (0, 131071, rows - 3):
        assert torch.equal(out[at:at + 3], moe.swiglu(y[at:at + 3].clone()))
    leaf = y.requires_grad_()
    dy = torch.autograd.grad(moe.swiglu(leaf), leaf, out)[0]
    for at in (0, 131071, rows - 3):
        few = y[at:at + 3].detach().clone().requires_grad_()
        assert torch.equal(dy[at:at + 3], torch.autograd.grad(moe.swiglu(few), few, out[at:at + 3])[0])


def test_replayed_and_on_another_stream():
    y = torch.randn(50, 512, device="cuda").bfloat16().requires_grad_()
    dout = torch.randn(50, 256, device="cuda").bfloat16()

    def step():
        out = moe.swiglu(y)
        return out.detach(), torch.autograd.grad(out, y, dout)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(on_side, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        with torch.no_grad():
            y.copy_(torch.randn(50, 512, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)
