"""Traced products on 4-bit weights on rows that ask for a gradient: they run where none is taken, as calls that are not traced do
under ``torch.no_grad()``, and refuse it in the backward pass."""

import pytest
import torch

import gpu_ragged_dot_amd as rd
from gpu_ragged_dot_amd import int4


class _StandIn:
    """A product of torch operations that, as the native one, refuses rows whose gradient is wanted."""

    @staticmethod
    def gmm_int4(x, *_):
        if torch.is_grad_enabled() and x.requires_grad:
            raise NotImplementedError("no gradient")
        return 2 * x.detach()


def _check(weights, device):
    gs = torch.tensor([1, 3], dtype=torch.int32, device=device)
    rows = lambda: torch.randn(4, 64).bfloat16().to(device)
    step = lambda x: rd.ragged_dot_int4(x, weights, gs)
    traced = torch.jit.trace(step, (rows(),), check_trace=False)
    x = rows().requires_grad_()
    with pytest.raises(NotImplementedError, match="no gradient"):
        step(x)
    with torch.no_grad():
        want = step(x)
        assert torch.equal(traced(x), want)
    assert torch.equal(traced(x.detach()), want) and not traced(x.detach()).requires_grad
    y = traced(x)
    assert torch.equal(y, want)
    with pytest.raises(NotImplementedError, match="no gradient"):
        y.sum().backward()


def test_with_a_stand_in_for_the_kernel(monkeypatch):
    monkeypatch.setattr(int4, "_native", _StandIn)
    _check(rd.Int4Weights(None, None, None, 64, 64, 32), "cpu")


@pytest.mark.gpu
def test_on_the_device():
    q = torch.randint(0, 16, (2, 64, 48), dtype=torch.uint8, device="cuda")
    _check(rd.pack_int4(q, torch.ones((2, 2, 48), device="cuda").bfloat16(), block=32), "cuda")
