"""Weights that are renormalised over one expert are `scale` whatever its logit: their gradient is 0, not a rounding of the terms that
cancel in it."""

import pytest
import torch

from gpu_ragged_dot_amd import moe

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("scale", [1.0, 2.5, 0.3, -0.7])
@pytest.mark.parametrize("experts,top_k", [(20, 1), (600, 1), (64, 6), (64, 20)])
def test_no_gradient(experts, top_k, scale, score, dtype):
    gen = torch.Generator(device="cuda").manual_seed(experts)
    logits = torch.randn((301, experts), generator=gen, device="cuda").to(dtype)
    if top_k > 1:  # one expert that is not shut
        at = torch.randint(experts, (301, 1), generator=gen, device="cuda")
        logits = torch.full_like(logits, -torch.inf).scatter(1, at, logits.gather(1, at))
    logits.requires_grad_()
    got = moe.gate(logits, top_k, score=score, scale=scale)
    assert torch.equal(got.weights[:, 0], torch.full((301,), scale, device="cuda"))
    dw = torch.randn(got.weights.shape, generator=gen, device="cuda")
    assert not torch.autograd.grad(got.weights, logits, dw)[0].any()
