"""Traced calls of the gate whose bias asks for a gradient, as a balance bias held as a parameter does: it gets none, as in a call that is
not traced, and does not stand in the way of the logits'."""

import pytest
import torch

from gpu_ragged_dot_amd import moe


class _StandIn:
    """A gate of torch operations that, as the native one, takes its bias's value alone."""

    @staticmethod
    def moe_gate(logits, bias, top_k, *spec):
        ranks = logits.detach() if bias is None else logits.detach() + bias.detach()
        ids = ranks.topk(top_k, dim=1).indices
        return ids.int(), torch.softmax(logits.gather(1, ids), 1)


def _check(device):
    rand = lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(sum(s))).to(device)
    logits, bias = rand(6, 10).requires_grad_(), (0.01 * rand(10)).requires_grad_()

    def step(logits, bias):
        ids, weights = moe.gate(logits, 3, bias=bias)
        return ids, weights

    dw = rand(6, 3)
    want_ids, want = step(logits, bias)
    want_grad = torch.autograd.grad(want, logits, dw)[0]
    example = (rand(6, 10).requires_grad_(), rand(10).requires_grad_())
    traced = torch.jit.trace(step, example, check_trace=False)
    ids, weights = traced(logits, bias)
    assert torch.equal(ids, want_ids) and torch.equal(weights, want)
    weights.backward(dw)
    assert torch.equal(logits.grad, want_grad) and bias.grad is None
    # the bias alone asks for one: nothing to take a gradient of
    ids, weights = traced(logits.detach(), bias)
    assert torch.equal(ids, want_ids) and torch.equal(weights, want) and not weights.requires_grad
    # a sum with something else that has a gradient
    other = rand(6, 3).requires_grad_()
    (traced(logits.detach(), bias)[1] * other).sum().backward()
    assert torch.equal(other.grad, want.detach()) and bias.grad is None


def test_with_a_stand_in_for_the_kernel(monkeypatch):
    monkeypatch.setattr(moe, "_native", _StandIn)
    _check("cpu")


@pytest.mark.gpu
def test_on_the_device():
    _check("cuda")
