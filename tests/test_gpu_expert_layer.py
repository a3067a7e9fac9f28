"""A mixture-of-experts layer from the router's logits to the summed rows, as a program runs it: gate, route, dispatch, product,
gated activation, product, combine.  Serving on 4-bit weights, training on bfloat16 ones with every gradient; padded tokens."""

import numpy as np
import pytest
import torch

import gpu_ragged_dot_amd as rd
from gpu_ragged_dot_amd import moe
from oracle import expert_ops_oracle as oracle

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8  # of bfloat16
GATE = dict(score="sigmoid", clusters=4, top_clusters=2, cluster_score="top2", scale=2.5)


def _inputs(tokens, experts, d, f, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")
    logits = 1.5 * rand(tokens, experts)
    logits[tokens // 2] = -torch.inf  # a padded token
    bias = 0.001 * (20 * rand(experts)).round()
    return rand(tokens, d).bfloat16(), logits, bias, rand(experts, d, 2 * f) * d ** -0.5, rand(experts, f, d) * f ** -0.5


def _serve(h, logits, bias, w_in, w_out, experts, top_k, product):
    ids, weights = moe.gate(logits, top_k, bias=bias, **GATE)
    r = moe.route(ids, experts)
    hidden = moe.swiglu(product(moe.dispatch(h, r), w_in, r.group_sizes))
    return moe.combine(product(hidden, w_out, r.group_sizes), r, weights)


def _exact(h, logits, bias, w_in, w_out, top_k):
    """The layer's sums in 64 bits, on experts that the gate's restatement chooses."""
    ids, _ = oracle.gate(logits.detach().double().cpu().numpy(), top_k, bias=bias.double().cpu().numpy(), **GATE)
    ids = torch.from_numpy(ids).long().cuda()
    s = torch.sigmoid(logits.double()).gather(1, ids.clamp(min=0)) * (ids >= 0)
    weights = 2.5 * s / s.sum(1, keepdim=True).clamp(min=1e-300)
    out = []
    for t in range(h.shape[0]):
        row = torch.zeros(h.shape[1], dtype=torch.float64, device="cuda")
        for j, e in enumerate(ids[t].tolist()):
            if e >= 0:
                gate_half, up = (h[t].double() @ w_in[e].double()).chunk(2)
                row = row + weights[t, j] * ((gate_half / (1 + torch.exp(-gate_half)) * up) @ w_out[e].double())
        out.append(row)
    return torch.stack(out)


def _quantised(a, block):
    """[g, k, n] float -> (packed weights, what they stand for)."""
    g, k, n = a.shape
    blocks = -(-k // block)
    padded = torch.nn.functional.pad(a, (0, 0, 0, blocks * block - k)).view(g, blocks, block, n)
    scales = (padded.abs().amax(2) / 7).bfloat16()
    q = (padded / scales.float()[:, :, None]).round().add(8).clamp(0, 15).to(torch.uint8).view(g, blocks * block, n)[:, :k].contiguous()
    dense = (q.double() - 8) * scales.double().repeat_interleave(block, 1)[:, :k]
    return rd.pack_int4(q, scales, block=block), dense


@pytest.mark.parametrize("tokens", [1, 8, 200])
def test_serving_on_4_bit_weights(tokens):
    experts, top_k, d, f = 16, 4, 256, 200
    h, logits, bias, w_in, w_out = _inputs(tokens + 1, experts, d, f, tokens)
    (q_in, a_in), (q_out, a_out) = _quantised(w_in, 64), _quantised(w_out, 128)
    with torch.no_grad():
        out = _serve(h, logits, bias, q_in, q_out, experts, top_k, rd.ragged_dot_int4)
    ref = _exact(h, logits, bias, a_in, a_out, top_k)
    assert not out[(tokens + 1) // 2].any()
    # relative errors of a rounding each: weights and result of the first product, twice in a product of its halves; the activation;
    # weights and result of the second product; the sum
    assert (out.double() - ref).norm() <= 8 * HALF * ref.norm()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        held = _serve(h, logits, bias, q_in, q_out, experts, top_k, rd.ragged_dot_int4)
    for seed in (1, 2, 3):
        h2, logits2 = _inputs(tokens + 1, experts, d, f, 100 + seed)[:2]
        h.copy_(h2), logits.copy_(logits2)
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(held, _serve(h, logits, bias, q_in, q_out, experts, top_k, rd.ragged_dot_int4))


def test_training_with_every_gradient():
    tokens, experts, top_k, d, f = 48, 16, 4, 128, 96
    h, logits, bias, w_in, w_out = _inputs(tokens, experts, d, f, 5)
    leaves = [h, logits, w_in.bfloat16(), w_out.bfloat16()]
    dout = torch.randn(tokens, d, device="cuda").bfloat16()
    for t in leaves:
        t.requires_grad_()
    out = _serve(leaves[0], leaves[1], bias, leaves[2], leaves[3], experts, top_k, rd.ragged_dot)
    got = torch.autograd.grad(out, leaves, dout)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    ref = _exact(wide[0], wide[1], bias, wide[2], wide[3], top_k)
    want = torch.autograd.grad(ref, wide, dout.double())
    # the roundings on the way of the forward pass (5: no weights are rounded), as many on the way back
    assert (out.detach().double() - ref.detach()).norm() <= 5 * HALF * ref.detach().norm()
    for a, b in zip(got, want):
        live = b.isfinite()  # (the derivative of exp(-inf) by the reference's own rules)
        assert not a[~live].any() and (a.double() - b)[live].norm() <= 10 * HALF * b[live].norm()


def test_traced_calls_run_their_kernels():
    gs = torch.tensor([5, 0, 11], dtype=torch.int32, device="cuda")
    w, _ = _quantised(torch.randn(3, 64, 32, device="cuda"), 32)

    def step(logits, y, x):
        ids, weights = moe.gate(logits, 2, score="sigmoid")
        return ids, weights, moe.swiglu(y), rd.ragged_dot_int4(x, w, gs)

    inputs = lambda: (torch.randn(6, 10, device="cuda", requires_grad=True), torch.randn(6, 10, device="cuda", requires_grad=True),
                      torch.randn(16, 64, device="cuda").bfloat16())
    traced = torch.jit.trace(step, inputs(), check_trace=False)
    args = inputs()
    for a, b in zip(traced(*args), step(*args)):
        assert torch.equal(a, b)
    for i, leaf in ((1, 0), (2, 1)):
        a, b = (torch.autograd.grad(fn(*args)[i].sum(), args[leaf])[0] for fn in (traced, step))
        assert torch.equal(a, b)


def test_two_streams_at_once():
    """Calls that run side by side on one device share nothing."""
    w, _ = _quantised(torch.randn(8, 512, 256, device="cuda") * 0.05, 128)
    gs = torch.full((8,), 40, dtype=torch.int32, device="cuda")
    xs = [torch.randn(320, 512, device="cuda").bfloat16() for _ in range(4)]
    logits = [torch.randn(300, 128, device="cuda") for _ in range(4)]
    bias = torch.zeros(128, device="cuda")
    one = lambda i: (rd.ragged_dot_int4(xs[i], w, gs), *moe.gate(logits[i], 8, bias=bias), moe.swiglu(xs[i]))
    want = [one(i) for i in range(4)]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got.append([one(i) for _ in range(5)])
    torch.cuda.synchronize()
    for i in range(4):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))
