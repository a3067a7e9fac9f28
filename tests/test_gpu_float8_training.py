"""The float8 operators and the orthogonalised update together, as programs run them: a layer served in 8 bits from the router's logits
on, and steps of training of an expert layer in 8 bits whose weights are moved by orthogonalised momenta."""

import numpy as np
import pytest
import torch

import gpu_ragged_dot_amd as rd
from gpu_ragged_dot_amd import moe
from gpu_ragged_dot_amd.ortho import COEFFICIENTS
from oracle import expert_ops_oracle, float8_oracle, moe_glue_oracle, ortho_oracle

pytestmark = pytest.mark.gpu


def _np(t):
    return t.detach().double().cpu().numpy()


def _swiglu(y):
    f = y.shape[1] // 2
    return y[:, :f] / (1 + np.exp(-y[:, :f])) * y[:, f:]


@pytest.mark.parametrize("tokens,experts,top_k,d,f", [(8, 16, 4, 256, 128), (100, 8, 2, 300, 200), (1, 4, 1, 128, 64)])
def test_a_layer_served_in_8_bits(tokens, experts, top_k, d, f):
    """Every stage against its statement in 64 bits on what the stage before it gave."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")
    h, logits = rand(tokens, d).bfloat16(), 1.5 * rand(tokens, experts)
    if tokens > 4:
        logits[tokens // 2] = -torch.inf  # a padded token
    w_in, w_out = (rand(experts, d, 2 * f) * d ** -0.5).bfloat16(), (rand(experts, d, f) * f ** -0.5).bfloat16()
    q_in, q_out = rd.quantize_weights(w_in), rd.quantize_weights(w_out)  # [g, k, n] and [g, n, k]

    ids, weights = moe.gate(logits, top_k)
    r = moe.route(ids, experts)
    x = moe.dispatch(h, r, float8=True)
    y = rd.ragged_dot_float8(x, q_in, r.group_sizes)
    hidden = moe.swiglu(y, float8=True)
    z = rd.ragged_dot_float8(hidden, q_out, r.group_sizes, trans_rhs=True)
    out = moe.combine(z, r, weights)

    sizes = r.group_sizes.cpu().numpy()
    x64 = float8_oracle.held(moe_glue_oracle.dispatch(_np(h), r.slot_of_row.cpu().numpy(), top_k))
    assert np.array_equal(_np(rd.dequantize(x, torch.float32)), x64.astype(np.float32))
    w64 = np.stack([float8_oracle.held(_np(a), 128) for a in w_in])
    y64 = float8_oracle.ragged_dot(x64, w64, sizes)
    assert np.abs(_np(y) - y64).max() <= 2.0 ** -7 * np.abs(y64).max()
    hidden64 = _np(rd.dequantize(hidden, torch.float32))
    exact = _swiglu(_np(y))
    scales = np.repeat(_np(hidden.scales)[:, :-(-f // 128)], 128, 1)[:, :f]
    assert np.all(np.abs(hidden64 - exact) <= np.maximum(2.0 ** -4 * np.abs(exact), 2.0 ** -10 * scales) * (1 + 2.0 ** -12))
    w64 = np.stack([float8_oracle.held(_np(a), 128) for a in w_out])
    z64 = float8_oracle.ragged_dot(hidden64, w64, sizes, trans_rhs=True)
    assert np.abs(_np(z) - z64).max() <= 2.0 ** -7 * np.abs(z64).max()
    out64 = moe_glue_oracle.combine(_np(z), r.row_of_slot.cpu().numpy(), top_k, _np(weights))
    assert np.all(np.abs(_np(out) - out64) <= 2.0 ** -8 * np.abs(out64) + 2.0 ** -20 * np.abs(_np(z)).max())
    if tokens > 4:
        assert not out[tokens // 2].any()


def _expert_loss(x, w_in, w_out, sizes, dout):
    y = rd.ragged_dot_float8(x, w_in, sizes)
    z = rd.ragged_dot_float8(moe.swiglu(y), w_out, sizes)
    return (z.float() * dout.float()).sum()


def test_steps_of_training():
    """Gradients of an expert layer in 8 bits near those of the same layer in 64 bits on quantised operands, its weights moved by
    orthogonalised momenta."""
    m, d, f, g = 300, 256, 192, 5
    gen = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")
    sizes = torch.tensor([100, 0, 37, 128, 35], dtype=torch.int32, device="cuda")
    params = [(rand(g, d, 2 * f) * d ** -0.5).bfloat16().requires_grad_(), (rand(g, f, d) * f ** -0.5).bfloat16().requires_grad_()]
    momenta = [torch.zeros(p.shape, device="cuda") for p in params]
    for step in range(3):
        x, dout = rand(m, d).bfloat16().requires_grad_(), rand(m, d).bfloat16()
        loss = _expert_loss(x, *params, sizes, dout)
        grads = torch.autograd.grad(loss, [x, *params])
        assert [t.shape for t in grads] == [t.shape for t in (x, *params)] and all(t.isfinite().all() for t in grads)

        # straight through, in 64 bits: quantised operands in the products, quantised cotangents in the rows' gradients
        row = 0
        for e, size in enumerate(sizes.tolist()):
            at = slice(row, row + size)
            row += size
            if not size:
                assert not grads[1][e].any() and not grads[2][e].any()
                continue
            xs, ds = _np(x)[at], _np(dout)[at]
            w1, w2 = (float8_oracle.held(_np(p[e]), 128) for p in params)
            y = float8_oracle.held(xs) @ w1
            hidden = _swiglu(y)
            dhidden = float8_oracle.held(ds) @ w2.T
            sig = 1 / (1 + np.exp(-y[:, :f]))
            dy = np.concatenate([dhidden * y[:, f:] * sig * (1 + y[:, :f] * (1 - sig)), dhidden * y[:, :f] * sig], 1)
            for got, ref in ((grads[2][e], hidden.T @ ds), (grads[1][e], xs.T @ dy), (grads[0][at], float8_oracle.held(dy) @ w1.T)):
                # bfloat16 between the stages: 2^-8 a rounding, three on the way, and codes that it moves by a step now and then
                assert np.linalg.norm(_np(got) - ref) <= 0.02 * np.linalg.norm(ref)

        with torch.no_grad():
            for p, mom, grad in zip(params, momenta, grads[1:]):
                mom.lerp_(grad.float(), 0.1)
                update = rd.orthogonalize(mom)
                for e in range(g):
                    exact = ortho_oracle.orthogonalize(_np(mom[e]), [COEFFICIENTS] * 5)
                    assert np.linalg.norm(_np(update[e]) - exact) <= 1e-4 * np.linalg.norm(exact) + 1e-12
                p -= (0.02 * update).to(p.dtype)


def test_a_gradient_keeps_only_what_it_reads():
    """Of weights held as float8 only dx is made, which needs no rows: they may be written over, and are not kept."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    leaf = torch.randn(50, 256, generator=gen, device="cuda").bfloat16().requires_grad_()
    w = rd.quantize_weights(torch.randn(2, 256, 128, generator=gen, device="cuda").bfloat16())
    gs, dy = torch.tensor([20, 25], dtype=torch.int32, device="cuda"), torch.randn(50, 128, generator=gen, device="cuda").bfloat16()
    x = leaf * 1
    y = rd.ragged_dot_float8(x, w, gs)
    want = rd.ragged_dot_float8(dy, w, gs, trans_rhs=True)
    x.detach().zero_()
    with torch.no_grad():
        x.zero_()
    got, = torch.autograd.grad(y, leaf, dy)
    assert torch.equal(got, want)
    kept = []
    A = torch.randn(2, 256, 128, generator=gen, device="cuda").bfloat16().requires_grad_()
    for rows, weights in ((leaf, A), (leaf, w), (leaf.detach(), A)):
        before = torch.cuda.memory_allocated()
        y = rd.ragged_dot_float8(rows, weights, gs)
        kept.append(torch.cuda.memory_allocated() - before)
        del y
    assert kept[0] > kept[1] and kept[0] > kept[2]


def test_two_calls_at_once_on_two_streams():
    """Nothing that a call writes is another's."""
    shapes = [(700, 512, 640), (90, 256, 1000)]
    work = []
    for m, k, n in shapes:
        x, A = torch.randn(m, k, device="cuda").bfloat16(), torch.randn(3, k, n, device="cuda").bfloat16()
        gs = torch.tensor([m // 2, 0, m // 3], dtype=torch.int32, device="cuda")
        work.append((x, A, gs, rd.ragged_dot_float8(x, A, gs), rd.orthogonalize(A)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, A, gs = work[i][:3]
                got[i].append((rd.ragged_dot_float8(x, A, gs), rd.orthogonalize(A)))
    torch.cuda.synchronize()
    for i in range(2):
        for y, o in got[i]:
            assert torch.equal(y, work[i][3]) and torch.equal(o, work[i][4])


def test_two_graphs_replayed_in_turn():
    """Graphs captured on their own: neither keeps an answer or a workspace of the other."""
    A = torch.randn(2, 300, 200, device="cuda").bfloat16()
    x = torch.randn(200, 300, device="cuda").bfloat16()
    gs = torch.tensor([120, 70], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rd.orthogonalize(A), rd.ragged_dot_float8(x, A, gs)
    torch.cuda.current_stream().wait_stream(side)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        o = rd.orthogonalize(A)
        y = rd.ragged_dot_float8(x, A, gs)
    with torch.cuda.graph(second):
        o2 = rd.orthogonalize(A.transpose(1, 2))
        held = moe.swiglu(x, float8=True)
    for _ in range(3):
        A.copy_(torch.randn(2, 300, 200, device="cuda"))
        x.copy_(torch.randn(200, 300, device="cuda"))
        first.replay()
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, rd.orthogonalize(A)) and torch.equal(y, rd.ragged_dot_float8(x, A, gs))
        assert torch.equal(o2, rd.orthogonalize(A.transpose(1, 2).contiguous()))
        want = moe.swiglu(x, float8=True)
        assert torch.equal(held.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(held.scales, want.scales)


def test_traced():
    """A trace calls the kernels again whenever it runs."""
    x, A = torch.randn(40, 256, device="cuda").bfloat16(), torch.randn(3, 256, 200, device="cuda").bfloat16()
    gs = torch.tensor([10, 0, 25], dtype=torch.int32, device="cuda")
    ids = torch.randint(0, 3, (20, 2), device="cuda", dtype=torch.int32)
    r = moe.route(ids, 3)
    w = rd.quantize_weights(A)

    def all_of(x, gs):
        held = moe.dispatch(x[:20], r, float8=True)
        y = rd.ragged_dot_float8(held, w, r.group_sizes)
        rows = rd.quantize_rows(x)
        return (rd.ragged_dot_float8(x, A, gs), rd.dequantize(rows, torch.float32), y, rd.dequantize(moe.swiglu(y, float8=True)),
                rd.orthogonalize(x), rd.dequantize(rd.quantize_weights(x[None])))

    traced = torch.jit.trace(all_of, (x, gs), check_trace=False)
    for seed in range(2):
        torch.manual_seed(seed)
        x2 = torch.randn(40, 256, device="cuda").bfloat16()
        gs2 = torch.tensor([[0, 30, 5], [5, 5, 5]][seed], dtype=torch.int32, device="cuda")
        for a, b in zip(traced(x2, gs2), all_of(x2, gs2)):
            assert torch.equal(a, b)
    leaf = x.clone().requires_grad_()
    step = torch.jit.trace(lambda x: rd.ragged_dot_float8(x, A, gs), (x,), check_trace=False)
    dout = torch.randn(40, 200, device="cuda").bfloat16()
    got, = torch.autograd.grad(step(leaf), leaf, dout)
    want, = torch.autograd.grad(rd.ragged_dot_float8(leaf, A, gs), leaf, dout)
    assert torch.equal(got, want)


@pytest.mark.parametrize("apart", [False, True], ids=["large products", "none"])
def test_gradient_by_differences(apart):
    """The output is linear in what x is held as: moved by whole steps of the codes, x moves it by what dx says.  All numbers are whole
    and every block's scale is 1.  Sums of eight products are cut 13 bits below the exponent of the largest: of products of at most 448 x 8
    (exponent 11) at a quarter, which whole products do not notice.  Where 448 meets 448 (exponent 17: at 16) seven may lose 16 each, in
    column 0 of y, whose cotangent is 448, before the move and behind it: 2 x 7 x 16 x 448.  Apart, 448 meets nothing but zeros."""
    x = torch.zeros(8, 128, device="cuda")
    x[:, 0] = 448.0
    x[:, 1:] = torch.randint(-8, 9, (8, 127), device="cuda").float()
    A = torch.randint(-8, 9, (2, 128, 128), device="cuda").float()
    A[:, 0, 0] = 448.0
    gs = torch.tensor([3, 5], dtype=torch.int32, device="cuda")
    dout = torch.randint(-8, 9, (8, 128), device="cuda").float()
    dout[:, 0] = 448.0
    if apart:
        A[:, 0] = 0
        A[:, :, 0] = 0
        A[:, 8, 8] = 448.0
        x[:, 8] = 0
        dout[:, 8] = 0
    leaf, A_leaf = x.clone().requires_grad_(), A.clone().requires_grad_()
    loss = lambda x, A: (rd.ragged_dot_float8(x, A, gs).double() * dout.double()).sum()
    dx, dA = torch.autograd.grad(rd.ragged_dot_float8(leaf, A_leaf, gs), (leaf, A_leaf), dout)
    for row, col in ((0, 1), (2, 77), (3, 127), (7, 64)):
        moved = x.clone()
        moved[row, col] += 1 if moved[row, col] < 8 else -1
        by = (moved - x)[row, col].item()
        assert abs((loss(moved, A) - loss(x, A)).item() - by * dx[row, col].item()) <= (0 if apart else 2 * 7 * 16 * 448)
    for e, row, col in ((0, 1, 5), (1, 127, 127), (1, 64, 1)):
        moved = A.clone()
        moved[e, row, col] += 1 if moved[e, row, col] < 8 else -1
        by = (moved - A)[e, row, col].item()
        assert (loss(x, moved) - loss(x, A)).item() == by * dA[e, row, col].item()


def test_operands_beyond_2_31_elements():
    """Rows, weights and results whose offsets do not fit 32 bits, at samples on both sides of them."""
    m, k, n = 300_000, 8192, 256
    print("big index: float8 rows", m, k, flush=True)
    x = torch.empty((m, k), dtype=torch.bfloat16, device="cuda").normal_()
    edge = 2 ** 31 // k
    sample = torch.tensor([0, 1, edge - 1, edge, edge + 1, m - 2, m - 1], device="cuda")
    held = rd.quantize_rows(x)
    few = rd.quantize_rows(x[sample])
    assert torch.equal(held.codes.view(torch.uint8)[sample], few.codes.view(torch.uint8)) and torch.equal(held.scales[sample], few.scales)
    assert torch.equal(rd.dequantize(held)[sample], rd.dequantize(few))
    A = torch.randn(2, k, n, device="cuda").bfloat16() * k ** -0.5
    w = rd.quantize_weights(A)
    y = rd.ragged_dot_float8(held, w, torch.tensor([edge + 1, m - edge - 3], dtype=torch.int32, device="cuda"))
    want = rd.ragged_dot_float8(few, w, torch.tensor([4, 2], dtype=torch.int32, device="cuda"))
    want[6] = 0  # rows behind the last group
    got = y[sample]
    assert not got[5:].any() and torch.equal(got[:5], want[:5])
    del x, held, y
    g, k, n = 150, 4096, 4096
    print("big index: float8 weights", g, k, n, flush=True)
    A = torch.empty((g, k, n), dtype=torch.bfloat16, device="cuda").normal_()
    w = rd.quantize_weights(A)
    sizes = torch.zeros(g, dtype=torch.int32, device="cuda")
    sizes[[0, 127, 128, 149]] = torch.tensor([3, 5, 70, 2], dtype=torch.int32, device="cuda")
    x = torch.randn(80, k, device="cuda").bfloat16()
    for trans in (False, True):
        y = rd.ragged_dot_float8(x, w, sizes, trans_rhs=trans)
        row = 0
        for e, size in ((0, 3), (127, 5), (128, 70), (149, 2)):
            one = rd.quantize_weights(A[e:e + 1])
            assert torch.equal(one.codes.view(torch.uint8)[0], w.codes.view(torch.uint8)[e]) and torch.equal(one.scales[0], w.scales[e])
            alone = rd.ragged_dot_float8(x[row:row + size], one, torch.tensor([size], dtype=torch.int32, device="cuda"), trans_rhs=trans)
            assert torch.equal(alone, y[row:row + size])
            row += size
    del w
    print("big index: orthogonalize", g, k, n, flush=True)
    out = rd.orthogonalize(A, steps=1)
    for e in (0, 127, 128, 149):
        assert torch.equal(rd.orthogonalize(A[e], steps=1), out[e])


@pytest.mark.parametrize("seed", range(12))
def test_random_products(seed):
    """Any sizes: against torch's products in float64 of what the operands are held as."""
    rng = np.random.default_rng(seed)
    m, k, n, g = (int(np.exp(rng.uniform(0, np.log(t)))) for t in (3000, 1500, 1500, 300))
    trans, pow2 = bool(rng.integers(2)), bool(rng.integers(2))
    dtype = [torch.bfloat16, torch.float16, torch.float32][rng.integers(3)]
    sizes = rng.multinomial(int(m * rng.uniform(0.5, 1.2)), rng.dirichlet(np.full(g, 0.3))).astype(np.int32)
    print(f"random {seed}: {m} x {k} x {n}, {g} groups, trans={trans} {dtype}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((m, k), generator=gen, device="cuda").to(dtype)
    A = torch.randn((g, n, k) if trans else (g, k, n), generator=gen, device="cuda").to(dtype)
    xq, wq = rd.quantize_rows(x, pow2=pow2), rd.quantize_weights(A, pow2=pow2)
    y = rd.ragged_dot_float8(xq, wq, torch.from_numpy(sizes), trans_rhs=trans, out_dtype=dtype)
    xv, wv = rd.dequantize(xq, torch.float32).double(), rd.dequantize(wq, torch.float32).double()
    ref, mag, row = torch.zeros(m, n, dtype=torch.float64, device="cuda"), torch.zeros(m, n, dtype=torch.float64, device="cuda"), 0
    for e, size in enumerate(sizes.tolist()):
        at = slice(row, min(m, row + size))
        w = wv[e].t().contiguous() if trans else wv[e]
        ref[at], mag[at] = xv[at] @ w, xv[at].abs() @ w.abs()
        row = min(m, row + size)
    # of eight products at most seven lose 2^-13 of the largest of them: less than 2^-10 of their sum; then fp32 sums, then the result's rounding
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
    assert ((y.double() - ref).abs() <= (2.0 ** -10 + k * 2.0 ** -24) * mag + half * ref.abs() + 2.0 ** -25).all()
    assert not y[row:].any()
