"""Expert ids and weights from a router's logits, and the gradient of the logits, against the float64 restatement."""

import numpy as np
import pytest
import torch

from gpu_ragged_dot_amd import moe
from oracle import expert_ops_oracle as oracle

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LEAST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # half the least number above 0
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _logits(seed, tokens, experts, dtype, spread=1.5):
    rng = np.random.default_rng(seed)
    return torch.from_numpy(spread * rng.standard_normal((tokens, experts))).to(dtype).cuda()


def _error_unit(l, score):
    """Relative error of a score in 32 bits: an exponential of an argument a (a rounding of a, and of a over log 2: 2^-24 |a| each,
    and 2 units of its own), sums and quotients of those; 24 units of 2^-23 for what does not grow with a."""
    a = np.where(np.isfinite(l), l, 0)
    far = np.abs(a).max(1, keepdims=True) if score == "sigmoid" else a.max(1, keepdims=True) - a.min(1, keepdims=True)
    return (24 + 4 * far) * 2.0 ** -23


def _check(logits, top_k, bias=None, grad=True, **kw):
    l = logits.double().cpu().numpy()
    b = None if bias is None else bias.double().cpu().numpy()
    ids, w = oracle.gate(l, top_k, bias=b, **kw)
    leaf = logits.detach().requires_grad_(grad)
    got = moe.gate(leaf, top_k, bias=bias, **kw)
    assert got.expert_ids.dtype == torch.int32 and got.weights.dtype == torch.float32
    assert np.array_equal(got.expert_ids.cpu().numpy(), ids)
    unit = 2 * _error_unit(l, kw.get("score", "softmax"))
    assert np.all(np.abs(got.weights.detach().double().cpu().numpy() - w) <= unit * np.abs(w) + 2.0 ** -126)
    if not grad:
        return
    dw = torch.randn(w.shape, generator=torch.Generator().manual_seed(7)).cuda()
    dl = torch.autograd.grad(got.weights, leaf, dw)[0]
    assert dl.dtype == logits.dtype
    dwn = dw.double().cpu().numpy()
    g_kw = {k: v for k, v in kw.items() if k in ("score", "renormalize", "scale")}
    ref = oracle.gate_grad(l, ids, dwn, **g_kw)
    # each term carries the error of a weight; the terms are q_i = w_i dw_i at the chosen ones and a share of their sum: of
    # w_i / scale where renormalised, of every expert's score where not (softmax)
    q = np.abs(w * dwn)
    magnitude = np.zeros_like(ref)
    shared = np.abs(w) / abs(kw.get("scale", 1.0)) * q.sum(1, keepdims=True) if kw.get("renormalize", True) else 0 * q
    for t in range(len(l)):
        live = ids[t] >= 0
        magnitude[t, ids[t][live]] += (q + shared)[t][live]
        if kw.get("score", "softmax") == "softmax" and not kw.get("renormalize", True):
            magnitude[t] += oracle.scores(l[t], "softmax") * q[t].sum()
    err = np.abs(dl.double().cpu().numpy() - ref)
    # (the restatement takes differences of terms of the size of q in 64 bits, 2^-52 of them, where the gradient is 0)
    magnitude += 2.0 ** -30 * q.sum(1, keepdims=True)
    assert np.all(err <= 2 * unit * magnitude + HALF_ULP[logits.dtype] * np.abs(ref) + LEAST[logits.dtype] + 2.0 ** -126)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (1, 128, 8), (3, 2, 2), (5, 7, 7), (64, 64, 6), (33, 65, 5), (17, 200, 16),
                                                  (9, 256, 8), (7, 257, 64), (6, 512, 3), (5, 1000, 10), (4, 1024, 64)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_plain(tokens, experts, top_k, score, dtype):
    print(f"gate {tokens} x {experts} top {top_k} {score} {dtype}", flush=True)
    logits = _logits(tokens + experts, tokens, experts, dtype)
    for renormalize in (True, False):
        _check(logits, top_k, score=score, renormalize=renormalize, scale=1.0 if renormalize else 2.5)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("experts,clusters,top_clusters,top_k", [(256, 8, 4, 8), (64, 64, 9, 9), (24, 4, 1, 6), (160, 8, 3, 6), (128, 2, 2, 4),
                                                                 (18, 6, 3, 5), (1024, 16, 2, 32), (320, 64, 7, 8)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_clusters_and_bias(experts, clusters, top_clusters, top_k, score, dtype):
    print(f"gate clusters {clusters} of {experts} {score} {dtype}", flush=True)
    logits = _logits(experts + clusters, 29, experts, dtype)
    steps = torch.randint(-40, 41, (experts,), generator=torch.Generator().manual_seed(experts)).float().cuda() * 0.001
    for cluster_score in ("max", "top2"):
        for bias in (None, steps):
            _check(logits, top_k, bias=bias, score=score, clusters=clusters, top_clusters=top_clusters, cluster_score=cluster_score, scale=2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_ties_go_to_the_lower_index(score, biased):
    """Logits of a handful of values (bfloat16 rows are full of equals), in and across lanes; whole rows of one value."""
    rng = np.random.default_rng(3)
    bias = torch.zeros(96, device="cuda") if biased else None
    for values in ([0.0], [0.5, -0.5], [1.0, 2.0, 3.0]):
        logits = torch.from_numpy(rng.choice(values, (41, 96)).astype(np.float32)).cuda()
        _check(logits, 8, bias=bias, score=score)
        for cluster_score in ("max", "top2"):
            _check(logits, 8, bias=bias, score=score, clusters=8, top_clusters=3, cluster_score=cluster_score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_near_ties_are_decided_in_64_bits(score):
    """Ranks score + bias that differ by less than a rounding of 32 bits: the bias makes up for the difference of two scores
    but for a part in 2^30 of it."""
    rng = np.random.default_rng(5)
    experts, tokens = 64, 200
    row = rng.standard_normal(experts).astype(np.float32)
    s = oracle.scores(row.astype(np.float64), score)
    bias = (1.0 - s).astype(np.float32)  # ranks 1 +- 2^-25: float32 sums are all equal
    logits = torch.from_numpy(np.stack([row] * tokens)).cuda()
    logits[1::2] += 0.5 * torch.randn((tokens // 2, experts), generator=torch.Generator().manual_seed(1)).cuda()
    _check(logits, 12, bias=torch.from_numpy(bias).cuda(), score=score)
    _check(logits, 12, bias=torch.from_numpy(bias).cuda(), score=score, clusters=8, top_clusters=3, cluster_score="top2")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,top_k", [(16, 1), (40, 11), (64, 12), (64, 13), (256, 15), (256, 16), (256, 17), (600, 9)])
def test_close_float32_logits(score, experts, top_k):
    """Rows in which a few, some or all logits lie units in the last place apart: what the leading ones settle, and what they do
    not (more close ones than that)."""
    gen = torch.Generator().manual_seed(experts + top_k)
    logits = torch.randn((64, experts), generator=gen)
    for t in range(64):
        crowd = torch.randperm(experts, generator=gen)[:1 + t * experts // 64]
        at = logits[t].topk(min(top_k, experts - 1)).values[-1]  # in the middle of the choice
        logits[t, crowd] = at + torch.randint(-6, 7, (len(crowd),), generator=gen) * 2.0 ** -23
    bias = torch.randint(-2, 3, (experts,), generator=gen).float().cuda() * 2.0 ** -22
    _check(logits.cuda(), top_k, score=score)
    _check(logits.cuda(), top_k, score=score, bias=bias)
    _check(logits.cuda(), top_k, score=score, bias=bias * 2.0 ** 22)
    if experts % 8 == 0 and top_k <= experts // 2:
        _check(logits.cuda(), top_k, score=score, clusters=8, top_clusters=4)
        _check(logits.cuda(), top_k, score=score, bias=bias, clusters=8, top_clusters=4, cluster_score="top2")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("cluster_score", ["max", "top2"])
@pytest.mark.parametrize("experts,clusters,dtype", [(256, 8, torch.float32), (64, 16, torch.float32), (96, 6, torch.float32), (32, 2, torch.float32),
                                                    (256, 8, torch.bfloat16), (128, 4, torch.float16)])
def test_close_clusters(score, cluster_score, experts, clusters, dtype):
    """Clusters whose best experts are those of another one but for units in the last place, or (16-bit types) all the same; in some
    rows a third expert is as close."""
    gen = torch.Generator().manual_seed(experts + clusters)
    size, tokens = experts // clusters, 64
    logits = 0.3 * torch.randn((tokens, clusters, size), generator=gen)
    best = 1.5 + torch.rand((tokens, 1, 2), generator=gen) + torch.randint(-4, 5, (tokens, clusters, 2), generator=gen) * 2.0 ** -23
    logits[:, :, :2] = best
    logits[::3, :, 2] = best[::3, :, 1] - torch.randint(0, 3, (tokens // 3 + 1, clusters), generator=gen) * 2.0 ** -23
    order = torch.stack([torch.randperm(size, generator=gen) for _ in range(tokens * clusters)]).view(tokens, clusters, size)
    logits = logits.gather(2, order).view(tokens, experts).to(dtype).cuda()
    bias = torch.zeros(experts) + (torch.randint(-1, 2, (clusters, 1), generator=gen) * 2.0 ** -24).expand(clusters, size).reshape(-1)
    for b in (None, bias.cuda()):
        for top_clusters in (1, clusters // 2):
            _check(logits, min(3, size), bias=b, score=score, clusters=clusters, top_clusters=top_clusters, cluster_score=cluster_score)


@pytest.mark.parametrize("seed", range(60))
def test_random_calls(seed):
    """Sizes, clusters, types, scores and biases of every kind at once: small, larger than the scores, of 1e30, -inf."""
    rng = np.random.default_rng(1000 + seed)
    experts = int(rng.integers(1, 1025) if seed % 3 else 8 * rng.integers(1, 65))
    clusters = int(rng.choice([c for c in range(1, 65) if experts % c == 0]))
    top_clusters = int(rng.integers(1, clusters + 1))
    top_k = int(rng.integers(1, min(64, top_clusters * (experts // clusters)) + 1))
    kw = dict(score=str(rng.choice(["softmax", "sigmoid"])), clusters=clusters, top_clusters=top_clusters, cluster_score=str(rng.choice(["max", "top2"])),
              renormalize=bool(rng.integers(2)), scale=float(rng.choice([1.0, 2.5, -0.5])))
    dtype = TYPES[seed % 3]
    logits = _logits(seed, int(rng.integers(1, 80)), experts, dtype)
    logits[torch.from_numpy(rng.random(logits.shape) < rng.choice([0, 0.1, 0.9])).cuda()] = -torch.inf
    bias = rng.integers(-9, 10, experts) * rng.choice([0.001, 1.0, 1e6, 1e30], experts if seed % 2 else 1)
    bias[rng.random(experts) < rng.choice([0, 0.1, 1.0], p=[0.5, 0.4, 0.1])] = -np.inf
    print(f"gate {tuple(logits.shape)} top {top_k} {dtype} {kw}", flush=True)
    _check(logits, top_k, bias=torch.from_numpy(bias.astype(np.float32)).cuda() if rng.integers(3) else None, **kw)


@pytest.mark.parametrize("experts", [64, 256, 1000])
def test_biases_that_are_not_finite(experts):
    """An infinite or NaN bias ranks its expert first and leaves the others' order and all weights finite."""
    logits = _logits(31, 9, experts, torch.float32)
    for score in ("softmax", "sigmoid"):
        for value in (torch.inf, torch.nan):
            bias = torch.zeros(experts, device="cuda")
            bias[[5, 40]] = value
            got, rest = moe.gate(logits, 6, score=score, bias=bias), moe.gate(logits, 8, score=score, bias=torch.zeros(experts, device="cuda"))
            assert got.weights.isfinite().all()
            for row, others in zip(got.expert_ids.tolist(), rest.expert_ids.tolist()):
                assert row[:2] == [5, 40] and row[2:] == [e for e in others if e not in (5, 40)][:4]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_shut_experts_and_rows(score, renormalize):
    logits = _logits(11, 24, 40, torch.float32)
    logits[:, 30:] = -torch.inf      # a padded table
    logits[3] = -torch.inf           # a masked token
    logits[4, 2:] = -torch.inf       # fewer experts than top_k
    logits[5, :39] = -torch.inf
    logits[5, 39] = 1.0
    _check(logits, 6, score=score, renormalize=renormalize)
    _check(logits, 6, score=score, renormalize=renormalize, clusters=4, top_clusters=2)
    _check(logits, 6, score=score, renormalize=renormalize, clusters=4, top_clusters=2, cluster_score="top2")
    bias = torch.zeros(40, device="cuda")
    bias[7] = -torch.inf
    _check(logits, 6, bias=bias, score=score, renormalize=renormalize)
    got = moe.gate(logits, 6, score=score)
    r = moe.route(got.expert_ids, 40)
    assert int(r.group_sizes.sum()) == int((got.expert_ids >= 0).sum())
    assert not got.weights[3].any()


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "f16", "f32"])
def test_extreme_logits(dtype):
    """Rows of the type's lowest value, of large ones, of scores that 32 bits do not hold; sigmoid scores all close to 0 divide
    by their sum all the same."""
    low = torch.finfo(dtype).min
    logits = torch.tensor([[low] * 12, [low] * 11 + [0.0], [60.0, 59.0] * 6, [-60.0, -59.0, -58.5, -61.0] * 3], dtype=dtype, device="cuda")
    for score in ("softmax", "sigmoid"):
        got = moe.gate(logits, 3, score=score)
        ids, _ = oracle.gate(logits.double().cpu().numpy(), 3, score="softmax")
        assert np.array_equal(got.expert_ids.cpu().numpy(), ids)
        assert torch.allclose(got.weights.sum(1), torch.ones(4, device="cuda"), rtol=0, atol=2.0 ** -20)
    _check(logits[3:], 3, score="sigmoid")
    _check(logits[2:], 3, score="softmax", renormalize=False)


def test_nan_and_infinity_stay_in_their_rows():
    logits = _logits(2, 6, 48, torch.float32)
    want = moe.gate(logits, 4)
    spoilt = logits.clone()
    spoilt[1, 5] = torch.nan
    spoilt[3] = torch.nan
    spoilt[4, 0] = torch.inf
    for score in ("softmax", "sigmoid"):
        for kw in (dict(), dict(clusters=8, top_clusters=2, cluster_score="top2"), dict(bias=torch.zeros(48, device="cuda"))):
            got = moe.gate(spoilt, 4, score=score, **kw)
            ids = got.expert_ids.cpu().numpy()
            assert ids.min() >= 0 and ids.max() < 48 and all(len(set(r)) == 4 for r in ids)
            assert got.weights[1].isnan().all() and got.weights[3].isnan().all()
            assert got.weights[4].isnan().all() if score == "softmax" else got.weights[4].isfinite().all()
            assert got.weights[[0, 2, 5]].isfinite().all()
    got = moe.gate(spoilt, 4)
    assert torch.equal(got.expert_ids[[0, 2, 5]], want.expert_ids[[0, 2, 5]]) and torch.equal(got.weights[[0, 2, 5]], want.weights[[0, 2, 5]])


def test_many_tokens():
    """More rows than any launch's blocks take at once, decided as in 64 bits on all of them (by torch, on the device)."""
    tokens, experts = 70001, 128
    logits = torch.randn((tokens, experts), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    bias = 0.001 * torch.randint(-20, 20, (experts,), device="cuda").float()
    rank = torch.sigmoid(logits.double()) + bias.double()
    ids = rank.sort(dim=1, descending=True, stable=True).indices[:, :6]
    got = moe.gate(logits, 6, score="sigmoid", bias=bias)
    assert torch.equal(got.expert_ids.long(), ids)
    s = torch.sigmoid(logits.double()).gather(1, ids)
    assert torch.allclose(got.weights.double(), s / s.sum(1, keepdim=True), rtol=2.0 ** -18, atol=0)


def test_strided_logits_other_types_of_bias_and_empty_batches():
    logits = _logits(8, 10, 64, torch.float32)
    wide = torch.randn(10, 128, device="cuda")
    wide[:, ::2] = logits
    got, want = moe.gate(wide[:, ::2], 4), moe.gate(logits, 4)
    assert torch.equal(got.expert_ids, want.expert_ids) and torch.equal(got.weights, want.weights)
    odd = torch.empty(641, device="cuda")[1:].view(10, 64).copy_(logits)  # not on a 16-byte boundary
    assert torch.equal(moe.gate(odd, 4).weights, want.weights)
    bias = (0.25 * torch.arange(64, device="cuda")).half()
    assert torch.equal(moe.gate(logits, 4, bias=bias).expert_ids, moe.gate(logits, 4, bias=bias.float()[None]).expert_ids)
    empty = moe.gate(torch.empty((0, 64), device="cuda", requires_grad=True), 4)
    assert empty.expert_ids.shape == (0, 4)
    learnt = bias.float().requires_grad_()  # moves the choice only: no gradient
    out = moe.gate(logits.detach().requires_grad_(), 4, bias=learnt)
    out.weights.sum().backward()
    assert learnt.grad is None and not out.expert_ids.requires_grad
    with pytest.raises(ValueError, match="bias"):
        moe.gate(logits, 4, bias=bias[:3])
    with pytest.raises(RuntimeError, match="same device"):
        moe.gate(logits, 4, bias=bias.cpu())


def test_replayed_and_on_another_stream():
    """A captured call with its gradient, replayed on new logits with eager work between the replays, and a call on a stream of
    its own."""
    logits = _logits(21, 64, 256, torch.float32).requires_grad_()
    dw = torch.randn(64, 8, device="cuda")
    kw = dict(score="sigmoid", clusters=8, top_clusters=4, cluster_score="top2", scale=2.5, bias=torch.zeros(256, device="cuda"))

    def step():
        got = moe.gate(logits, 8, **kw)
        return got.expert_ids, got.weights, torch.autograd.grad(got.weights, logits, dw)[0]

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
    for seed in (22, 23, 24):
        with torch.no_grad():
            logits.copy_(_logits(seed, 64, 256, torch.float32))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)
