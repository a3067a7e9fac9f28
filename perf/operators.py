"""The operators around the ragged products of a mixture of experts, as cases that a timing program can prepare, run and
compare:

* ``gate``    expert scores to expert ids and weights (softmax or sigmoid, a balance bias, clusters, top-k, renormalised);
              ``train`` adds the gradient of the logits;
* ``swiglu``  the gated activation between an expert's two products; ``train`` adds the gradient of its input;
* ``int4``    the ragged product on weights held as 4-bit integers with a scale (and a zero point) per block.

With ``own`` false a pass is computed by elementary torch operations, with ``own`` true by this package.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _gate(tokens, experts, top_k, dtype="f32", score="softmax", biased=False, clusters=1, top_clusters=1,
          cluster_score="max", renormalize=True, scale=1.0, absent=0, train=False, **name):
    """``absent``: experts at the end whose logits are -inf, as where a table of experts is padded."""
    return dict(kind="gate", tokens=tokens, experts=experts, top_k=top_k, dtype=dtype, score=score, biased=biased,
                clusters=clusters, top_clusters=top_clusters, cluster_score=cluster_score, renormalize=renormalize,
                scale=scale, absent=absent, train=train, **name)


def _swiglu(rows, f, dtype="bf16", train=False, **name):
    return dict(kind="swiglu", rows=rows, f=f, dtype=dtype, train=train, **name)


def _int4(m, k, n, g, block=128, zeros=False, dtype="bf16", routing="topk", fill=1.0, **name):
    """``fill``: which share of the m rows belongs to a group (a padded batch has a tail of rows that do not)."""
    return dict(kind="int4", m=m, k=k, n=n, g=g, block=block, zeros=zeros, dtype=dtype, routing=routing, fill=fill, **name)


def listed():
    return [
        # one decoding step of 8 sequences, top-8 of 128 experts: nothing but latency
        _gate(8, 128, 8, dtype="bf16", name="gate_decode_8_tokens"),
        # a prompt of 4096 tokens in serving: sigmoid scores, a balance bias, 4 of 8 clusters, top-8 of 256 experts
        _gate(4096, 256, 8, score="sigmoid", biased=True, clusters=8, top_clusters=4, cluster_score="top2", scale=2.5,
              name="gate_prefill_clusters"),
        # the same router in a training step of 32768 tokens, with the gradient of its logits
        _gate(32768, 256, 8, score="sigmoid", biased=True, clusters=8, top_clusters=4, cluster_score="top2", scale=2.5,
              train=True, name="gate_train_clusters"),
        # softmax scores used as they are, a table padded from 60 to 64 experts, an odd number of tokens, float16
        _gate(4099, 64, 4, dtype="f16", renormalize=False, absent=4, train=True, name="gate_train_padded_table"),
        # the activation of one decoding step: 8 sequences x top-8 rows
        _swiglu(64, 768, name="swiglu_decode_8_tokens"),
        # float32 training, a width that no vector divides
        _swiglu(4099, 1515, dtype="f32", train=True, name="swiglu_train_odd_float32"),
        # a training step's rows: 4096 tokens x top-8 of experts 2048 wide
        _swiglu(32768, 2048, train=True, name="swiglu_train"),
        # one decoding step of 8 sequences, top-8 of 128 experts: a stream over the 4-bit weights
        _int4(64, 2048, 768, 128, name="int4_decode_8_tokens"),
        # a batch of 64 sequences on the finest blocks in common use below 128, with zero points, float16
        _int4(512, 2048, 768, 128, block=64, zeros=True, dtype="f16", name="int4_decode_64_tokens_zeros"),
        # sizes that nothing divides, the smallest blocks, a padded batch
        _int4(515, 1001, 1515, 12, block=32, zeros=True, routing="softmax", fill=0.9, name="int4_odd_sizes"),
        # a prompt's rows on 32 experts, softmax-distributed
        _int4(8192, 7168, 2048, 32, routing="softmax", name="int4_prefill_32_experts"),
        # long prompts on 8 large experts: the matrix cores are what bounds it
        _int4(16384, 4096, 14336, 8, name="int4_prefill_8_large_experts"),
    ]


def _log_int(rng, lo, hi, step=1):
    """An integer in [lo, hi], uniform in its logarithm, rounded to a multiple of ``step``."""
    return max(lo, min(hi, step * round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)))


def draw(rng):
    while True:
        kind = rng.choice(["gate", "swiglu", "int4", "int4"])
        if kind == "gate":
            clusters = rng.choice([1, 1, 4, 8])
            experts = clusters * _log_int(rng, 8 // clusters + 1, 512 // clusters)
            top_clusters = rng.randint(1, clusters)
            top_k = rng.randint(1, min(16, experts // clusters * top_clusters))
            case = _gate(_log_int(rng, 1, 32768), experts, top_k, dtype=rng.choice(["bf16", "f16", "f32", "f32"]),
                         score=rng.choice(["softmax", "sigmoid"]), biased=rng.random() < 0.5, clusters=clusters,
                         top_clusters=top_clusters, cluster_score=rng.choice(["max", "top2"]),
                         renormalize=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), train=rng.random() < 0.5)
            if case["tokens"] * experts > 32768 * 256:
                continue
        elif kind == "swiglu":
            case = _swiglu(_log_int(rng, 1, 65536), _log_int(rng, 64, 8192, rng.choice([1, 64])),
                           dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), train=rng.random() < 0.6)
            if case["rows"] * case["f"] * _BYTES[case["dtype"]] > 32768 * 2048 * 2:
                continue
        else:
            step = rng.choice([1, 64, 64])
            case = _int4(_log_int(rng, 1, 16384), _log_int(rng, 256, 8192, step), _log_int(rng, 256, 14336, step),
                         _log_int(rng, 2, 256), block=rng.choice([32, 64, 128, 128]), zeros=rng.random() < 0.5,
                         dtype=rng.choice(["bf16", "f16"]), routing=rng.choice(["topk", "softmax", "zipf"]),
                         fill=rng.choice([1.0, 1.0, 0.8]))
            if case["g"] * case["k"] * case["n"] > 8 * 4096 * 14336 or work(case)["flops"] > 2.0 * 16384 * 4096 * 14336:
                continue
        return case


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _shares(routing, g, rng):
    """The probability of each expert: equal, softmax of N(0, 1) logits, or a permuted Zipf law with a tenth empty."""
    if routing == "softmax":
        p = np.exp(rng.standard_normal(g))
    elif routing == "zipf":
        p = (rng.permutation(g) + 1.0) ** -1.1
        p[rng.choice(g, size=g // 10, replace=False)] = 0.0
    else:
        p = np.ones(g)
    return p / p.sum()


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _gate_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    tokens, experts = case["tokens"], case["experts"]
    # a router's logits spread over a few units, and some experts are liked better than others
    logits = 1.2 * _randn(gen, tokens, experts) + 0.5 * _randn(gen, 1, experts)
    if case["absent"]:
        logits[:, experts - case["absent"]:] = -math.inf
    # a bias that moved in steps of 0.001 until the load was even
    bias = (30 * _randn(gen, experts)).round() * 0.001 if case["biased"] else None
    return dict(logits=logits.to(_TYPES[case["dtype"]]), bias=bias, dweights=_randn(gen, tokens, case["top_k"]))


def _swiglu_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    y = torch.empty((case["rows"], 2 * case["f"]), dtype=dtype, device="cuda")
    dout = torch.empty((case["rows"], case["f"]), dtype=dtype, device="cuda")
    for t in (y, dout):
        for part in t.split(8192):
            part.copy_(_randn(gen, *part.shape))
    return dict(y=y, dout=dout)


def _int4_inputs(case, seed):
    """Normal weights quantised block by block: symmetric (codes 1..15 around 8) or from the least to the largest."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    m, k, n, g, block, dtype = (case[c] for c in ("m", "k", "n", "g", "block", "dtype"))
    dtype, blocks = _TYPES[dtype], -(-k // block)
    q = torch.empty((g, n, k), dtype=torch.uint8, device="cuda")
    scales = torch.empty((g, n, blocks), dtype=dtype, device="cuda")
    zeros = torch.empty((g, n, blocks), dtype=torch.uint8, device="cuda") if case["zeros"] else None
    for e in range(g):
        w = _randn(gen, n, blocks, block).mul_(k ** -0.5)
        if zeros is None:
            s = (w.abs().amax(2, keepdim=True) / 7).to(dtype)
            z = 8.0
        else:
            lo, hi = w.amin(2, keepdim=True), w.amax(2, keepdim=True)
            s = ((hi - lo) / 15).to(dtype)
            z = (-lo / s.float()).round_().clamp_(0, 15)
            zeros[e] = z[..., 0].to(torch.uint8)
        scales[e] = s[..., 0]
        w.div_(s.float()).add_(z).round_().clamp_(0, 15)
        q[e] = w.to(torch.uint8).view(n, blocks * block)[:, :k]
    sizes = rng.multinomial(round(m * case["fill"]), _shares(case["routing"], g, rng)).astype(np.int32)
    return dict(x=_randn(gen, m, k).to(dtype), q=q, scales=scales, zeros=zeros, sizes=sizes)


_INPUTS = {"gate": _gate_inputs, "swiglu": _swiglu_inputs, "int4": _int4_inputs}


def prepare(case, seed):
    state = _INPUTS[case["kind"]](case, seed)
    state["case"] = case
    if case.get("train"):
        state["logits" if case["kind"] == "gate" else "y"].requires_grad_()
    if case["kind"] == "int4":
        state["group_sizes"] = torch.from_numpy(state["sizes"]).cuda()
        if own:  # weights are laid out once, when a program loads them
            import gpu_ragged_dot_amd as rd
            state["weights"] = rd.pack_int4(state["q"], state["scales"], state["zeros"], block=case["block"], trans_rhs=True)
            del state["q"], state["scales"], state["zeros"]
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return (_run_own if own else _run_plain)[case["kind"]](case, state)


def _own_gate(case, s):
    import gpu_ragged_dot_amd as rd
    with torch.set_grad_enabled(case["train"]):
        ids, weights = rd.moe.gate(s["logits"], case["top_k"], score=case["score"], bias=s["bias"], clusters=case["clusters"],
                                   top_clusters=case["top_clusters"], cluster_score=case["cluster_score"],
                                   renormalize=case["renormalize"], scale=case["scale"])
    if not case["train"]:
        return ids, weights
    return (ids, weights.detach()) + torch.autograd.grad(weights, s["logits"], s["dweights"])


def _own_swiglu(case, s):
    import gpu_ragged_dot_amd as rd
    with torch.set_grad_enabled(case["train"]):
        out = rd.moe.swiglu(s["y"])
    if not case["train"]:
        return out
    return (out.detach(),) + torch.autograd.grad(out, s["y"], s["dout"])


def _own_int4(case, s):
    import gpu_ragged_dot_amd as rd
    return rd.ragged_dot_int4(s["x"], s["weights"], s["group_sizes"])


def _plain_gate(case, s):
    logits, bias = s["logits"].detach(), s["bias"]
    tokens, experts = logits.shape
    # which experts: compared in 64 bits (without a bias and sums of scores, by the logits themselves, which is the same order)
    wide = logits.double()
    if bias is None and (case["clusters"] == 1 or case["cluster_score"] == "max"):
        choice = wide
    else:
        choice = torch.softmax(wide, 1) if case["score"] == "softmax" else torch.sigmoid(wide)
        if bias is not None:
            choice = choice + bias.double()
        choice = choice.masked_fill(wide == -math.inf, -math.inf)
    if case["clusters"] > 1:
        inside = choice.view(tokens, case["clusters"], -1).sort(dim=2, descending=True).values
        best = inside[..., 0] if case["cluster_score"] == "max" else inside[..., :2].sum(2)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :case["top_clusters"]]
        shut = torch.ones_like(best, dtype=torch.bool).scatter_(1, kept, False)
        choice = choice.masked_fill(shut.repeat_interleave(experts // case["clusters"], 1), -math.inf)
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
    # their weights
    with torch.set_grad_enabled(case["train"]):
        leaf = logits.float().requires_grad_(case["train"])
        scores = torch.softmax(leaf, 1) if case["score"] == "softmax" else torch.sigmoid(leaf)
        weights = scores.gather(1, ids)
        if case["renormalize"]:
            weights = weights / weights.sum(1, keepdim=True)
        weights = weights * case["scale"]
    if not case["train"]:
        return ids.int(), weights
    return ids.int(), weights.detach(), torch.autograd.grad(weights, leaf, s["dweights"])[0].to(logits.dtype)


def _plain_swiglu(case, s):
    y = s["y"].detach()
    gate, up = y.float().chunk(2, dim=1)
    sig = 1 / (1 + torch.exp(-gate))
    out = (gate * sig * up).to(y.dtype)
    if not case["train"]:
        return out
    dout = s["dout"].float()
    dgate = dout * up * sig * (1 + gate * (1 - sig))
    return out, torch.cat((dgate, dout * gate * sig), 1).to(y.dtype)


def _dequantised(s, e, dtype, block):
    k = s["q"].shape[2]
    zero = 8.0 if s["zeros"] is None else s["zeros"][e].to(dtype).repeat_interleave(block, 1)[:, :k]
    return (s["q"][e].to(dtype) - zero) * s["scales"][e].to(dtype).repeat_interleave(block, 1)[:, :k]


def _plain_int4(case, s):
    x, row = s["x"], 0
    y = torch.zeros((case["m"], case["n"]), dtype=x.dtype, device=x.device)
    for e, size in enumerate(s["sizes"].tolist()):
        if size:
            y[row:row + size] = (x[row:row + size].float() @ _dequantised(s, e, torch.float32, case["block"]).t()).to(x.dtype)
        row += size
    return y


_run_plain = {"gate": _plain_gate, "swiglu": _plain_swiglu, "int4": _plain_int4}
_run_own = {"gate": _own_gate, "swiglu": _own_swiglu, "int4": _own_int4}


# ---- from the definitions, in 64 bits ------------------------------------------------------------------------------------
def _exact_gate(case, s):
    logits = s["logits"].detach().double()
    tokens, experts = logits.shape
    top = logits.amax(1, keepdim=True)
    if case["score"] == "softmax":
        e = (logits - top).exp()
        score, one_less = e / e.sum(1, keepdim=True), None
    else:
        score, one_less = 1 / (1 + (-logits).exp()), 1 / (1 + logits.exp())
    by_logit = s["bias"] is None and (case["clusters"] == 1 or case["cluster_score"] == "max")
    rank = logits if by_logit else score + (0.0 if s["bias"] is None else s["bias"].double())
    rank = torch.where(logits == -math.inf, torch.full_like(rank, -math.inf), rank)

    def leading(values, count):  # the largest ones one by one, the first of equals
        values, out = values.clone(), []
        width = torch.arange(values.shape[1], device=values.device)
        for _ in range(count):
            at = torch.where(values == values.amax(1, keepdim=True), width, values.shape[1]).amin(1, keepdim=True)
            out.append(at)
            values.scatter_(1, at, -math.inf)
        return torch.cat(out, 1)

    if case["clusters"] > 1:
        parts = rank.view(tokens * case["clusters"], -1)
        best = parts.amax(1)
        if case["cluster_score"] == "top2" and parts.shape[1] > 1:
            best = best + parts.scatter(1, leading(parts, 1), -math.inf).amax(1)
        keep = leading(best.view(tokens, -1), case["top_clusters"])
        mask = torch.zeros((tokens, case["clusters"]), dtype=torch.bool, device=rank.device).scatter_(1, keep, True)
        rank = torch.where(mask[:, :, None].expand(-1, -1, parts.shape[1]).reshape(tokens, experts), rank, -math.inf)
    ids = leading(rank, case["top_k"])
    chosen = score.gather(1, ids)
    total = chosen.sum(1, keepdim=True)
    weights = chosen * case["scale"] / (total if case["renormalize"] else 1.0)
    if not case["train"]:
        return ids.int(), weights
    dw = s["dweights"].double()
    inner = (dw * weights).sum(1, keepdim=True)
    if case["renormalize"]:
        # weights are homogeneous of degree 0 in the chosen scores, whose logarithms move by 1 (softmax) or 1 - score
        chosen_grad = weights * (dw - inner / case["scale"])
        if case["score"] == "sigmoid":
            chosen_grad = chosen_grad * one_less.gather(1, ids)
        grad = torch.zeros_like(logits).scatter_(1, ids, chosen_grad)
    elif case["score"] == "sigmoid":
        grad = torch.zeros_like(logits).scatter_(1, ids, weights * dw * one_less.gather(1, ids))
    else:
        grad = torch.zeros_like(logits).scatter_(1, ids, weights * dw) - score * inner
    return ids.int(), weights, grad


def _exact_swiglu(case, s):
    y = s["y"].detach().double()
    f = case["f"]
    gate, up = y[:, :f], y[:, f:]
    silu = gate / (1 + (-gate).exp())
    if not case["train"]:
        return silu * up
    dout = s["dout"].double()
    grad = torch.empty_like(y)
    grad[:, :f] = dout * up * (silu + (1 - silu) / (1 + (-gate).exp()))  # silu' = silu + sigmoid (1 - silu)
    grad[:, f:] = dout * silu
    return silu * up, grad


def _exact_int4(case, s):
    m, k, n, block = case["m"], case["k"], case["n"], case["block"]
    y = torch.zeros((m, n), dtype=torch.float64, device="cuda")
    first = np.concatenate(([0], np.cumsum(s["sizes"])))
    for e in np.flatnonzero(s["sizes"]):
        rows = slice(int(first[e]), int(first[e + 1]))
        for b in range(0, k, 16 * block):  # a few blocks of the contraction at a time
            part = slice(b, min(b + 16 * block, k))
            at = torch.arange(part.start, part.stop, device="cuda") // block
            codes = s["q"][e, :, part].double()
            codes -= 8.0 if s["zeros"] is None else s["zeros"][e].double()[:, at]
            y[rows] += s["x"][rows, part].double() @ (codes * s["scales"][e].double()[:, at]).t().contiguous()
    return y


_EXACT = {"gate": _exact_gate, "swiglu": _exact_swiglu, "int4": _exact_int4}


def exact(case, seed):
    with torch.no_grad():
        return _EXACT[case["kind"]](case, _INPUTS[case["kind"]](case, seed))


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    e = _BYTES[case["dtype"]]
    if case["kind"] == "gate":
        tokens, slots = case["tokens"], case["tokens"] * case["top_k"]
        scores = tokens * case["experts"] * e
        train = case["train"]
        return {"bytes": scores * (2 if train else 1) + slots * (12 if train else 8) + (4 * case["experts"] if case["biased"] else 0),
                "flops": 6.0 * tokens * case["experts"]}
    if case["kind"] == "swiglu":
        cells = case["rows"] * case["f"]
        return {"bytes": cells * e * (6 if case["train"] else 3), "flops": cells * (20.0 if case["train"] else 6.0)}
    m, k, n, g = case["m"], case["k"], case["n"], case["g"]
    rows = round(m * case["fill"])
    p = _shares(case["routing"], g, np.random.default_rng(0))
    live = float((1.0 - (1.0 - p) ** rows).sum())  # experts with a row at all, on average
    per_block = e + (1 if case["zeros"] else 0)
    return {"bytes": live * n * (k / 2 + -(-k // case["block"]) * per_block) + rows * k * e + m * n * e + 4 * g,
            "flops": 2.0 * rows * k * n}
