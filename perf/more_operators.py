"""The operators of training and serving an expert layer in 8 bits, and of updating its weights, as cases that a timing
program can prepare, run and compare:

* ``rows8``   rows to float8 with a scale for each block of 128 and back: as they are, sorted by expert on the way
              (``dispatch``) or behind the gated activation (``swiglu``);
* ``block8``  the ragged product on float8 rows and weights, a scale for each 128 of a row and each 128 x 128 of a weight
              matrix; ``train`` quantises both operands, and adds the gradients of both;
* ``ortho``   a stack of updates orthogonalised by Newton-Schulz products.

With ``own`` false a pass is computed by elementary torch operations, with ``own`` true by this package.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_BLOCK = 128
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _rows8(rows, k, source="rows", top_k=1, g=1, dtype="bf16", pow2=False, **name):
    """``source``: ``rows`` as they are, ``dispatch`` of rows / top_k tokens to g experts, or ``swiglu`` of [rows, 2 k]."""
    return dict(kind="rows8", rows=rows, k=k, source=source, top_k=top_k, g=g, dtype=dtype, pow2=pow2, **name)


def _block8(m, k, n, g, dtype="bf16", trans_rhs=False, routing="topk", fill=1.0, held=True, train=False, pow2=False, **name):
    """``held``: the rows come in 8 bits already, else the call quantises them.  ``fill``: which share of the m rows belongs
    to a group (a padded batch has a tail of rows that do not)."""
    return dict(kind="block8", m=m, k=k, n=n, g=g, dtype=dtype, trans_rhs=trans_rhs, routing=routing, fill=fill, held=held,
                train=train, pow2=pow2, **name)


def _ortho(g, k, n, dtype="bf16", **name):
    return dict(kind="ortho", g=g, k=k, n=n, dtype=dtype, **name)


def listed():
    return [
        # one decoding step of 8 sequences, top-8 of 128 experts: nothing but latency
        _rows8(64, 2048, source="dispatch", top_k=8, g=128, name="rows8_decode_dispatch"),
        # float32 activations of a width that nothing divides, scales that are powers of two
        _rows8(4099, 1515, dtype="f32", pow2=True, name="rows8_odd_float32"),
        # a training step's activation, 4096 tokens x top-8 of experts 2048 wide
        _rows8(32768, 2048, source="swiglu", name="rows8_train_swiglu"),
        # a training step's tokens on their way to 256 experts
        _rows8(32768, 7168, source="dispatch", top_k=8, g=256, name="rows8_train_dispatch"),
        # one decoding step of 8 sequences on weights stored [g, n, k], as checkpoints hold them: a stream over the weights
        _block8(64, 2048, 768, 128, trans_rhs=True, name="block8_decode_8_tokens"),
        # sizes that nothing divides, a padded batch, rows that the call quantises
        _block8(515, 1001, 1515, 12, dtype="f16", routing="softmax", fill=0.9, held=False, name="block8_odd_sizes"),
        # a prompt's rows on 32 experts, softmax-distributed
        _block8(8192, 7168, 2048, 32, trans_rhs=True, routing="softmax", name="block8_prefill_32_experts"),
        # long prompts on 8 large experts: the matrix cores are what bounds it
        _block8(16384, 4096, 14336, 8, held=False, name="block8_prefill_8_large_experts"),
        # a training step on 256 experts of very uneven load: quantised rows and weights, the product, both gradients
        _block8(32768, 7168, 2048, 256, routing="zipf", held=False, train=True, name="block8_train_256_experts"),
        # the smallest stack: a toy layer's gradients, where launches count
        _ortho(4, 256, 512, name="ortho_tiny"),
        # float32 momentum of odd shape
        _ortho(12, 1515, 1001, dtype="f32", name="ortho_odd_float32"),
        # the gradients of 128 experts, taller than wide
        _ortho(128, 2048, 768, name="ortho_128_experts"),
    ]


def _log_int(rng, lo, hi, step=1):
    """An integer in [lo, hi], uniform in its logarithm, rounded to a multiple of ``step``."""
    return max(lo, min(hi, step * round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)))


def draw(rng):
    while True:
        kind = rng.choice(["rows8", "block8", "block8", "ortho"])
        if kind == "rows8":
            source = rng.choice(["rows", "dispatch", "swiglu"])
            top_k = rng.choice([1, 2, 4, 8]) if source == "dispatch" else 1
            # (an activation computed in 32 bits lies next to a border of two codes now and then: 16-bit results)
            case = _rows8(top_k * _log_int(rng, 1, 32768 // top_k), _log_int(rng, 64, 8192, rng.choice([1, 64])), source=source,
                          top_k=top_k, g=_log_int(rng, max(2, top_k), 256), pow2=rng.random() < 0.4,
                          dtype=rng.choice(["bf16", "bf16", "f16"] + ([] if source == "swiglu" else ["f32"])))
            if case["rows"] * case["k"] * _BYTES[case["dtype"]] > 32768 * 7168 * 2:
                continue
        elif kind == "block8":
            step, train = rng.choice([1, 64, 128]), rng.random() < 0.3
            case = _block8(_log_int(rng, 1, 16384), _log_int(rng, 128, 8192, step), _log_int(rng, 128, 8192, step),
                           _log_int(rng, 2, 256), dtype=rng.choice(["bf16", "bf16", "f16"]), trans_rhs=rng.random() < 0.5,
                           routing=rng.choice(["topk", "softmax", "zipf"]), fill=rng.choice([1.0, 1.0, 0.8]),
                           held=not train and rng.random() < 0.5, train=train, pow2=rng.random() < 0.3)
            if work(case)["flops"] > 1.5e12 or case["g"] * case["k"] * case["n"] > 256 * 7168 * 2048 // 4:
                continue
        else:
            dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
            step = rng.choice([1, 64])
            case = _ortho(_log_int(rng, 1, 128), _log_int(rng, 32, 4096, step), _log_int(rng, 32, 8192, step), dtype=dtype)
            if work(case)["flops"] > work(_ortho(128, 2048, 768))["flops"] / (3 if dtype == "f32" else 1):
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


def _activations(gen, rows, k, dtype):
    """Normal rows of different sizes, with a few channels that are much larger than the others, as activations have them."""
    out = torch.empty((rows, k), dtype=dtype, device="cuda")
    channel = torch.where(torch.rand(k, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    for part in out.split(8192):
        part.copy_(_randn(gen, *part.shape) * channel * (0.5 * _randn(gen, len(part), 1)).exp())
    return out


def _rows8_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, k, dtype = case["rows"], case["k"], _TYPES[case["dtype"]]
    if case["source"] != "dispatch":
        return dict(x=_activations(gen, rows, 2 * k if case["source"] == "swiglu" else k, dtype))
    tokens = rows // case["top_k"]
    ids = torch.rand((tokens, case["g"]), generator=gen, device="cuda").argsort(1)[:, :case["top_k"]].int().contiguous()
    return dict(x=_activations(gen, tokens, k, dtype), ids=ids)


def _block8_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    m, k, n, g, dtype = (case[c] for c in ("m", "k", "n", "g", "dtype"))
    dtype = _TYPES[dtype]
    A = torch.empty((g, n, k) if case["trans_rhs"] else (g, k, n), dtype=dtype, device="cuda")
    for e in range(g):
        A[e] = _randn(gen, *A.shape[1:]) * k ** -0.5
    sizes = rng.multinomial(round(m * case["fill"]), _shares(case["routing"], g, rng)).astype(np.int32)
    return dict(x=_activations(gen, m, k, dtype), A=A, sizes=sizes, dout=_randn(gen, m, n).to(dtype) if case["train"] else None)


def _ortho_inputs(case, seed):
    """Gradients: a few directions that the tokens share, and noise."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g, k, n = case["g"], case["k"], case["n"]
    G = torch.empty((g, k, n), dtype=_TYPES[case["dtype"]], device="cuda")
    rank = max(1, min(k, n) // 16)
    for e in range(g):
        G[e] = 1e-3 * (_randn(gen, k, rank) @ _randn(gen, rank, n) * rank ** -0.5 + 0.3 * _randn(gen, k, n))
    return dict(G=G)


_INPUTS = {"rows8": _rows8_inputs, "block8": _block8_inputs, "ortho": _ortho_inputs}


def prepare(case, seed):
    s = _INPUTS[case["kind"]](case, seed)
    s["case"] = case
    if case["kind"] == "rows8" and case["source"] == "dispatch":
        if own:  # the router's work, the same for 16-bit rows
            import gpu_ragged_dot_amd as rd
            s["routing"] = rd.moe.route(s["ids"], case["g"])
        else:
            s["slots"] = s["ids"].reshape(-1).long().sort(stable=True).indices
    if case["kind"] == "block8":
        s["group_sizes"] = torch.from_numpy(s["sizes"]).cuda()
        if case["train"]:
            s["x"].requires_grad_()
            s["A"].requires_grad_()
            return s
        # weights are quantised once, when a program loads them, and `held` rows by what computed them
        if own:
            import gpu_ragged_dot_amd as rd
            s["weights"] = rd.quantize_weights(s.pop("A"), pow2=case["pow2"])
            if case["held"]:
                s["x"] = rd.quantize_rows(s["x"], pow2=case["pow2"])
        else:
            parts = [_plain_blocks(a, _BLOCK, case["pow2"]) for a in s.pop("A")]
            s["codes"], s["scales"] = (torch.stack(t) for t in zip(*parts))
            if case["held"]:
                s["x"] = _plain_blocks(s["x"], 1, case["pow2"])
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return (_run_own if own else _run_plain)[case["kind"]](case, state)


def _own_rows8(case, s):
    import gpu_ragged_dot_amd as rd
    if case["source"] == "dispatch":
        rows = rd.moe.dispatch(s["x"], s["routing"], float8=True, pow2=case["pow2"])
    elif case["source"] == "swiglu":
        rows = rd.moe.swiglu(s["x"], float8=True, pow2=case["pow2"])
    else:
        rows = rd.quantize_rows(s["x"], pow2=case["pow2"])
    return rd.dequantize(rows, s["x"].dtype)


def _own_block8(case, s):
    import gpu_ragged_dot_amd as rd
    how = dict(trans_rhs=case["trans_rhs"], out_dtype=_TYPES[case["dtype"]], pow2=case["pow2"])
    if not case["train"]:
        return rd.ragged_dot_float8(s["x"], s["weights"], s["group_sizes"], **how)
    y = rd.ragged_dot_float8(s["x"], s["A"], s["group_sizes"], **how)
    return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["A"]), s["dout"])


def _own_ortho(case, s):
    import gpu_ragged_dot_amd as rd
    return rd.orthogonalize(s["G"])


def _plain_blocks(x, height, pow2):
    """Codes of blocks of ``height`` x 128 and their scales: the least that maps a block to +-448, or the next power of two."""
    rows, cols = x.shape
    down, across = -(-rows // height), -(-cols // _BLOCK)
    x = torch.nn.functional.pad(x.detach().float(), (0, across * _BLOCK - cols, 0, down * height - rows))
    blocks = x.view(down, height, across, _BLOCK)
    largest = blocks.abs().amax((1, 3), keepdim=True)
    # (a tensor of 448: torch multiplies by the reciprocal of a Python number, and ties between codes hang on the last bit)
    scale = largest.clamp_min(2.0 ** -80) / torch.full_like(largest, 448)
    if pow2:
        mantissa, exponent = torch.frexp(scale)
        scale = torch.ldexp(torch.ones_like(scale), exponent - (mantissa == 0.5).int())
    scale = torch.where(largest.isfinite(), scale, math.nan)
    codes = (blocks / scale).to(torch.float8_e4m3fn).view(down * height, across * _BLOCK)[:rows, :cols]
    return codes, scale.view(down, across)


def _plain_values(codes, scale, height):
    wide = scale.repeat_interleave(height, 0)[:codes.shape[0]].repeat_interleave(_BLOCK, 1)[:, :codes.shape[1]]
    return codes.float() * wide


def _plain_rows8(case, s):
    x = s["x"]
    if case["source"] == "dispatch":
        x = x[s["slots"] // case["top_k"]]
    elif case["source"] == "swiglu":
        gate, up = x.float().chunk(2, dim=1)
        x = gate / (1 + torch.exp(-gate)) * up
    return _plain_values(*_plain_blocks(x, 1, case["pow2"]), 1).to(s["x"].dtype)


def _plain_block8(case, s):
    x, trans, train, pow2 = s["x"], case["trans_rhs"], case["train"], case["pow2"]
    dtype, m, k, n = _TYPES[case["dtype"]], case["m"], case["k"], case["n"]
    xv = _plain_values(*(x if case["held"] else _plain_blocks(x, 1, pow2)), 1)
    y = torch.zeros((m, n), dtype=dtype, device=xv.device)
    if train:
        dout = s["dout"].float()
        dv = _plain_values(*_plain_blocks(dout, 1, pow2), 1)
        dx, dA = torch.zeros((m, k), dtype=dtype, device=xv.device), torch.zeros_like(s["A"])
    row = 0
    for e, size in enumerate(s["sizes"].tolist()):
        if not size:
            continue
        at = slice(row, row + size)
        w = _plain_values(*(_plain_blocks(s["A"][e], _BLOCK, pow2) if train else (s["codes"][e], s["scales"][e])), _BLOCK)
        y[at] = (xv[at] @ (w.t() if trans else w)).to(dtype)
        if train:
            dx[at] = (dv[at] @ (w if trans else w.t())).to(dtype)
            xt = x.detach()[at].float()
            dA[e] = (dout[at].t() @ xt if trans else xt.t() @ dout[at]).to(dtype)
        row += size
    return (y, dx, dA) if train else y


def _plain_ortho(case, s):
    G, (a, b, c) = s["G"], _COEFFICIENTS
    out = torch.empty_like(G)
    for e in range(len(G)):
        X = G[e].float()
        X = X / (G[e].double().square().sum().sqrt() + 1e-7).float()
        tall = X.shape[0] > X.shape[1]
        if tall:
            X = X.t().contiguous()
        for _ in range(5):
            gram = X @ X.t()
            X = a * X + (b * gram + c * (gram @ gram)) @ X
        out[e] = X.t() if tall else X
    return out


_run_plain = {"rows8": _plain_rows8, "block8": _plain_block8, "ortho": _plain_ortho}
_run_own = {"rows8": _own_rows8, "block8": _own_block8, "ortho": _own_ortho}


# ---- from the definitions, in 64 bits ------------------------------------------------------------------------------------
def _exact_values(x, down, pow2):
    """What x [rows, cols] stands for once each block of ``down`` x 128 is held as multiples of a scale in e4m3: the scale is
    the block's largest magnitude over 448, a number of 24 bits, and so is the quotient that is rounded to e4m3."""
    x = x.detach().double()
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], _BLOCK):
        strip = x[:, c:c + _BLOCK]
        top = strip.abs().amax(1)
        if down > 1:
            whole = torch.nn.functional.pad(top, (0, -len(top) % down)).view(-1, down)
            top = whole.amax(1, keepdim=True).expand_as(whole).reshape(-1)[:len(x)]
        scale = (torch.clamp(top, min=2.0 ** -80) / 448).float().double()
        if pow2:
            scale = torch.exp2(torch.ceil(torch.log2(scale)))
        ratio = (strip / scale[:, None]).float().double()
        # e4m3: three bits behind the leading one down to 2^-6, multiples of 2^-9 below
        step = torch.exp2(torch.floor(torch.log2(ratio.abs().clamp_min(2.0 ** -6))) - 3)
        out[:, c:c + _BLOCK] = torch.clamp(torch.round(ratio / step) * step, -448, 448) * scale[:, None]
    return out


def _exact_rows8(case, s):
    x = s["x"].double()
    if case["source"] == "swiglu":
        x = x[:, :case["k"]] * torch.sigmoid(x[:, :case["k"]]) * x[:, case["k"]:]
    values = _exact_values(x.float() if case["source"] == "swiglu" else x, 1, case["pow2"])
    if case["source"] == "dispatch":
        tokens = torch.arange(case["rows"], device=x.device) // case["top_k"]
        order = torch.argsort(s["ids"].reshape(-1).double() * case["rows"] + torch.arange(case["rows"], device=x.device))
        values = values[tokens[order]]
    return values


def _exact_block8(case, s):
    m, k, n, pow2 = case["m"], case["k"], case["n"], case["pow2"]
    first = np.concatenate(([0], np.cumsum(s["sizes"])))
    x8 = _exact_values(s["x"], 1, pow2)
    y = torch.zeros((m, n), dtype=torch.float64, device="cuda")
    if case["train"]:
        d = s["dout"].double()
        d8 = _exact_values(d, 1, pow2)
        dx, dA = torch.zeros((m, k), dtype=torch.float64, device="cuda"), torch.zeros(s["A"].shape, dtype=torch.float64, device="cuda")
    for e in np.flatnonzero(s["sizes"]):
        rows = slice(int(first[e]), int(first[e + 1]))
        w = _exact_values(s["A"][e], _BLOCK, pow2)
        wkn = w.t().contiguous() if case["trans_rhs"] else w
        y[rows] = x8[rows] @ wkn
        if case["train"]:
            dx[rows] = d8[rows] @ wkn.t().contiguous()
            grad = s["x"][rows].double().t().contiguous() @ d[rows]
            dA[e] = grad.t() if case["trans_rhs"] else grad
    return (y, dx, dA) if case["train"] else y


def _exact_ortho(case, s):
    a, b, c = _COEFFICIENTS
    out = torch.empty(s["G"].shape, dtype=torch.float64, device="cuda")
    for e, G in enumerate(s["G"]):
        X = G.double() / (torch.linalg.vector_norm(G.double()) + 1e-7)
        wide = X.shape[0] <= X.shape[1]
        for _ in range(5):  # p(X X') X = X p(X' X), whichever is smaller
            S = X @ X.t().contiguous() if wide else X.t().contiguous() @ X
            P = c * S @ S + b * S
            P.diagonal().add_(a)
            X = P @ X if wide else X @ P
        out[e] = X
    return out


_EXACT = {"rows8": _exact_rows8, "block8": _exact_block8, "ortho": _exact_ortho}


def exact(case, seed):
    with torch.no_grad():
        return _EXACT[case["kind"]](case, _INPUTS[case["kind"]](case, seed))


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    e = _BYTES[case["dtype"]]
    if case["kind"] == "rows8":
        rows, k = case["rows"], case["k"]
        read = {"rows": rows * k, "swiglu": 2 * rows * k, "dispatch": rows // case["top_k"] * k}[case["source"]]
        return {"bytes": (read + rows * k) * e + (8 * rows if case["source"] == "dispatch" else 0), "flops": 4.0 * rows * k}
    if case["kind"] == "ortho":
        g, r, c = case["g"], min(case["k"], case["n"]), max(case["k"], case["n"])
        # a step: the two symmetric products by half, and the full one
        return {"bytes": 2 * g * r * c * e, "flops": 5.0 * g * (r * r * c + r * r * r + 2 * r * r * c)}
    m, k, n, g = case["m"], case["k"], case["n"], case["g"]
    rows = round(m * case["fill"])
    p = _shares(case["routing"], g, np.random.default_rng(0))
    live = float((1.0 - (1.0 - p) ** rows).sum())  # experts with a row at all, on average
    if case["train"]:
        return {"bytes": (live + g) * k * n * e + (2 * rows * k + 2 * m * n) * e + 4 * g, "flops": 6.0 * rows * k * n}
    row_bytes = k + 4 * -(-k // _BLOCK) if case["held"] else k * e
    return {"bytes": live * (k * n + 4 * -(-k // _BLOCK) * -(-n // _BLOCK)) + rows * row_bytes + m * n * e + 4 * g,
            "flops": 2.0 * rows * k * n}
