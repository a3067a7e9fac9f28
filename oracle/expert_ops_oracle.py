"""Plain restatements in float64 of the operators around the ragged products of a mixture of experts: the gate, the gated
activation, and products on 4-bit weights.  Used by tests only; the reference has no counterpart."""

from __future__ import annotations

import numpy as np


def _leading(values, count):
    """Indices of the ``count`` largest values, falling, ties to the lower index; shut ones (-inf) and beyond: -1."""
    order = np.argsort(-values, kind="stable")[:count]
    return [int(i) if values[i] > -np.inf else -1 for i in order]


def gate(logits, top_k, *, score="softmax", bias=None, clusters=1, top_clusters=None, cluster_score="max", renormalize=True,
         scale=1.0):
    """(expert_ids, weights) for finite or -inf logits [tokens, experts]."""
    logits = np.asarray(logits, np.float64)
    tokens, experts = logits.shape
    top_clusters = clusters if top_clusters is None else top_clusters
    ids = np.full((tokens, top_k), -1, np.int32)
    weights = np.zeros((tokens, top_k))
    for t in range(tokens):
        row = logits[t]
        s = scores(row, score)
        by_logit = bias is None and (clusters == 1 or cluster_score == "max")
        rank = row.copy() if by_logit else s + (0.0 if bias is None else np.asarray(bias, np.float64))
        rank[row == -np.inf] = -np.inf
        if clusters > 1:
            size = experts // clusters
            best = []
            for c in range(clusters):
                inside = np.sort(rank[c * size:(c + 1) * size])[::-1]
                best.append(inside[0] if cluster_score == "max" else inside[:2].sum())
            kept = np.argsort(-np.array(best), kind="stable")[:top_clusters]
            for c in range(clusters):
                if c not in kept:
                    rank[c * size:(c + 1) * size] = -np.inf
        ids[t] = _leading(rank, top_k)
        live = ids[t] >= 0
        w = np.where(live, s[ids[t]], 0.0)
        if renormalize and w.sum() > 0:
            w = w / w.sum()
        weights[t] = scale * w
    return ids, weights


def scores(row, score):
    if score == "sigmoid":
        return 1.0 / (1.0 + np.exp(-row))
    if np.all(row == -np.inf):
        return np.zeros_like(row)
    e = np.exp(row - row.max())
    return e / e.sum()


def gate_grad(logits, ids, dweights, *, score="softmax", renormalize=True, scale=1.0):
    """The gradient of the logits, by the chain rule through every score's own derivative."""
    logits = np.asarray(logits, np.float64)
    out = np.zeros_like(logits)
    for t in range(logits.shape[0]):
        s, live = scores(logits[t], score), ids[t] >= 0
        chosen, dw = s[ids[t][live]], np.asarray(dweights[t], np.float64)[live]
        if renormalize and chosen.sum() > 0:
            total = chosen.sum()
            dchosen = scale * (dw / total - (dw * chosen).sum() / total ** 2)
        else:
            dchosen = scale * dw
        ds = np.zeros_like(s)
        ds[ids[t][live]] = dchosen
        out[t] = ds * s * (1 - s) if score == "sigmoid" else s * (ds - (ds * s).sum())
    return out


def swiglu(y):
    y = np.asarray(y, np.float64)
    f = y.shape[1] // 2
    gate_half, up = y[:, :f], y[:, f:]
    return gate_half / (1 + np.exp(-gate_half)) * up


def swiglu_grad(y, dout):
    y, dout = np.asarray(y, np.float64), np.asarray(dout, np.float64)
    f = y.shape[1] // 2
    gate_half, up = y[:, :f], y[:, f:]
    sig = 1 / (1 + np.exp(-gate_half))
    return np.concatenate([dout * up * (sig + gate_half * sig * (1 - sig)), dout * gate_half * sig], 1)


def int4_dense(q, scales, zeros, block):
    """A [g, k, n] from codes [g, k, n] and scales (zeros) [g, ceil(k / block), n]."""
    at = np.arange(q.shape[1]) // block
    z = 8.0 if zeros is None else np.asarray(zeros, np.float64)[:, at]
    return (np.asarray(q, np.float64) - z) * np.asarray(scales, np.float64)[:, at]
