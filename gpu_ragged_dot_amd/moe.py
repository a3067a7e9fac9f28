"""Token routing around ``ragged_dot`` for a mixture of experts, on the device.

``ragged_dot`` takes rows sorted by group; the reference leaves producing them to its caller (its tests build sorted
rows directly, tests.py:51-71).  This module is that caller's side, each function one call across the C ABI
(``rd_moe_*`` in ``include/ragged_dot_hip.h``):

    expert_ids, weights = gate(h @ w_router, top_k)         # the router's choice
    routing = route(expert_ids, num_groups)                 # group_sizes, row_of_slot, slot_of_row
    x = dispatch(h, routing)                                # [tokens * top_k, d], rows sorted by expert
    y = ragged_dot(x, W_in, routing.group_sizes)            # the op itself, [tokens * top_k, 2 f]
    y = ragged_dot(swiglu(y), W_out, routing.group_sizes)   # [tokens * top_k, n]
    out = combine(y, routing, weights)                      # [tokens, n]

``gate`` (by its weights), ``dispatch``, ``swiglu`` and ``combine`` are differentiable (the backward of ``dispatch`` and of
``combine`` is the other one's kernel; the gradient of the combine weights is ``rd_moe_combine_wgrad``).  torch supplies device memory, the stream and the autograd engine; the host side of
each call is native (``csrc/rd_torch.cpp``).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _tracing
from ._native import lib as _native
from .float8 import Float8Rows

__all__ = ["Gating", "Routing", "gate", "route", "dispatch", "swiglu", "combine"]


class Routing(NamedTuple):
    group_sizes: torch.Tensor   # int32 [g]      rows per expert
    row_of_slot: torch.Tensor   # int32 [tokens * top_k]  row of the sorted matrix each (token, choice) went to, -1 = dropped
    slot_of_row: torch.Tensor   # int32 [tokens * top_k]  inverse; -1 for rows past sum(group_sizes)
    tokens: int
    top_k: int


class Gating(NamedTuple):
    expert_ids: torch.Tensor    # int32 [tokens, top_k]    for ``route``; -1 = no expert
    weights: torch.Tensor       # float32 [tokens, top_k]  for ``combine``; 0 where there is no expert


_gating = tuple.__new__                         # Gating(*results) without its keyword arguments' 0.2 us

_SCORES = {"softmax": 0, "sigmoid": 1}         # RD_GATE_SIGMOID
_CLUSTER_SCORES = {"max": 0, "top2": 2}        # RD_GATE_TOP2
_RENORMALIZE = 4                               # RD_GATE_RENORMALIZE


def gate(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None, clusters: int = 1,
         top_clusters: Optional[int] = None, cluster_score: str = "max", renormalize: bool = True, scale: float = 1.0) -> Gating:
    """The ``top_k`` experts of every token and their weights, from a router's logits ``[tokens, experts]``.

    Scores are the ``softmax`` or the ``sigmoid`` of the logits.  Experts rank by score plus ``bias`` ([experts], a correction
    that balances the load; it moves the choice and not the weights), ties to the lower index.  With ``clusters`` > 1 only the
    ``top_clusters`` best runs of experts / clusters neighbours stand for choice, judged by their largest rank (``"max"``) or by
    the sum of the two largest (``"top2"``).  Weights are the chosen scores, divided by their sum with ``renormalize``, times
    ``scale``.  An expert with a logit or a bias of -inf is never chosen; where that leaves fewer than ``top_k``, ids are -1
    and weights 0, which ``route`` and ``combine`` take as dropped.  Differentiable: weights by logits."""
    if score not in _SCORES:
        raise ValueError(f"score is one of {sorted(_SCORES)}, not {score!r}")
    if cluster_score not in _CLUSTER_SCORES:
        raise ValueError(f"cluster_score is one of {sorted(_CLUSTER_SCORES)}, not {cluster_score!r}")
    flags = _SCORES[score] | _CLUSTER_SCORES[cluster_score] | (_RENORMALIZE if renormalize else 0)
    spec = (top_k, clusters, clusters if top_clusters is None else top_clusters, flags, scale)
    if _tracing.active():
        return Gating(*_tracing.record(lambda l, *b: _native.moe_gate(l, b[0] if b else None, *spec), logits,
                                       *(() if bias is None else (bias.detach(),))))  # (no gradient: it moves the choice alone)
    return _gating(Gating, _native.moe_gate(logits, bias, *spec))


def route(expert_ids: torch.Tensor, num_groups: int) -> Routing:
    """Stable counting sort of the (token, choice) pairs by expert id.  ``expert_ids`` is integer ``[tokens, top_k]``;
    ids outside ``[0, num_groups)`` mark dropped pairs."""
    if _tracing.active():
        outs = _tracing.record(lambda ids: _native.moe_route(ids, num_groups), expert_ids)
        return Routing(*outs, *map(int, expert_ids.shape))
    group_sizes, row_of_slot, slot_of_row = _native.moe_route(expert_ids, num_groups)
    return Routing(group_sizes, row_of_slot, slot_of_row, *expert_ids.shape)


def _dispatch(h, r: Routing, row_scale):
    """The kernel alone (no autograd node); ``row_scale``: a float32 factor per slot, or None."""
    return _native.moe_dispatch_rows(h, row_scale, r.row_of_slot, r.slot_of_row, r.tokens, r.top_k)


def _combine(y, r: Routing, weights):
    """The kernel alone (no autograd node)."""
    with torch.no_grad():
        return _native.moe_combine(y, weights, r.row_of_slot, r.slot_of_row, r.tokens, r.top_k)


def dispatch(h: torch.Tensor, routing: Routing, *, float8: bool = False, pow2: bool = False):
    """``x[row] = h[token of row]``: ``[tokens, d] -> [tokens * top_k, d]`` sorted by expert; rows past
    ``sum(group_sizes)`` are zero.  With ``float8`` the rows are held as ``quantize_rows(..., pow2=pow2)`` holds them, a token's
    quantised once for all its rows, for ``ragged_dot_float8``; no gradient."""
    if float8:
        call = lambda h, rows, slots: _native.moe_dispatch_float8(h, rows, slots, routing.tokens, routing.top_k, pow2)
        if _tracing.active():
            held = _tracing.record(lambda h, *r: call(h.detach(), *r), h, routing.row_of_slot, routing.slot_of_row)
            return Float8Rows(*held, int(h.shape[1]))
        return Float8Rows(*call(h, routing.row_of_slot, routing.slot_of_row), h.shape[1])
    if _tracing.active():
        return _tracing.record(lambda *t: dispatch(t[0], routing._replace(row_of_slot=t[1], slot_of_row=t[2])),
                               h, routing.row_of_slot, routing.slot_of_row)
    return _native.moe_dispatch(h, routing.row_of_slot, routing.slot_of_row, routing.tokens, routing.top_k)


def swiglu(y: torch.Tensor, *, float8: bool = False, pow2: bool = False):
    """``silu(gate) * up`` of rows ``[gate | up]``: ``[rows, 2 f] -> [rows, f]``, in fp32 and rounded once.  With ``float8`` the
    result is held as ``quantize_rows(..., pow2=pow2)`` would hold the fp32 values, for ``ragged_dot_float8``; no gradient."""
    if float8:
        if _tracing.active():
            return Float8Rows(*_tracing.record(lambda y: _native.moe_swiglu_float8(y.detach(), pow2), y), int(y.shape[1]) // 2)
        return Float8Rows(*_native.moe_swiglu_float8(y, pow2), y.shape[1] // 2)
    if _tracing.active():
        return _tracing.record(_native.moe_swiglu, y)
    return _native.moe_swiglu(y)


def combine(y: torch.Tensor, routing: Routing, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[token] = sum_choice weights[token, choice] * y[row of (token, choice)]`` with fp32 accumulation;
    ``weights`` is ``[tokens, top_k]`` (None = 1)."""
    if _tracing.active():
        return _tracing.record(lambda *t: combine(t[0], routing._replace(row_of_slot=t[1], slot_of_row=t[2]), *t[3:]),
                               y, routing.row_of_slot, routing.slot_of_row, *(() if weights is None else (weights,)))
    return _native.moe_combine(y, weights, routing.row_of_slot, routing.slot_of_row, routing.tokens, routing.top_k)
