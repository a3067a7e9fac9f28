"""``ragged_dot`` on weights held as 4-bit integers: an expert's matrix is ``scale * (q - zero)``, q in 0 .. 15, with one scale
(and one zero point) per ``block`` contraction indices of every output column.

    weights = pack_int4(q, scales, zeros, block=128)       # once, when a checkpoint is loaded
    y = ragged_dot_int4(x, weights, group_sizes)           # as ragged_dot(x, A, group_sizes)

Forward products of bfloat16 and float16 rows, for serving; the reference has no counterpart.  The kernels are behind
``rd_int4_pack`` and ``rd_gmm_int4`` of the C ABI (``include/ragged_dot_hip.h``), the host side in ``csrc/rd_torch.cpp``.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _capi, _tracing
from ._native import lib as _native
from .ops import _group_offset, _sizes

__all__ = ["Int4Weights", "pack_int4", "ragged_dot_int4"]


class Int4Weights(NamedTuple):
    codes: torch.Tensor            # int32 [g, ceil(n / 16), ceil(k / 128), 64, 4]  eight codes to a word, in the kernels' order
    scales: torch.Tensor           # [g, ceil(k / 128), n, 128 / block]  bfloat16 or float16
    zeros: Optional[torch.Tensor]  # uint8, the scales' shape; None = 8
    k: int
    n: int
    block: int


def pack_int4(q: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, *, block: int = 128,
              trans_rhs: bool = False) -> Int4Weights:
    """Lays out codes ``q`` (uint8, one of 0 .. 15 per byte) ``[g, k, n]`` with ``scales`` (and ``zeros``)
    ``[g, ceil(k / block), n]``; with ``trans_rhs`` ``[g, n, k]`` and ``[g, n, ceil(k / block)]``, as most checkpoints hold
    them.  ``block`` is 32, 64 or 128, scales are bfloat16 or float16.  Codes above 15 lose their upper bits."""
    assert q.ndim == 3, f"but {q.ndim=}"
    assert block in (32, 64, 128), f"block is 32, 64 or 128, not {block}"
    g, k, n = (q.shape[0], q.shape[2], q.shape[1]) if trans_rhs else q.shape
    if zeros is not None and zeros.dtype != torch.uint8:
        raise TypeError(f"zeros are uint8, not {zeros.dtype}")
    blocks = -(-k // block)
    wanted = (g, n, blocks) if trans_rhs else (g, blocks, n)
    for name, t in (("scales", scales), ("zeros", zeros)):
        if t is not None and tuple(t.shape) != wanted:
            raise ValueError(f"{name} must be {list(wanted)}, not {list(t.shape)}")
    if scales.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"unsupported dtype {scales.dtype}; scales are bfloat16 or float16")
    runs, per_run = -(-k // 128), 128 // block

    def laid_out(t):  # a run's scales of a column beside each other, zeros past k
        if t is None:
            return None
        out = t.new_zeros((g, n, runs * per_run))
        out[:, :, :blocks] = t.detach() if trans_rhs else t.detach().transpose(1, 2)
        return out.view(g, n, runs, per_run).transpose(1, 2).contiguous()

    return Int4Weights(_native.int4_pack(q, bool(trans_rhs)), laid_out(scales), laid_out(zeros), k, n, int(block))


def ragged_dot_int4(x: torch.Tensor, weights: Int4Weights, group_sizes, *, group_offset=None, exact_weights: bool = False) -> torch.Tensor:
    """``(m, k) x (g, k, n) -> (m, n)`` on 4-bit weights; rows past ``sum(group_sizes)`` are zero.  ``x`` is bfloat16 or float16,
    and so is the result, rounded once from fp32.  Where the sizes of the call make it cheaper, groups of more than 48 rows multiply
    weights that are rounded to that type, too; with ``exact_weights`` none do, which takes up to twice as long for long prompts.
    ``group_offset`` as in ``gmm``: ``weights`` hold the groups from there on, the rows of the others are zero.  No gradient: an
    ``x`` that requires one raises ``NotImplementedError``."""
    return _ragged_dot_int4(x, weights, group_sizes, group_offset, _capi.RD_INT4_STREAM if exact_weights else _capi.RD_INT4_AUTO)


def _ragged_dot_int4(x, weights, group_sizes, group_offset=None, kernel=_capi.RD_INT4_AUTO):
    """With the choice of the kernel (``rd_int4_kernel`` in the header)."""
    assert x.ndim == 2, f"but {x.ndim=}"
    g_first = -1 if group_offset is None else _group_offset(group_offset)
    assert group_offset is None or g_first >= 0
    call = lambda x, gs: _native.gmm_int4(x, weights.codes, weights.scales, weights.zeros, weights.k, weights.n, weights.block, gs, g_first,
                                          kernel)
    if _tracing.active():
        # (a trace's node does not know whether its caller wants gradients: it refuses in the backward pass, and not where x asks for
        # one under torch.no_grad())
        return _tracing.record(lambda x, gs: call(x.detach(), gs), x, _sizes(group_sizes))
    return call(x, _sizes(group_sizes))
