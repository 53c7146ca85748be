"""Tokens sorted by expert and back, as operators of their own, with gradients.

The layer (``mega.py``) keeps these steps inside its one kernel.  Here they are calls, for models that put
something of their own between them, and for training::

    plan = plan_tokens_by_expert(topk_idx, num_experts)
    rows = sort_tokens_by_expert(x, plan)                  # [tokens * topk, hidden], one expert after the other
    ...                                                    # fp8_grouped_matmul(..., plan.offsets)
    y = unsort_tokens_by_expert(rows, plan, topk_weights)  # [tokens, hidden]

Pair ``p = token * topk + j``; inside an expert the rows lie in ascending pair order (the order of the layer's own
dispatch), so a plan, and everything computed with it, is the same on every run.  Calls run on the current stream
of the tensors' device, allocate only their results and can be captured into CUDA graphs.  There is no forward-mode
derivative: inputs with a tangent are refused, and so are calls under a tracer (``torch.jit.trace``, ``make_fx``).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib


class ExpertPlan(NamedTuple):
    """The tables of a routing, int32 on the device.

    ``row_of_pair`` ``[tokens, topk]``: the row of every pair, -1 for a dropped one.
    ``pair_of_row`` ``[tokens * topk]``: its inverse, -1 behind the last row in use.
    ``offsets`` ``[num_experts + 1]``: expert e's rows are ``offsets[e] .. offsets[e + 1]``.

    ``plan_tokens_by_expert`` builds it; tables of one's own in the same form serve as well.  An entry of
    ``row_of_pair`` out of range counts as a dropped pair, also one that had a row when the plan was made: that row, which no
    pair names any more, is zero in sorted rows and in gradients.  (Two pairs with one row, or a ``pair_of_row`` that is not the
    inverse of what is kept, are the caller's mistake.)"""
    row_of_pair: torch.Tensor
    pair_of_row: torch.Tensor
    offsets: torch.Tensor


def plan_tokens_by_expert(topk_idx: torch.Tensor, num_experts: int, first_expert: int = 0) -> ExpertPlan:
    """The plan of a routing ``topk_idx`` (int64 or int32 ``[tokens, topk]``) over the experts
    ``first_expert .. first_expert + num_experts`` (all of them, or one rank's).  A pair with any other id (-1, for
    one) is dropped; a token may name an expert twice."""
    return ExpertPlan(*_lib.ops().plan_tokens(topk_idx, num_experts, first_expert))


def sort_tokens_by_expert(x: torch.Tensor, plan: ExpertPlan, x_sf: Optional[torch.Tensor] = None):
    """The rows of ``x`` ``[tokens, hidden]`` in expert order, ``[tokens * topk, hidden]``: row
    ``plan.row_of_pair[t, j]`` is ``x[t]``.  Rows that no pair names (those behind ``plan.offsets[-1]``, as many as pairs were
    dropped) are zero.

    ``x`` is bf16, fp16 or fp32 (differentiable: the gradient of a token is the sum over its rows, in FP32), or 8-bit;
    with ``x_sf`` (uint8 ``[tokens, ...]`` scale bytes) the scales travel along and ``(rows, rows_sf)`` is returned."""
    return _lib.ops().sort_tokens(x, *plan, x_sf)


def unsort_tokens_by_expert(rows: torch.Tensor, plan: ExpertPlan, topk_weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The sorted rows brought back and summed per token, ``y[t] = sum_j topk_weights[t, j] *
    rows[plan.row_of_pair[t, j]]`` (j ascending, in FP32, rounded once), dropped pairs left out; without weights the
    plain sum.  ``rows`` ``[tokens * topk, hidden]`` is bf16, fp16 or fp32, ``topk_weights`` fp32 ``[tokens, topk]``.

    Differentiable in ``rows`` (rows that no pair names get zeros) and in ``topk_weights`` (dropped pairs get 0);
    a second time only without weights."""
    return _lib.ops().unsort_tokens(rows, *plan, topk_weights)
