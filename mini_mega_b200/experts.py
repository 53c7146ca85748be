"""Tokens sorted by expert and back, as operators of their own, with gradients.

The layer (``mega.py``) keeps these steps inside its one kernel.  Here they are calls, for models that put
something of their own between them, and for training::

    plan = plan_tokens_by_expert(topk_idx, num_experts)
    rows = sort_tokens_by_expert(x, plan)                  # [tokens * topk, hidden], one expert after the other
    ...                                                    # fp8_grouped_matmul(..., plan.offsets)
    y = unsort_tokens_by_expert(rows, plan, topk_weights)  # [tokens, hidden]

Pair ``p = token * topk + j``; inside an expert the rows lie in ascending pair order (the order of the layer's own
dispatch), so a plan, and everything computed with it, is the same on every run.  Calls run on the current stream
of the tensors' device, allocate only their results and can be captured into CUDA graphs.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import check

_MAX_EXPERTS = 1024
_MAX_TOPK = 256
_DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_SORT_DTYPES = (torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.float8_e5m2, torch.uint8, torch.int8)


class ExpertPlan(NamedTuple):
    """The tables of a routing, int32 on the device.

    ``row_of_pair`` ``[tokens, topk]``: the row of every pair, -1 for a dropped one.
    ``pair_of_row`` ``[tokens * topk]``: its inverse, -1 behind the last row in use.
    ``offsets`` ``[num_experts + 1]``: expert e's rows are ``offsets[e] .. offsets[e + 1]``.

    ``plan_tokens_by_expert`` builds it; tables of one's own in the same form serve as well (an entry out of
    range counts as a dropped pair; two pairs with one row are the caller's mistake)."""
    row_of_pair: torch.Tensor
    pair_of_row: torch.Tensor
    offsets: torch.Tensor


def _launch(device: torch.device, fn, name: str, *args) -> None:
    """One call of the library on the current stream of `device`."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            check(fn(*args, torch.cuda.current_stream().cuda_stream), name)
    else:
        check(fn(*args, torch.cuda.current_stream().cuda_stream), name)


def _same_cuda_device(fn: str, *tensors: torch.Tensor) -> torch.device:
    device = tensors[0].device
    for t in tensors:
        if t.device != device:
            raise ValueError(f"{fn}: all tensors must be on one device, got {device} and {t.device}")
    if device.type != "cuda":
        raise ValueError(f"{fn} runs on CUDA tensors only, got {device}")
    return device


def plan_tokens_by_expert(topk_idx: torch.Tensor, num_experts: int, first_expert: int = 0) -> ExpertPlan:
    """The plan of a routing ``topk_idx`` (int64 or int32 ``[tokens, topk]``) over the experts
    ``first_expert .. first_expert + num_experts`` (all of them, or one rank's).  A pair with any other id (-1, for
    one) is dropped; a token may name an expert twice."""
    if not isinstance(topk_idx, torch.Tensor) or topk_idx.dtype not in (torch.int64, torch.int32):
        raise TypeError("topk_idx must be an int64 or int32 tensor")
    if topk_idx.dim() != 2 or not 1 <= topk_idx.shape[1] <= _MAX_TOPK:
        raise ValueError(f"topk_idx must be [tokens, topk] with 1 <= topk <= {_MAX_TOPK}, got {tuple(topk_idx.shape)}")
    if not 1 <= num_experts <= _MAX_EXPERTS:
        raise ValueError(f"num_experts must be in [1, {_MAX_EXPERTS}], got {num_experts}")
    if not 0 <= first_expert < 2 ** 31:
        raise ValueError(f"first_expert must be in [0, 2^31), got {first_expert}")
    tokens, topk = topk_idx.shape
    if tokens * topk > 1 << 30:
        raise ValueError(f"tokens * topk must be at most 2^30, got {tokens * topk}")
    device = _same_cuda_device("plan_tokens_by_expert", topk_idx)
    if topk > 1 and topk_idx.stride(1) != 1:
        topk_idx = topk_idx.contiguous()
    row_of_pair = torch.empty((tokens, topk), dtype=torch.int32, device=device)
    pair_of_row = torch.empty(tokens * topk, dtype=torch.int32, device=device)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=device)
    _launch(device, _lib.lib().mxk_plan_tokens, "mxk_plan_tokens", topk_idx.data_ptr(), topk_idx.element_size(),
            topk_idx.stride(0), tokens, topk, first_expert, num_experts, row_of_pair.data_ptr(), pair_of_row.data_ptr(),
            offsets.data_ptr())
    return ExpertPlan(row_of_pair, pair_of_row, offsets)


def _check_plan(fn: str, plan: ExpertPlan):
    row_of_pair, pair_of_row, offsets = plan
    for t in plan:
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
            raise TypeError(f"{fn}: the plan's tables must be int32 tensors")
        if not t.is_contiguous():
            raise ValueError(f"{fn}: the plan's tables must be contiguous")
    if row_of_pair.dim() != 2 or not 1 <= row_of_pair.shape[1] <= _MAX_TOPK or row_of_pair.numel() > 1 << 30:
        raise ValueError(f"{fn}: row_of_pair must be [tokens, topk], got {tuple(row_of_pair.shape)}")
    if pair_of_row.dim() != 1 or pair_of_row.shape[0] != row_of_pair.numel():
        raise ValueError(f"{fn}: pair_of_row must be [tokens * topk], got {tuple(pair_of_row.shape)}")
    if offsets.dim() != 1 or not 2 <= offsets.shape[0] <= _MAX_EXPERTS + 1:
        raise ValueError(f"{fn}: offsets must be [num_experts + 1], got {tuple(offsets.shape)}")
    return row_of_pair, offsets


def _row_stride(t: torch.Tensor) -> int:
    """Bytes between rows of a 2-d tensor whose rows are contiguous."""
    return t.stride(0) * t.element_size()


def _rows_contiguous(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _sort(x, x_sf, row_of_pair, offsets):
    tokens, topk = row_of_pair.shape
    x = _rows_contiguous(x)
    rows = torch.empty((tokens * topk, x.shape[1]), dtype=x.dtype, device=x.device)
    sf_args, rows_sf = (None, 0, 0), None
    if x_sf is not None:
        x_sf = _rows_contiguous(x_sf)
        rows_sf = torch.empty((tokens * topk, x_sf.shape[1]), dtype=x_sf.dtype, device=x.device)
        sf_args = (x_sf.data_ptr(), _row_stride(x_sf), x_sf.shape[1])
    _launch(x.device, _lib.lib().mxk_sort_tokens, "mxk_sort_tokens", x.data_ptr(), _row_stride(x),
            x.shape[1] * x.element_size(), *sf_args, tokens, topk, offsets.shape[0] - 1, row_of_pair.data_ptr(),
            offsets.data_ptr(), rows.data_ptr(), None if rows_sf is None else rows_sf.data_ptr())
    return rows if rows_sf is None else (rows, rows_sf)


def _unsort(rows, weights, row_of_pair):
    tokens, topk = row_of_pair.shape
    rows = _rows_contiguous(rows)
    y = torch.empty((tokens, rows.shape[1]), dtype=rows.dtype, device=rows.device)
    if weights is not None:
        weights = _rows_contiguous(weights)
    _launch(rows.device, _lib.lib().mxk_unsort_tokens, "mxk_unsort_tokens", rows.data_ptr(), _DTYPE_CODE[rows.dtype],
            _row_stride(rows), None if weights is None else weights.data_ptr(), 0 if weights is None else weights.stride(0),
            tokens, topk, rows.shape[1], row_of_pair.data_ptr(), y.data_ptr())
    return y


class _Sort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, row_of_pair, offsets):
        ctx.save_for_backward(row_of_pair)
        return _sort(x, None, row_of_pair, offsets)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, drows):
        (row_of_pair,) = ctx.saved_tensors
        return _unsort(drows, None, row_of_pair), None, None


class _Unsort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, row_of_pair, offsets):
        # rows are kept for the gradient of the weights only
        ctx.save_for_backward(rows if ctx.needs_input_grad[1] else None, weights, row_of_pair, offsets)
        return _unsort(rows, weights, row_of_pair)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        rows, weights, row_of_pair, offsets = ctx.saved_tensors
        if weights is None:
            return _sort(dy, None, row_of_pair, offsets), None, None, None
        tokens, topk = row_of_pair.shape
        dy, weights = _rows_contiguous(dy), _rows_contiguous(weights)
        drows = dweights = None
        if ctx.needs_input_grad[0]:
            drows = torch.empty((tokens * topk, dy.shape[1]), dtype=dy.dtype, device=dy.device)
        if ctx.needs_input_grad[1]:
            rows = _rows_contiguous(rows)
            dweights = torch.empty((tokens, topk), dtype=torch.float32, device=dy.device)
        _launch(dy.device, _lib.lib().mxk_unsort_tokens_grad, "mxk_unsort_tokens_grad", dy.data_ptr(), _row_stride(dy),
                None if rows is None else rows.data_ptr(), 0 if rows is None else _row_stride(rows), _DTYPE_CODE[dy.dtype],
                weights.data_ptr(), weights.stride(0), tokens, topk, offsets.shape[0] - 1, dy.shape[1],
                row_of_pair.data_ptr(), offsets.data_ptr(), None if drows is None else drows.data_ptr(),
                None if dweights is None else dweights.data_ptr())
        return drows, dweights, None, None


def _note_leaves(fn: str, out: torch.Tensor) -> None:
    """A leaf's gradient is accumulated on the stream of the leaf's first use while that use's graph lives.  When that
    was another stream than the one under capture, the captured backward pass would have to join it, which CUDA
    answers by invalidating the capture and PyTorch by ending the process; the call is refused here instead."""
    stream = torch.cuda.current_stream(out.device).cuda_stream
    capturing = torch.cuda.is_current_stream_capturing()
    for node, _ in out.grad_fn.next_functions:
        if node is not None and not node.next_functions:
            seen = node.metadata.setdefault("mxk_stream", stream)
            if capturing and seen != stream:
                raise RuntimeError(f"{fn}: a graph of an earlier call with the same leaf tensor is still alive and belongs to "
                                   "another stream; drop its outputs before the capture begins")


def sort_tokens_by_expert(x: torch.Tensor, plan: ExpertPlan, x_sf: Optional[torch.Tensor] = None):
    """The rows of ``x`` ``[tokens, hidden]`` in expert order, ``[tokens * topk, hidden]``: row
    ``plan.row_of_pair[t, j]`` is ``x[t]``.  Rows behind ``plan.offsets[-1]`` (as many as pairs were dropped) are zero.

    ``x`` is bf16, fp16 or fp32 (differentiable: the gradient of a token is the sum over its rows, in FP32), or 8-bit;
    with ``x_sf`` (uint8 ``[tokens, ...]`` scale bytes) the scales travel along and ``(rows, rows_sf)`` is returned."""
    fn = "sort_tokens_by_expert"
    row_of_pair, offsets = _check_plan(fn, plan)
    if not isinstance(x, torch.Tensor) or x.dtype not in _SORT_DTYPES:
        raise TypeError(f"{fn}: x must be a bf16, fp16, fp32 or 8-bit tensor")
    if x.dim() != 2 or x.shape[0] != row_of_pair.shape[0] or x.shape[1] < 1:
        raise ValueError(f"{fn}: x must be [{row_of_pair.shape[0]}, hidden], got {tuple(x.shape)}")
    if x_sf is None:
        _same_cuda_device(fn, x, *plan)
        if x.requires_grad and torch.is_grad_enabled():
            if x.dtype not in _DTYPE_CODE:
                raise TypeError(f"{fn}: only bf16, fp16 and fp32 rows have a gradient")
            rows = _Sort.apply(x, row_of_pair, offsets)
            _note_leaves(fn, rows)
            return rows
        return _sort(x, None, row_of_pair, offsets)
    if not isinstance(x_sf, torch.Tensor) or x_sf.dtype != torch.uint8 or x.element_size() != 1:
        raise TypeError(f"{fn}: x_sf are uint8 exponents of 8-bit rows")
    if x_sf.dim() != 2 or x_sf.shape[0] != x.shape[0] or x_sf.shape[1] < 1:
        raise ValueError(f"{fn}: x_sf must be [{x.shape[0]}, hidden / 128], got {tuple(x_sf.shape)}")
    _same_cuda_device(fn, x, x_sf, *plan)
    return _sort(x, x_sf, row_of_pair, offsets)


def unsort_tokens_by_expert(rows: torch.Tensor, plan: ExpertPlan, topk_weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The sorted rows brought back and summed per token, ``y[t] = sum_j topk_weights[t, j] *
    rows[plan.row_of_pair[t, j]]`` (j ascending, in FP32, rounded once), dropped pairs left out; without weights the
    plain sum.  ``rows`` ``[tokens * topk, hidden]`` is bf16, fp16 or fp32, ``topk_weights`` fp32 ``[tokens, topk]``.

    Differentiable in ``rows`` (rows behind ``plan.offsets[-1]`` get zeros) and in ``topk_weights`` (dropped pairs get 0)."""
    fn = "unsort_tokens_by_expert"
    row_of_pair, offsets = _check_plan(fn, plan)
    if not isinstance(rows, torch.Tensor) or rows.dtype not in _DTYPE_CODE:
        raise TypeError(f"{fn}: rows must be a bf16, fp16 or fp32 tensor")
    if rows.dim() != 2 or rows.shape[0] != row_of_pair.numel() or rows.shape[1] < 1:
        raise ValueError(f"{fn}: rows must be [{row_of_pair.numel()}, hidden], got {tuple(rows.shape)}")
    needs_grad = rows.requires_grad
    if topk_weights is not None:
        if not isinstance(topk_weights, torch.Tensor) or topk_weights.dtype != torch.float32:
            raise TypeError(f"{fn}: topk_weights must be a float32 tensor")
        if topk_weights.shape != row_of_pair.shape:
            raise ValueError(f"{fn}: topk_weights must be {tuple(row_of_pair.shape)}, got {tuple(topk_weights.shape)}")
        _same_cuda_device(fn, rows, topk_weights, *plan)
        needs_grad = needs_grad or topk_weights.requires_grad
    else:
        _same_cuda_device(fn, rows, *plan)
    if needs_grad and torch.is_grad_enabled():
        y = _Unsort.apply(rows, topk_weights, row_of_pair, offsets)
        _note_leaves(fn, y)
        return y
    return _unsort(rows, topk_weights, row_of_pair)
