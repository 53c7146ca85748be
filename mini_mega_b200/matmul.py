"""8-bit products with block scales, as operators of their own.

Operands are ``(data, sf)`` pairs in the formats of ``quant.py``: E4M3 (or E5M2) bytes and UE8M0 exponent bytes, one
per 128 columns of a row of ``x`` and one per 128 x 128 block of a weight; a raw tensor stands for scales of one.
They serve what lies beside the layer: a dense expert that every token visits, projections, and, with
``sort_tokens_by_expert`` before and ``unsort_tokens_by_expert`` behind, the experts themselves.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple, Union

import torch

from . import _lib

Operand = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]


def fp8_matmul(x: Operand, w: Operand, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w.T`` in bf16, accumulated in FP32: ``x`` ``[rows, depth]`` with scales ``[rows, ceil(depth / 128)]``,
    ``w`` ``[cols, depth]`` with scales ``[ceil(cols / 128), ceil(depth / 128)]`` (128 x 128 blocks) or
    ``[cols, ceil(depth / 128)]`` (per row: the form in which both factors are activations, such as a weight gradient
    from its two factors quantised along the tokens).  ``depth`` is a multiple of 16; rows of both operands are 16-byte
    aligned and may be apart.  Scale byte e stands for ``2**(e - 127)``; 255 is NaN.  There is no
    gradient: operands that ask for one are refused while gradients are recorded, operands with a forward-mode tangent and
    calls under a tracer (``torch.jit.trace``, ``make_fx``) always."""
    xd, xs = x if isinstance(x, tuple) else (x, None)
    wd, ws = w if isinstance(w, tuple) else (w, None)
    return _lib.ops().fp8_matmul(xd, xs, wd, ws, out)


def fp8_grouped_matmul(x: Operand, w: Operand, offsets: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows ``offsets[e] .. offsets[e + 1]`` of ``x`` times ``w[e].T``: ``w`` ``[experts, cols, depth]`` with scales
    ``[experts, ceil(cols / 128), ceil(depth / 128)]`` (or per row), ``offsets`` int32 on the device, as in
    ``ExpertPlan.offsets``; otherwise as ``fp8_matmul``.  The host never reads the offsets.  They ascend; what they hold
    beyond that or out of range is clamped.  Rows that belong to no expert (before ``offsets[0]``, behind the last
    one) are zero in a result allocated here and left as they were in a given ``out``."""
    xd, xs = x if isinstance(x, tuple) else (x, None)
    wd, ws = w if isinstance(w, tuple) else (w, None)
    return _lib.ops().fp8_grouped_matmul(xd, xs, wd, ws, offsets, out)


def matmul_status() -> int:
    """0, or the device code of the first product on the current device whose bounded wait expired (its output is then
    undefined).  Waits for the device."""
    v = C.c_int32()
    _lib.check(_lib.lib().mxk_matmul_status(C.byref(v)), "mxk_matmul_status")
    return v.value
