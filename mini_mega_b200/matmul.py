"""8-bit products with block scales, as operators of their own.

Operands are ``(data, sf)`` pairs in the formats of ``quant.py``: E4M3 (or E5M2) bytes and UE8M0 exponent bytes, one
per 128 columns of a row of ``x`` and one per 128 x 128 block of a weight; a raw tensor stands for scales of one.
They serve what lies beside the layer: a dense expert that every token visits, projections, and, with
``sort_tokens_by_expert`` before and ``unsort_tokens_by_expert`` behind, the experts themselves.
"""
from __future__ import annotations

import struct
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .experts import _launch, _same_cuda_device

Operand = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]

_FORMAT = {torch.float8_e4m3fn: 0, torch.uint8: 0, torch.float8_e5m2: 1}
# MxkMatmulArgs of include/mxk_b200.h: six pointers, four strides, nine 32-bit fields, padding
_ARGS = struct.Struct("@6P4q9i4x")


def _operand(fn: str, name: str, w: Operand, dim: int):
    data, sf = w if isinstance(w, tuple) else (w, None)
    if not isinstance(data, torch.Tensor) or data.dtype not in _FORMAT:
        raise TypeError(f"{fn}: {name} must be a float8_e4m3fn, float8_e5m2 (or raw uint8 E4M3) tensor")
    if data.dim() != dim:
        raise ValueError(f"{fn}: {name} must have {dim} dimensions, got {tuple(data.shape)}")
    if sf is not None and (not isinstance(sf, torch.Tensor) or sf.dtype != torch.uint8):
        raise TypeError(f"{fn}: {name} scales must be uint8 exponents")
    return data, sf


def _matmul(fn: str, x: Operand, w: Operand, offsets: Optional[torch.Tensor], out: Optional[torch.Tensor]) -> torch.Tensor:
    xd, xs = _operand(fn, "x", x, 2)
    wd, ws = _operand(fn, "w", w, 2 if offsets is None else 3)
    rows, depth = xd.shape
    cols = wd.shape[-2]
    experts = 1 if offsets is None else wd.shape[0]
    blocks = (depth + 127) // 128
    if wd.shape[-1] != depth:
        raise ValueError(f"{fn}: x has {depth} columns, w {wd.shape[-1]}")
    if depth < 16 or depth % 16 or cols < 1 or not 1 <= experts <= 1024:
        raise ValueError(f"{fn}: needs a depth that is a multiple of 16, at least one weight row and 1 to 1024 experts, got "
                         f"x {tuple(xd.shape)} and w {tuple(wd.shape)}")
    if rows > 1 << 30 or depth > 1 << 30 or experts * cols > 1 << 30:
        raise ValueError(f"{fn}: more than 2^30 rows")
    tensors = [t for t in (xd, xs, wd, ws, offsets, out) if t is not None]
    if xs is not None and (tuple(xs.shape) != (rows, blocks) or (xs.stride(1) != 1 and blocks > 1)):
        raise ValueError(f"{fn}: x scales must be [{rows}, {blocks}] with contiguous rows, got {tuple(xs.shape)}")
    per_row = 0
    if ws is not None:
        lead = () if offsets is None else (experts,)
        if tuple(ws.shape) == lead + ((cols + 127) // 128, blocks):
            per_row = 0
        elif tuple(ws.shape) == lead + (cols, blocks):
            per_row = 1
        else:
            raise ValueError(f"{fn}: w scales must be {lead + ((cols + 127) // 128, blocks)} (128 x 128 blocks) or "
                             f"{lead + (cols, blocks)} (per row), got {tuple(ws.shape)}")
        if not ws.is_contiguous():
            raise ValueError(f"{fn}: w scales must be contiguous")
    if xd.stride(1) != 1 or (rows > 1 and (xd.stride(0) < depth or xd.stride(0) % 16)) or xd.data_ptr() % 16:
        raise ValueError(f"{fn}: x needs contiguous rows, 16-byte aligned and not overlapping")
    w_stride = wd.stride(-2) if cols > 1 else depth
    if wd.stride(-1) != 1 or w_stride < depth or w_stride % 16 or wd.data_ptr() % 16 or \
            (experts > 1 and wd.stride(0) != cols * w_stride):
        raise ValueError(f"{fn}: w needs contiguous rows, 16-byte aligned, and the experts' matrices one behind the other")
    zero_tail = 0
    if offsets is not None:
        if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.shape[0] != experts + 1 or not offsets.is_contiguous():
            raise ValueError(f"{fn}: offsets must be a contiguous int32 tensor of {experts + 1} entries")
    device = _same_cuda_device(fn, *tensors)
    if out is None:
        out = torch.empty((rows, cols), dtype=torch.bfloat16, device=device)
        zero_tail = 1
    elif out.dtype != torch.bfloat16 or tuple(out.shape) != (rows, cols) or (cols > 1 and out.stride(1) != 1) or \
            (rows > 1 and out.stride(0) < cols):
        raise ValueError(f"{fn}: out must be a bf16 [{rows}, {cols}] tensor with contiguous rows")
    if rows == 0:
        return out
    args = _ARGS.pack(xd.data_ptr(), 0 if xs is None else xs.data_ptr(), wd.data_ptr(), 0 if ws is None else ws.data_ptr(),
                      out.data_ptr(), 0 if offsets is None else offsets.data_ptr(),
                      xd.stride(0) if rows > 1 else depth, 0 if xs is None else xs.stride(0), w_stride, out.stride(0),
                      rows, cols, depth, experts, _FORMAT[xd.dtype], _FORMAT[wd.dtype], per_row, zero_tail, 0)
    _launch(device, _lib.lib().mxk_fp8_matmul, "mxk_fp8_matmul", args)
    return out


def fp8_matmul(x: Operand, w: Operand, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w.T`` in bf16, accumulated in FP32: ``x`` ``[rows, depth]`` with scales ``[rows, ceil(depth / 128)]``,
    ``w`` ``[cols, depth]`` with scales ``[ceil(cols / 128), ceil(depth / 128)]`` (128 x 128 blocks) or
    ``[cols, ceil(depth / 128)]`` (per row: the form in which both factors are activations, such as a weight gradient
    from its two factors quantised along the tokens).  ``depth`` is a multiple of 16; rows of both operands are 16-byte
    aligned and may be apart.  Scale byte e stands for ``2**(e - 127)``; 255 is NaN.  The operands carry no gradient."""
    return _matmul("fp8_matmul", x, w, None, out)


def fp8_grouped_matmul(x: Operand, w: Operand, offsets: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows ``offsets[e] .. offsets[e + 1]`` of ``x`` times ``w[e].T``: ``w`` ``[experts, cols, depth]`` with scales
    ``[experts, ceil(cols / 128), ceil(depth / 128)]`` (or per row), ``offsets`` int32 on the device, as in
    ``ExpertPlan.offsets``; otherwise as ``fp8_matmul``.  The host never reads the offsets.  They ascend; what they hold
    beyond that or out of range is clamped.  Rows that belong to no expert (before ``offsets[0]``, behind the last
    one) are zero in a result allocated here and left as they were in a given ``out``."""
    if not isinstance(offsets, torch.Tensor):
        raise TypeError("fp8_grouped_matmul: offsets must be an int32 tensor")
    return _matmul("fp8_grouped_matmul", x, w, offsets, out)


def matmul_status() -> int:
    """0, or the device code of the first product on the current device whose bounded wait expired (its output is then
    undefined).  Waits for the device."""
    import ctypes
    v = ctypes.c_int32()
    _lib.check(_lib.lib().mxk_matmul_status(ctypes.byref(v)), "mxk_matmul_status")
    return v.value
