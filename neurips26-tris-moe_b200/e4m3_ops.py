"""Products in 8 bits: rows and weights in e4m3 with a scale for each 128 columns of a row and each block of 128 x 128 weights.

The reference leaves dense projections to PyTorch in fp16 (``nn.Linear`` of its model files, modeling_olmoe.py:300-618).
``add_rms_norm_e4m3(..., group_size=128)`` or ``quantize_e4m3`` makes the rows, ``quantize_e4m3(weight, group_rows=128)`` the weights, once, and
``linear_e4m3`` multiplies them.  Like the operators of ``decode_ops`` these run on the current stream, never synchronise, can be captured
in a CUDA graph, and have neither a CPU path nor a backward pass.
"""
from __future__ import annotations

import struct
from typing import Optional

import torch

from .decode_ops import _DTYPES, _LOGIT_TYPES, _ROWS, _fail, _launch, _matrix, _same_device

GROUP = 128  # columns of a scale
_E4M3 = torch.float8_e4m3fn
_QUANTIZE = struct.Struct("@3Q3q4i")
_LINEAR = struct.Struct("@7Q5q6i")


def _rows(what: str, name: str, t: torch.Tensor) -> torch.Tensor:
    """``[..., columns]`` as a matrix whose rows lie side by side in themselves."""
    if t.dim() == 0:
        _fail(what, f"{name} must be [..., columns]")
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.numel() else t.new_empty((t.shape[:-1].numel(), t.shape[-1]))
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def quantize_e4m3(x: torch.Tensor, *, group_rows: int = 1):
    """``x`` [..., columns] in fp16 or bf16 as ``(values, scales)`` with ``x = values * scales``: values in ``torch.float8_e4m3fn``, a scale (fp32, the largest
    magnitude / 448) for each 128 columns of a row - scales [..., ceil(columns / 128)] - or, ``group_rows=128``, of 128 rows of a matrix: weights, scales
    [ceil(rows / 128), ceil(columns / 128)].  The last groups may be smaller.  Rows of values start on 16-byte boundaries, as ``linear_e4m3`` wants them."""
    what = "quantize_e4m3"
    _same_device(what, x)
    dtype, x2 = x.dtype, x
    if dtype not in _ROWS:
        _fail(what, "x must be fp16 or bf16")
    if group_rows != 1 and (group_rows != GROUP or x.dim() != 2):
        _fail(what, f"a scale is for 1 row, or for {GROUP} of a matrix, not {group_rows} of {tuple(x.shape)}")
    if x.dim() != 2 or x.stride(1) != 1:
        x2 = _rows(what, "x", x)
    rows, columns = x2.shape
    groups, line = (columns + GROUP - 1) // GROUP, (columns + 15) // 16 * 16
    if line == columns:
        values = torch.empty_like(x2, dtype=_E4M3, memory_format=torch.contiguous_format)
    else:
        values = x2.new_empty((rows, line), dtype=_E4M3)[:, :columns]
    scales = x2.new_empty((rows if group_rows == 1 else (rows + GROUP - 1) // GROUP, groups), dtype=torch.float32)
    _launch(what, "tris_quantize_e4m3", x.device, _QUANTIZE.pack(x2.data_ptr(), values.data_ptr(), scales.data_ptr(), x2.stride(0), line, groups, rows, columns, group_rows,
                                                                 _DTYPES[dtype]))
    if x.dim() != 2:
        return values.view(x.shape), scales.view(x.shape[:-1] + (groups,))
    return values, scales


def linear_e4m3(x: torch.Tensor, x_scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                dtype: torch.dtype = torch.float16, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``(x * x_scales) @ (weight * weight_scales).T + bias`` with sums in fp32, rounded once to ``dtype`` (fp16, bf16 or fp32).

    ``x`` [..., in_features] and ``weight`` [out_features, in_features] in ``torch.float8_e4m3fn``, their rows on 16-byte boundaries; ``x_scales``
    [..., ceil(in_features / 128)] and ``weight_scales`` [ceil(out_features / 128), ceil(in_features / 128)] in fp32; ``bias`` [out_features] in fp16, bf16 or fp32.
    ``status``: optional int32 tensor of one element, zero at first, set where a kernel gives up a wait (``raise_on_status``)."""
    what = "linear_e4m3"
    _same_device(what, x, x_scales, weight, weight_scales, bias, status)
    shape, x2, xs2 = x.shape, x, x_scales
    if x.dtype is not _E4M3 or weight.dtype is not _E4M3 or len(weight.shape) != 2 or not shape or shape[-1] != weight.shape[1]:
        _fail(what, f"x [..., in_features] and weight [out_features, in_features] must be {_E4M3}, got {x.dtype} {tuple(shape)} and {weight.dtype} {tuple(weight.shape)}")
    if dtype not in _LOGIT_TYPES:
        _fail(what, f"outputs are fp16, bf16 or fp32, not {dtype}")
    outputs, inputs = weight.shape
    groups = (inputs + GROUP - 1) // GROUP
    if len(shape) != 2 or x.stride(1) != 1:
        if x_scales.shape[:-1] != shape[:-1]:
            _fail(what, f"x_scales must be {tuple(shape[:-1])} x {groups}, got {tuple(x_scales.shape)}")
        x2, xs2 = _rows(what, "x", x), _rows(what, "x_scales", x_scales)
    rows = x2.shape[0]
    xs_at, xs_stride, _ = _matrix(what, "x_scales", xs2, torch.float32, rows, groups)
    ws_at, ws_stride, _ = _matrix(what, "weight_scales", weight_scales, torch.float32, (outputs + GROUP - 1) // GROUP, groups)
    w_stride, along = weight.stride()
    if along != 1 and inputs > 1:
        _fail(what, "weight must have a row side by side")
    bias_at = bias_type = status_at = 0
    if bias is not None:
        if bias.dtype not in _LOGIT_TYPES or bias.shape != (outputs,) or not bias.is_contiguous():
            _fail(what, f"bias must be contiguous fp16, bf16 or fp32 [{outputs}], got {bias.dtype} {tuple(bias.shape)}")
        bias_at, bias_type = bias.data_ptr(), _DTYPES[bias.dtype]
    if status is not None:
        if status.dtype is not torch.int32 or status.numel() != 1:
            _fail(what, "status must be an int32 tensor of one element")
        status_at = status.data_ptr()
    out = x2.new_empty((rows, outputs), dtype=dtype)
    _launch(what, "tris_e4m3_linear", x.device, _LINEAR.pack(x2.data_ptr(), xs_at, weight.data_ptr(), ws_at, bias_at, out.data_ptr(), status_at, x2.stride(0), xs_stride, w_stride,
                                                             ws_stride, outputs, rows, inputs, outputs, _DTYPES[dtype], bias_type, 0))
    return out if len(shape) == 2 else out.view(shape[:-1] + (outputs,))
