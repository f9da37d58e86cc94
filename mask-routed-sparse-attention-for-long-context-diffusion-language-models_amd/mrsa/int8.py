"""Linear layers in 8-bit integers: rows with one scale each, and their matrix product.

A row of activations, or of a weight matrix (an output channel), is held as int8 values in
[-127, 127] and one fp32 scale: y_k is about values_k * scale, scale = max |y_k| / 127 (rounded so
that 127 * scale is finite where the row is).

    quantize_rows      rows in 8 bits (activations; weights, once)
    dequantize_rows    the values that 8-bit rows stand for
    add_rms_norm_int8  ``dream.add_rms_norm`` with its result in 8 bits
    swiglu_int8        ``dream.swiglu`` with its result in 8 bits
    int8_linear        8-bit rows times an 8-bit matrix, scaled, with a bias

The operators check their arguments themselves: on the GPU in csrc/torch_int8.cpp, for fake and CPU
tensors in int8_checks.py, the same checks in the same words.  (They stand there, since at one token
the time of a call is the host's.)

``DreamWeights.int8()`` makes a model's projections 8-bit and ``dream_forward`` runs on them.
Rounding to 8 bits has no useful derivative: the operators refuse tensors that ask for one, in
either mode and under torch.func's transforms (the autograd kernels of csrc/torch_int8.cpp; dual
tensors already here, before any trace).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import ops  # noqa: F401  (defines the operators)
from .int8_checks import _no_gradient

_quantize_rows = torch.ops.mrsa.quantize_rows.default
_dequantize_rows = torch.ops.mrsa.dequantize_rows.default
_add_rms_norm_int8 = torch.ops.mrsa.add_rms_norm_int8.default
_swiglu_int8 = torch.ops.mrsa.swiglu_int8.default
_int8_linear = torch.ops.mrsa.int8_linear.default


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows in 8 bits: x [..., dim] in bf16, fp16 or fp32, any strides -> (values int8
    [..., dim], scales fp32 [...]).

    scale = max |x_k| / 127, values_k = round(x_k * 127 / max |x_k|), ties to even.  A row of
    zeros has scale 0; a row that holds an infinity or a NaN has scale NaN and values 0, so that
    what is made from it is NaN."""

    if forward_ad._current_level >= 0:
        _no_gradient("quantize_rows", x)
    return _quantize_rows(x)


def dequantize_rows(values: torch.Tensor, scales: torch.Tensor,
                    dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """values_k * scale in ``dtype`` (bf16, fp16 or fp32): what 8-bit rows stand for."""

    if forward_ad._current_level >= 0:
        _no_gradient("dequantize_rows", scales)
    return _dequantize_rows(values, scales, dtype)


def add_rms_norm_int8(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                      eps: float) -> Tuple[Optional[torch.Tensor], torch.Tensor, torch.Tensor]:
    """(x + residual in x's type or None, values int8, scales): the sum, and its
    root-mean-square norm times the weight in 8-bit rows as ``quantize_rows`` makes them.

    x, residual [..., dim] in bf16, fp16 or fp32, any strides; weight [dim] of the same type;
    eps from 1e-24 to 1e24.  The norm is that of the rounded sum, computed in fp32 with no
    rounding before the 8 bits; a result past fp32 counts as an infinity."""

    if forward_ad._current_level >= 0:
        _no_gradient("add_rms_norm_int8", x, residual, weight)
    total, values, scales = _add_rms_norm_int8(x, residual, weight, eps)
    return (None if residual is None else total), values, scales


def swiglu_int8(gate_up: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """silu(gate) * up in 8-bit rows: gate_up [..., 2 dim] in bf16, fp16 or fp32 (gate columns
    first), any strides -> (values int8 [..., dim], scales fp32 [...]).  fp32 arithmetic, no
    rounding before the 8 bits; a product past fp32 counts as an infinity."""

    if forward_ad._current_level >= 0:
        _no_gradient("swiglu_int8", gate_up)
    return _swiglu_int8(gate_up)


def int8_linear(x: torch.Tensor, x_scales: torch.Tensor, weight: torch.Tensor,
                weight_scales: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out[..., n] = x_scales[...] weight_scales[n] sum_k x[..., k] weight[n, k] + bias[n].

    x int8 [..., dim] with fp32 scales [...], weight int8 [out_dim, dim] with fp32 scales
    [out_dim] (``quantize_rows`` makes both), bias [out_dim] of the result's ``dtype`` (bf16,
    fp16 or fp32).  Any row strides; rows and matrices that are 16-byte aligned with dim a
    multiple of 16 are fastest.  The sum is exact in int32 (dim up to 131071); scales (the row's
    first), bias and the rounding follow in fp32, so equal inputs give equal bits."""

    if forward_ad._current_level >= 0:
        _no_gradient("int8_linear", x_scales, weight_scales, bias)
    return _int8_linear(x, x_scales, weight, weight_scales, bias, dtype)
