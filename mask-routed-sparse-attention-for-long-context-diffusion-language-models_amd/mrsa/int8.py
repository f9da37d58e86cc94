"""Linear layers in 8-bit integers: rows with one scale each, and their matrix product.

A row of activations, or of a weight matrix (an output channel), is held as int8 values in
[-127, 127] and one fp32 scale: y_k is about values_k * scale, scale = max |y_k| / 127.

    quantize_rows      rows in 8 bits (activations; weights, once)
    dequantize_rows    the values that 8-bit rows stand for
    add_rms_norm_int8  ``dream.add_rms_norm`` with its result in 8 bits
    swiglu_int8        ``dream.swiglu`` with its result in 8 bits
    int8_linear        8-bit rows times an 8-bit matrix, scaled, with a bias

The operators check their arguments themselves: on the GPU in csrc/torch_int8.cpp, for fake and CPU
tensors by the _check functions here, the same checks in the same words.  (They stand there, since
at one token the time of a call is the host's.  Only what torch.func.jvp differentiates, which no
kernel sees, is refused here.)

``DreamWeights.int8()`` makes a model's projections 8-bit and ``dream_forward`` runs on them.
Rounding to 8 bits has no useful derivative: the operators refuse tensors that ask for one.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from .rotary import DTYPES

MAX_DIM = 131071   # of int8_linear: products of 2^14, summed in 32 bits


def _no_gradient(name: str, *tensors) -> None:
    """Refuse tensors whose derivative a caller would wait for in vain, in either mode."""

    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no gradient: call it under torch.no_grad()")
    if forward_ad._current_level >= 0:   # (of dual tensors and of torch.func.jvp)
        wrapped = torch._C._functorch.is_functorch_wrapped_tensor
        for t in tensors:
            if t is not None and (wrapped(t) or forward_ad.unpack_dual(t).tangent is not None):
                raise ValueError(f"{name} has no forward-mode derivative")


def _check_rows(t, name: str) -> None:
    if t.ndim < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} must have rows of at least one value, got {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in DTYPES:
        raise ValueError(f"{name} must be bf16, fp16 or fp32, got {t.dtype}")


def _check_values(values, scales, name: str) -> None:
    if values.dtype != torch.int8 or not values.is_cuda or values.ndim < 1:
        raise ValueError(f"{name} must be CUDA int8 rows, got {tuple(values.shape)} "
                         f"{values.dtype} on {values.device}")
    if scales.shape != values.shape[:-1] or scales.dtype != torch.float32:
        raise ValueError(f"{name} of shape {tuple(values.shape)} need fp32 scales of shape "
                         f"{tuple(values.shape[:-1])}, got {tuple(scales.shape)} {scales.dtype}")
    if scales.device != values.device:
        raise ValueError(f"{name} and their scales must be on one device")


def _check_quantize(x) -> None:
    _check_rows(x, "x")
    _no_gradient("quantize_rows", x)


def _check_dequantize(values, scales, dtype) -> None:
    _check_values(values, scales, "values")
    if values.shape[-1] < 1:
        raise ValueError(f"values must have rows of at least one value, got {tuple(values.shape)}")
    if dtype not in DTYPES:
        raise ValueError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
    _no_gradient("dequantize_rows", scales)


def _check_norm(x, residual, weight, eps) -> None:
    _check_rows(x, "x")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype
                                 or residual.device != x.device):
        raise ValueError(f"residual must match x, got {tuple(residual.shape)} {residual.dtype} "
                         f"on {residual.device} for {tuple(x.shape)} {x.dtype} on {x.device}")
    if weight.shape != x.shape[-1:] or weight.dtype != x.dtype or weight.device != x.device:
        raise ValueError(f"weight must be [{x.shape[-1]}] {x.dtype} on {x.device}, got "
                         f"{tuple(weight.shape)} {weight.dtype} on {weight.device}")
    if not 1e-24 <= eps <= 1e24:
        raise ValueError(f"eps must be in [1e-24, 1e24], got {eps}")
    _no_gradient("add_rms_norm_int8", x, residual, weight)


def _check_swiglu(gate_up) -> None:
    _check_rows(gate_up, "gate_up")
    if gate_up.shape[-1] % 2:
        raise ValueError(f"gate_up must have an even last dim, got {tuple(gate_up.shape)}")
    _no_gradient("swiglu_int8", gate_up)


def _check_linear(x, x_scales, weight, weight_scales, bias, dtype) -> None:
    _check_values(x, x_scales, "x")
    _check_values(weight, weight_scales, "weight")
    dim = x.shape[-1]
    if weight.ndim != 2 or weight.shape[1] != dim:
        raise ValueError(f"weight must be [out_dim, {dim}], got {tuple(weight.shape)}")
    if weight.device != x.device:
        raise ValueError("x and weight must be on one device")
    if not 1 <= dim <= MAX_DIM:
        raise ValueError(f"rows of 1 to {MAX_DIM} values have a sum in 32 bits, got {dim}")
    if dtype not in DTYPES:
        raise ValueError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
    if bias is not None and (bias.shape != weight.shape[:1] or bias.dtype != dtype
                             or bias.device != x.device):
        raise ValueError(f"bias must be [{weight.shape[0]}] {dtype} on {x.device}, got "
                         f"{tuple(bias.shape)} {bias.dtype} on {bias.device}")
    _no_gradient("int8_linear", x_scales, weight_scales, bias)


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows in 8 bits: x [..., dim] in bf16, fp16 or fp32, any strides -> (values int8
    [..., dim], scales fp32 [...]).

    scale = max |x_k| / 127, values_k = round(x_k * 127 / max |x_k|), ties to even.  A row of
    zeros has scale 0; a row that holds an infinity or a NaN has scale NaN and values 0, so that
    what is made from it is NaN."""

    if forward_ad._current_level >= 0:
        _no_gradient("quantize_rows", x)
    return torch.ops.mrsa.quantize_rows.default(x)


def dequantize_rows(values: torch.Tensor, scales: torch.Tensor,
                    dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """values_k * scale in ``dtype`` (bf16, fp16 or fp32): what 8-bit rows stand for."""

    if forward_ad._current_level >= 0:
        _no_gradient("dequantize_rows", scales)
    return torch.ops.mrsa.dequantize_rows.default(values, scales, dtype)


def add_rms_norm_int8(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                      eps: float) -> Tuple[Optional[torch.Tensor], torch.Tensor, torch.Tensor]:
    """(x + residual in x's type or None, values int8, scales): the sum, and its
    root-mean-square norm times the weight in 8-bit rows as ``quantize_rows`` makes them.

    x, residual [..., dim] in bf16, fp16 or fp32, any strides; weight [dim] of the same type;
    eps from 1e-24 to 1e24.  The norm is that of the rounded sum, computed in fp32 with no
    rounding before the 8 bits."""

    if forward_ad._current_level >= 0:
        _no_gradient("add_rms_norm_int8", x, residual, weight)
    total, values, scales = torch.ops.mrsa.add_rms_norm_int8.default(x, residual, weight,
                                                                     float(eps))
    return (None if residual is None else total), values, scales


def swiglu_int8(gate_up: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """silu(gate) * up in 8-bit rows: gate_up [..., 2 dim] in bf16, fp16 or fp32 (gate columns
    first), any strides -> (values int8 [..., dim], scales fp32 [...]).  fp32 arithmetic, no
    rounding before the 8 bits; a product past fp32 counts as an infinity."""

    if forward_ad._current_level >= 0:
        _no_gradient("swiglu_int8", gate_up)
    return torch.ops.mrsa.swiglu_int8.default(gate_up)


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
    return torch.ops.mrsa.int8_linear.default(x, x_scales, weight, weight_scales, bias, dtype)
