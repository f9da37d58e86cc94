"""What the 8-bit operators (``mrsa.int8``) refuse, for fake and CPU tensors; csrc/torch_int8.cpp has
the same checks in the same words for the GPU's."""

from __future__ import annotations

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
