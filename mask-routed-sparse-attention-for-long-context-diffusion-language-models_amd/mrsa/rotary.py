"""Rotary positions: frequencies, tables, and the rotation with its gradient.

``rotary_qk`` is the general form of the rotation that ``dream.rope_qkv`` applies
to a fused projection: any head layout, part of the head, neighbouring or
half-apart pairs, a position per token, bf16 / fp16 / fp32, and autograd.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib

DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
SCALINGS = ("none", "linear", "ntk", "yarn")


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none",
                       factor: float = 1.0, original_max: int = 2048, beta_fast: float = 32.0,
                       beta_slow: float = 1.0) -> Tuple[torch.Tensor, float]:
    """fp64 inverse frequencies [rotary_dim / 2] and the factor on cos and sin.

    scaling stretches the context by ``factor``:
        "none"    base^(-2 i / rotary_dim)
        "linear"  positions divided by factor (Chen et al. 2023, position interpolation)
        "ntk"     base grown to base * factor^(R / (R - 2)), so that the slowest
                  frequency is divided by factor and the fastest kept
        "yarn"    per frequency between the two by its turns over original_max:
                  kept above beta_fast turns, divided by factor below beta_slow,
                  linear between; cos and sin times 0.1 ln(factor) + 1
                  (Peng et al. 2023; ``dream.yarn_inv_freq``'s formula)
    """

    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even, got {rotary_dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if not (base > 1.0 and math.isfinite(base)):
        raise ValueError(f"base must be finite and above 1, got {base}")
    if not (factor > 0.0 and math.isfinite(factor)):
        raise ValueError(f"factor must be finite and positive, got {factor}")
    R = rotary_dim
    exponent = torch.arange(0, R, 2, dtype=torch.float64) / R
    if scaling == "ntk":
        if R == 2:
            raise ValueError("ntk scaling needs rotary_dim above 2")
        return 1.0 / (base * factor ** (R / (R - 2))) ** exponent, 1.0
    inv = 1.0 / base ** exponent
    if scaling == "none" or factor == 1.0:
        return inv, 1.0
    if scaling == "linear":
        return inv / factor, 1.0
    if original_max <= 0 or not beta_fast > beta_slow > 0:
        raise ValueError("yarn scaling needs original_max > 0 and beta_fast > beta_slow > 0")

    def dim_of(turns):
        return R * math.log(original_max / (turns * 2 * math.pi)) / (2 * math.log(base))

    low = max(math.floor(dim_of(beta_fast)), 0)
    high = min(math.ceil(dim_of(beta_slow)), R - 1)
    if high <= low:
        high = low + 0.001
    ramp = ((torch.arange(R // 2, dtype=torch.float64) - low) / (high - low)).clamp(0, 1)
    return inv / factor * ramp + inv * (1 - ramp), 0.1 * math.log(factor) + 1.0


def rotary_tables(rows: int, inv_freq: torch.Tensor, attention_factor: float = 1.0,
                  device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 cos and sin tables [rows, rotary_dim / 2] of positions 0 .. rows - 1,
    times ``attention_factor``.  Angles are computed in fp64: an fp32 product of a
    position of 10^5 and a frequency is off by up to 4e-3 radians."""

    if rows < 0 or inv_freq.ndim != 1:
        raise ValueError(f"rotary tables need rows >= 0 and 1-D inv_freq, got {rows}, "
                         f"{tuple(inv_freq.shape)}")
    angles = torch.outer(torch.arange(rows, dtype=torch.float64, device=device),
                         inv_freq.to(device=device, dtype=torch.float64))
    return ((angles.cos() * attention_factor).float(), (angles.sin() * attention_factor).float())


def dense_rows(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy of it whose last dim is dense (the kernels take any other strides)."""

    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def check_tables(cos, sin, head_dim: int, device) -> None:
    shape = cos.shape
    if len(shape) != 2 or sin.shape != shape:
        raise ValueError(f"cos and sin must have the same shape [rows, rotary_dim / 2], got "
                         f"{tuple(shape)} and {tuple(sin.shape)}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be fp32")
    if cos.device != device or sin.device != device:
        raise ValueError("cos and sin must be on the device of the heads")
    if 2 * shape[1] > head_dim:
        raise ValueError(f"tables for {2 * shape[1]} dims do not fit heads of {head_dim}")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("cos and sin get no gradient")


def check_token_ints(t, name: str, batch: int, seq_len: int, device) -> torch.Tensor:
    """An int64 value per token, [seq_len] for all sequences or [batch, seq_len]."""

    if t.dtype != torch.long or t.device != device:
        raise ValueError(f"{name} must be torch.long on the device of the heads")
    if t.shape == (batch, seq_len):
        return t
    if t.shape != (seq_len,):
        raise ValueError(f"{name} must have shape {(batch, seq_len)} or {(seq_len,)}, "
                         f"got {tuple(t.shape)}")
    return t.expand(batch, seq_len)


def refuse_tangents(name: str, *tensors) -> None:
    """For the operators themselves, which have no forward-mode derivative: what a compiler has
    traced, or calls them directly, reaches them past the checks of the public functions."""

    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{name} has no forward-mode derivative here")


def _rotary_impl(q, k, cos, sin, positions, interleaved, inverse):
    refuse_tangents("mrsa::rotary", q, k)
    shape = q.shape
    B, L, Hq, D = shape
    qc, ct, st = dense_rows(q), cos.contiguous(), sin.contiguous()
    qb, ql, qh, _ = qc.stride()
    if k is None:
        Hkv, kp, kb, kl, kh = 0, None, 0, 0, 0
    else:
        kc = dense_rows(k)
        Hkv, kp = k.shape[2], kc.data_ptr()
        kb, kl, kh, _ = kc.stride()
    pp, pb, pl = (None, 0, 0) if positions is None else (positions.data_ptr(), *positions.stride())
    q_out, k_out = q.new_empty(shape), q.new_empty((B, L, Hkv, D))
    rows, half = cos.shape
    status = _lib.call_on(
        q.device, "mrsa_rotary_fwd", qc.data_ptr(), qb, ql, qh, kp, kb, kl, kh, ct.data_ptr(),
        st.data_ptr(), rows, pp, pb, pl, B, L, Hq, Hkv, D, 2 * half, DTYPES[q.dtype], interleaved,
        inverse, q_out.data_ptr(), k_out.data_ptr(), _lib.stream_of(q))
    _lib.check(status, "rotary_qk")
    return q_out, k_out


def _turn(q, k, cos, sin, positions, interleaved, inverse):
    return torch.ops.mrsa.rotary.default(q, k, cos, sin, positions, interleaved, inverse)


class _Rotary(torch.autograd.Function):
    # A rotation is linear and its transpose turns the other way, so the
    # gradient is the same operator (and differentiable itself).
    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, interleaved, inverse):
        ctx.save_for_backward(cos, sin, positions)
        ctx.interleaved, ctx.inverse = interleaved, inverse
        ctx.set_materialize_grads(False)
        return _turn(q, k, cos, sin, positions, interleaved, inverse)

    @staticmethod
    def backward(ctx, grad_q, grad_k):
        cos, sin, positions = ctx.saved_tensors
        if not ctx.needs_input_grad[0]:
            grad_q = None
        if not ctx.needs_input_grad[1]:
            grad_k = None
        args = (cos, sin, positions, ctx.interleaved, not ctx.inverse)
        dq = dk = None
        if grad_q is not None:
            dq, dk = _rotate(grad_q, grad_k, *args)
        elif grad_k is not None:
            dk, _ = _rotate(grad_k, None, *args)
        return dq, None if grad_k is None else dk, None, None, None, None, None


class _RotaryTransformed(_Rotary):
    # The form for forward-mode derivatives and torch.func's transforms (a call of it takes
    # longer, hence two forms): the derivative along a tangent is the tangent, turned.
    generate_vmap_rule = True

    @staticmethod
    def forward(q, k, cos, sin, positions, interleaved, inverse):
        return _turn(q, k, cos, sin, positions, interleaved, inverse)

    @staticmethod
    def setup_context(ctx, inputs, output):
        q, k, cos, sin, positions, ctx.interleaved, ctx.inverse = inputs
        ctx.save_for_backward(cos, sin, positions)
        ctx.save_for_forward(cos, sin, positions)
        ctx.q_shape, ctx.k_shape = q.shape, output[1].shape
        ctx.set_materialize_grads(False)

    @staticmethod
    def jvp(ctx, q_tangent, k_tangent, *_):
        args = (*ctx.saved_tensors, ctx.interleaved, ctx.inverse)
        if q_tangent is None:
            return k_tangent.new_zeros(ctx.q_shape), _rotate(k_tangent, None, *args)[0]
        dq, dk = _rotate(q_tangent, k_tangent, *args)
        return dq, dk if k_tangent is not None else dk.new_zeros(ctx.k_shape)


def _rotate(q, k, *args):
    """The operator, recorded where a derivative of it may be asked for."""

    if forward_ad._current_level >= 0:   # (of dual tensors and of torch.func.jvp)
        return _RotaryTransformed.apply(q, k, *args)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        if torch._C._are_functorch_transforms_active():
            return _RotaryTransformed.apply(q, k, *args)
        return _Rotary.apply(q, k, *args)
    return _turn(q, k, *args)


def check_heads(t, name: str) -> None:
    if t.ndim != 4:
        raise ValueError(f"{name} must have shape [B, L, heads, head_dim], got {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in DTYPES:
        raise ValueError(f"{name} must be bf16, fp16 or fp32, got {t.dtype}")


def rotary_qk(q: torch.Tensor, k: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor,
              positions: Optional[torch.Tensor] = None, *, interleaved: bool = False
              ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Query and key heads turned by their positions; differentiable in q and k (reverse and
    forward mode, and under torch.func's transforms; what torch.compile has traced refuses
    dual tensors).

    q [B, L, Hq, D] and k [B, L, Hkv, D] (or None) in bf16, fp16 or fp32, any
    strides; cos, sin fp32 [rows, R / 2] (``rotary_tables``), R <= D: the first R dims
    of a head turn, in pairs (i, i + R / 2), or (2 i, 2 i + 1) if interleaved, the
    others are copied.  positions: torch.long [B, L] or [L]; None: row i is at
    position i.  A position outside the tables makes its rows' turned dims NaN.
    Returns new dense (q', k'); fp32 arithmetic with one rounding.
    To capture a backward pass, take it by torch.autograd.grad inside the capture, with no
    eager graph of the same leaves alive.
    """

    check_heads(q, "q")
    B, L, _, D = q.shape
    if k is not None:
        check_heads(k, "k")
        if k.shape != (B, L, k.shape[2], D) or k.dtype != q.dtype:
            raise ValueError(f"q and k must agree in batch, length, head_dim and dtype, got "
                             f"{tuple(q.shape)} {q.dtype} and {tuple(k.shape)} {k.dtype}")
        if k.device != q.device:
            raise ValueError("q and k must be on one device")
    check_tables(cos, sin, D, q.device)
    if positions is not None:
        positions = check_token_ints(positions, "positions", B, L, q.device)
    elif L > cos.shape[0]:
        raise ValueError(f"tables of {cos.shape[0]} rows do not reach {L} positions")
    q_out, k_out = _rotate(q, k, cos, sin, positions, bool(interleaved), False)
    return q_out, None if k is None else k_out
