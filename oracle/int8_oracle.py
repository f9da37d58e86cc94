"""8-bit rows and their matrix product in 64 bits: the definitions themselves.

A row y of real numbers is held as whole numbers v and a scale: a = max |y_k|, scale = a / 127,
v_k the whole number nearest to 127 y_k / a (ties to even).  A row of zeros has scale 0 and
values 0, a row that is not finite scale NaN and values 0.
"""

import torch


def quantized(y):
    """fp64 rows -> (127 y / a before rounding, scale), both fp64."""

    top = y.abs().amax(dim=-1)
    top = torch.where(torch.isfinite(y).all(dim=-1), top, torch.nan)
    real = 127.0 * (y / torch.where(top > 0, top, 1.0)[..., None])
    return torch.where(torch.isnan(top)[..., None], 0.0, real), top / 127.0


def norm_rows(t, weight, eps):
    """Root-mean-square norm of fp64 rows."""

    return t / torch.sqrt((t * t).mean(dim=-1, keepdim=True) + eps) * weight


def swiglu_rows(gate_up):
    gate, up = gate_up.chunk(2, dim=-1)
    return gate / (1.0 + torch.exp(-gate)) * up


def linear(x, x_scales, weight, weight_scales, bias=None):
    """(result, the product before the bias) in fp64 from int8 operands: sums below 2^53 are
    exact."""

    sums = torch.matmul(x.double(), weight.double().T)
    product = sums * x_scales.double()[..., None] * weight_scales.double()
    return (product if bias is None else product + bias.double()), product
