"""Linear layers in 8-bit integers as a program calls them.

A row of activations or of a weight matrix is held as int8 values and one fp32 scale: the
largest magnitude of the row stands for 127.  Sizes are those of the package's own
model shape (hidden size 3584, 18944 inside the MLP, 28 + 2 * 4 heads of 128 behind the fused
projection, 32-token decode blocks, 16384-token sequences), of the shapes it is tested at, or
odd ones.  Values are seeded N(0, 1) activations, a few channels of them ten times as large as
the others, and N(0, 0.02) weights.

Families ("kind"):
    quantize  rows of activations in 8 bits             mrsa.quantize_rows
    norm      a residual's addition, the root-mean-square norm of the sum, its rows
              in 8 bits                                 mrsa.add_rms_norm_int8
    swiglu    the gated activation, its rows in 8 bits  mrsa.swiglu_int8
    linear    8-bit rows times an 8-bit matrix          mrsa.int8_linear

What is held in 8 bits is returned as the values that it stands for, in bf16
(mrsa.dequantize_rows), beside its scales.
"""

import glob
import math
import os
import sys

import torch

sys.path[:0] = glob.glob(os.path.join(os.getcwd(), "mask-routed-*_amd"))

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


def _quantize(**more):
    return {"kind": "quantize", "rows": 1, "dim": 3584, "type": "bf16", "sliced": False,
            "padded": False, **more}


def _norm(**more):
    return {"kind": "norm", "rows": 1, "dim": 3584, "type": "bf16", "residual": True,
            "padded": False, **more}


def _swiglu(**more):
    return {"kind": "swiglu", "rows": 1, "dim": 18944, "type": "bf16", "padded": False, **more}


def _linear(**more):
    return {"kind": "linear", "rows": 1, "out": 4608, "dim": 3584, "type": "bf16", "bias": False,
            "sliced": False, **more}


def listed():
    return [
        # attention outputs of a decode block before the output projection: latency
        _quantize(name="quantize_block", rows=32),
        # the same of a whole sequence
        _quantize(name="quantize_16k", rows=16384),
        # one token before a layer's projections: latency
        _norm(name="norm_token"),
        # a layer's norm over a whole sequence
        _norm(name="norm_16k", rows=16384),
        # rows that nothing is aligned to, the first norm (no residual yet), padding behind
        _norm(name="norm_odd", rows=2003, dim=1001, type="fp16", residual=False, padded=True),
        # the MLP's activations of a decode block
        _swiglu(name="swiglu_block", rows=32),
        # the same of a whole sequence
        _swiglu(name="swiglu_16k", rows=16384),
        # one token through the fused projection of queries, keys and values: the weights' bytes
        _linear(name="linear_token", bias=True),
        # a decode block into the MLP: the weights' bytes
        _linear(name="linear_block_mlp", rows=32, out=37888),
        # a prompt of odd length out of the MLP: few output tiles, a long sum
        _linear(name="linear_prompt_down", rows=1003, out=3584, dim=18944, type="fp16"),
        # odd sizes everywhere, a 32-bit result
        _linear(name="linear_odd", rows=517, out=1001, dim=1003, type="fp32", bias=True),
        # a whole sequence into the MLP: the matrix products
        _linear(name="linear_16k_mlp", rows=16384, out=37888),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "norm", "swiglu", "linear", "linear", "linear", "linear"])
    type_ = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind != "linear":
        dim = rng.choice([3584, 896, 8192, _log_int(rng, 1, 20000), _log_int(rng, 64, 20000)])
        # no more values than a sequence's rows in the MLP
        rows = _log_int(rng, 1, min(65536, 16384 * 18944 / 2 / dim))
        padded = rng.random() < 0.3
        if kind == "quantize":
            return _quantize(rows=rows, dim=dim, type=type_, sliced=rng.random() < 0.3,
                             padded=padded)
        if kind == "norm":
            return _norm(rows=rows, dim=dim, type=type_, residual=rng.random() < 0.7,
                         padded=padded)
        return _swiglu(rows=rows, dim=dim, type=type_, padded=padded)
    out, dim = rng.choice([(4608, 3584), (3584, 3584), (37888, 3584), (3584, 18944), (64, 3584),
                           (_log_int(rng, 1, 40000), _log_int(rng, 16, 20000)),
                           (_log_int(rng, 64, 10000), _log_int(rng, 64, 10000)),
                           (16 * _log_int(rng, 4, 1000), 16 * _log_int(rng, 4, 1000))])
    # no more products than the largest listed case
    rows = _log_int(rng, 1, min(16384, 16384 * 37888 * 3584 / (out * dim)))
    rows = rng.choice([rows, rows, rows, 1, 32])
    return _linear(rows=rows, out=out, dim=dim, type=type_, bias=rng.random() < 0.4,
                   sliced=rng.random() < 0.2)


def _in_8_bits(y):
    """fp32 rows [rows, dim] as whole numbers in [-127, 127] (fp32) and a scale for each row."""
    top = y.abs().amax(dim=-1, keepdim=True)
    up = torch.where(top > 0, 127.0 / top, 0.0)
    return (y * up).round(), (top / 127.0)[:, 0]


def prepare(case, seed):
    c, device = case, torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    rows, dim = c["rows"], c["dim"]

    def activations(width, dtype, sliced=False):
        x = torch.empty(rows, width + (24 if sliced else 0), device=device)
        x.normal_(0.0, 1.0, generator=gen)
        # the channels that stand out
        loud = torch.rand(x.shape[1], generator=gen, device=device) < 0.003
        x *= torch.where(loud, 10.0, 1.0)
        if c.get("padded"):
            x[rows - rows // 8:] = 0.0  # tokens behind the sequence's end
        x = x.to(dtype)
        return x[:, 8:8 + width] if sliced else x

    s = {"case": c}
    if c["kind"] == "linear":
        x, s["x_scales"] = _in_8_bits(activations(dim, torch.float32))
        x = x.to(torch.int8)
        if c["sliced"]:  # part of wider rows
            wide = torch.zeros(rows, dim + 48, dtype=torch.int8, device=device)
            wide[:, 16:16 + dim] = x
            x = wide[:, 16:16 + dim]
        s["x"] = x
        w = torch.empty(c["out"], dim, device=device).normal_(0.0, 0.02, generator=gen)
        w, s["w_scales"] = _in_8_bits(w)
        s["w"] = w.to(torch.int8)
        s["bias"] = None
        if c["bias"]:
            s["bias"] = torch.empty(c["out"], device=device).normal_(0.0, 0.1, generator=gen)
            s["bias"] = s["bias"].to(TYPES[c["type"]])
        return s
    dtype = TYPES[c["type"]]
    s["x"] = activations(2 * dim if c["kind"] == "swiglu" else dim, dtype, c.get("sliced", False))
    if c["kind"] == "norm":
        s["residual"] = activations(dim, dtype) if c["residual"] else None
        s["weight"] = (1.0 + 0.1 * torch.randn(dim, generator=gen, device=device)).to(dtype)
    return s


def _plain_rows(y):
    """What rows in 8 bits stand for, and their scales."""
    values, scales = _in_8_bits(y)
    return (values * scales[:, None]).to(torch.bfloat16), scales


def _run_quantize(s):
    if own:
        import mrsa

        values, scales = mrsa.quantize_rows(s["x"])
        return mrsa.dequantize_rows(values, scales, torch.bfloat16), scales
    return _plain_rows(s["x"].float())


def _run_norm(s):
    if own:
        import mrsa

        total, values, scales = mrsa.add_rms_norm_int8(s["x"], s["residual"], s["weight"], EPS)
        return total, mrsa.dequantize_rows(values, scales, torch.bfloat16), scales
    total, x = None, s["x"]
    if s["residual"] is not None:  # the sum is kept in the inputs' type, and normed as kept
        total = x = (x.float() + s["residual"].float()).to(x.dtype)
    x = x.float()
    r = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS)
    values, scales = _plain_rows(x * r * s["weight"].float())
    return total, values, scales


def _run_swiglu(s):
    if own:
        import mrsa

        values, scales = mrsa.swiglu_int8(s["x"])
        return mrsa.dequantize_rows(values, scales, torch.bfloat16), scales
    dim = s["case"]["dim"]
    gate, up = s["x"][:, :dim].float(), s["x"][:, dim:].float()
    return _plain_rows(gate / (1.0 + torch.exp(-gate)) * up)


def _run_linear(s):
    dtype = TYPES[s["case"]["type"]]
    if own:
        import mrsa

        return mrsa.int8_linear(s["x"], s["x_scales"], s["w"], s["w_scales"], s["bias"],
                                dtype=dtype)
    out = torch.matmul(s["x"].float(), s["w"].float().T)
    out = out * s["x_scales"][:, None] * s["w_scales"]
    if s["bias"] is not None:
        out = out + s["bias"].float()
    return out.to(dtype)


_RUNS = {"quantize": _run_quantize, "norm": _run_norm, "swiglu": _run_swiglu,
         "linear": _run_linear}


def run(state):
    return _RUNS[state["case"]["kind"]](state)


def work(case):
    c = case
    size, rows, dim = SIZES[c["type"]], c["rows"], c["dim"]
    if c["kind"] == "linear":
        out = c["out"]
        return {"bytes": rows * dim + out * dim + 4 * (rows + out) + rows * out * size
                + (out * size if c["bias"] else 0), "flops": 2 * rows * out * dim}
    # the rows' values (in bf16, as they are returned) and scales
    written = rows * (2 * dim + 4)
    if c["kind"] == "quantize":
        return {"bytes": rows * dim * size + written, "flops": 3 * rows * dim}
    if c["kind"] == "norm":
        moved = rows * dim * size * (3 if c["residual"] else 1) + dim * size
        return {"bytes": moved + written, "flops": 8 * rows * dim}
    return {"bytes": 2 * rows * dim * size + written, "flops": 8 * rows * dim}


def _exact_rows(y):
    top = y.abs().max(dim=-1).values
    step = top / 127
    whole = torch.round(y / torch.where(step > 0, step, 1.0)[:, None])
    return whole * step[:, None], step


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["kind"] == "quantize":
        return _exact_rows(x)
    if case["kind"] == "swiglu":
        gate, up = x.chunk(2, dim=-1)
        return _exact_rows(gate * torch.sigmoid(gate) * up)
    if case["kind"] == "norm":
        total = None
        if s["residual"] is not None:
            total = x + s["residual"].double()
            x = total.to(s["x"].dtype).double()  # as it is kept
        size = torch.linalg.vector_norm(x, dim=-1, keepdim=True) / math.sqrt(case["dim"])
        y = x / torch.hypot(size, torch.full_like(size, math.sqrt(EPS))) * s["weight"].double()
        return (total, *_exact_rows(y))
    # whole numbers below 2^53: each product in 64 bits is exact; a slice of the channels at a time
    out = torch.empty(case["rows"], case["out"], dtype=torch.float64, device=x.device)
    x = x * s["x_scales"].double()[:, None]
    for n in range(0, case["out"], 8192):
        at = slice(n, n + 8192)
        w = s["w"][at].double() * s["w_scales"][at].double()[:, None]
        out[:, at] = torch.nn.functional.linear(x, w)
        if s["bias"] is not None:
            out[:, at] += s["bias"][at].double()
    return out
