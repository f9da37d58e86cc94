"""The Dream-shaped forward on 8-bit projections.

Every call of an 8-bit operator that the forward makes is checked against the definition in 64
bits on its own inputs (tolerances: tests/test_gpu_int8_linear.py), and the logits against the
bf16 model's.  An 8-bit row is off by a uniform error of one step, top / 127, whose deviation is
step / sqrt(12); at a top of about 4.5 deviations that is 1% of the row, for both factors 1.5% of a
projection's output.  A sublayer is two projections in a row (2.1%), and its error and the
others' add in quadrature to a residual stream that holds the embeddings beside them: 10% bounds
it for the few layers here.
"""

import pytest
import torch

import mrsa.dream as dream_mod
from mrsa.dream import DreamShape, DreamWeights, Int8Rows, dream_forward, landmark_layout
from mrsa.route_layer import RouteLayerConfig
from oracle import int8_oracle as O8
from test_gpu_int8_linear import U, check_linear, check_rows

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
SHAPE = DreamShape(layers=4, hidden=512, intermediate=1408, q_heads=28, kv_heads=4, vocab=1024,
                   mask_token_id=1023, route=RouteLayerConfig())


def _inputs(shape, L, seed):
    S = shape.route.chunk_size
    g = torch.Generator().manual_seed(seed)
    text = torch.randint(0, shape.vocab, (1, L // S * (S - 1)), generator=g)
    text[torch.rand(text.shape, generator=g) < 0.25] = shape.mask_token_id
    return landmark_layout(text, shape)[0].to(DEV)


def test_int8_forward_calls_and_logits(monkeypatch):
    w = DreamWeights.random(SHAPE, DEV, seed=5)
    w8 = w.int8()
    assert w8.layers[0].is_int8 and not w.layers[0].is_int8 and w8.lm_head is w.lm_head
    assert w8.int8().layers[1].qkv_weight is w8.layers[1].qkv_weight
    for a, b in zip(w.layers, w8.layers):
        for name in ("qkv_weight", "o_weight", "gate_up_weight", "down_weight", "qcal_down"):
            if getattr(a, name) is None:
                assert getattr(b, name) is None
                continue
            check_rows(*getattr(b, name), getattr(a, name).double(), 127 * 3 * U, U)
    ids = _inputs(SHAPE, 2048, 6)
    calls = []

    def spy(name):
        plain = getattr(dream_mod, name)

        def call(*args):
            out = plain(*args)
            calls.append((name, args, out))
            return out

        monkeypatch.setattr(dream_mod, name, call)

    for name in ("quantize_rows", "add_rms_norm_int8", "swiglu_int8", "int8_linear"):
        spy(name)
    logits = dream_forward(w8, ids)
    names = [c[0] for c in calls]
    layers, routes = SHAPE.layers, len(SHAPE.route_layers())
    assert routes == 1 and names.count("int8_linear") == 4 * layers + routes
    assert names.count("add_rms_norm_int8") == 2 * layers
    assert names.count("swiglu_int8") == names.count("quantize_rows") == layers
    for name, args, out in calls:
        if name == "int8_linear":
            check_linear(out, *args)
        elif name == "quantize_rows":
            check_rows(*out, args[0].double(), 127 * 3 * U, U)
        elif name == "swiglu_int8":
            slack = (1.5 * float(args[0].abs().max()) + 8) * U
            check_rows(*out, O8.swiglu_rows(args[0].double()), 127 * 2 * slack, 2 * slack)
        else:
            x, res, norm_w, eps = args
            t = x if res is None else (x.float() + res.float()).bfloat16()
            assert res is None or torch.equal(out[0], t)
            y = O8.norm_rows(t.double(), norm_w.double(), eps)
            check_rows(out[1], out[2], y, 127 * 5 * U, ((SHAPE.hidden / 64 + 24) / 2 + 8) * U)
    ref = dream_forward(w, ids).double()
    rel = float((logits.double() - ref).norm() / ref.norm())
    print(f"[gpu-case] int8 dream logits rel={rel:.3e}", flush=True)
    assert torch.isfinite(logits).all() and rel < 0.1


def test_some_layers_in_8_bits():
    """Layers of both forms in one model: each norm's output has the next projection's form."""

    w = DreamWeights.random(SHAPE, DEV, seed=7)
    ids = _inputs(SHAPE, 1024, 8)
    ref = dream_forward(w, ids).double()
    for which in ((0,), (1, 3), (2,)):
        mixed = DreamWeights(**{**vars(w), "layers": [
            lw.int8() if i in which else lw for i, lw in enumerate(w.layers)]})
        out = dream_forward(mixed, ids, return_hidden=False).double()
        assert 0 < float((out - ref).norm() / ref.norm()) < 0.1
    assert isinstance(mixed.layers[2].o_weight, Int8Rows)
