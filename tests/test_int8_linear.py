"""The 8-bit operators without a GPU: refusals, C entry points, shapes and traced graphs; and the
oracle against closed forms."""

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mrsa
from mrsa import _lib
from mrsa.dream import DreamLayerWeights, DreamShape, DreamWeights
from oracle import int8_oracle as O8


def _fake(*shape, dtype=torch.bfloat16, device="cuda"):
    return torch.empty(*shape, dtype=dtype, device=device)


def test_oracle_rows():
    y = torch.tensor([[127.0, -63.5, 1.0, 0.0], [0.0, 0.0, 0.0, 0.0],
                      [1.0, float("inf"), 0.0, 2.0], [float("nan"), 1.0, 2.0, 3.0],
                      [-2.0, 1.0, 0.5, 0.25]], dtype=torch.float64)
    real, scale = O8.quantized(y)
    assert real[0].tolist() == [127.0, -63.5, 1.0, 0.0] and scale[0] == 1.0
    assert not real[1:4].any() and scale[1] == 0 and scale[2:4].isnan().all()
    assert real[4].tolist() == [-127.0, 63.5, 31.75, 15.875] and scale[4] == 2.0 / 127.0


def test_oracle_norm_swiglu_linear():
    t = torch.tensor([[3.0, 4.0]], dtype=torch.float64)
    w = torch.tensor([2.0, 0.5], dtype=torch.float64)
    r = 1 / math.sqrt(12.5 + 0.5)
    torch.testing.assert_close(O8.norm_rows(t, w, 0.5), torch.tensor([[6 * r, 2 * r]]).double())
    g = torch.tensor([[0.0, math.log(3.0), 5.0, 4.0]], dtype=torch.float64)
    torch.testing.assert_close(O8.swiglu_rows(g),
                               torch.tensor([[0.0, math.log(3.0) * 0.75 * 4.0]]).double())
    x = torch.tensor([[-128, 127], [1, 2]], dtype=torch.int8)
    out, product = O8.linear(x, torch.tensor([0.5, 2.0]), x, torch.tensor([1.0, 0.25]),
                             torch.tensor([1.0, -1.0]))
    assert product.tolist() == [[0.5 * (128 ** 2 + 127 ** 2), 0.125 * (-128 + 254)],
                                [2.0 * (-128 + 254), 0.5 * 5]]
    assert torch.equal(out, product + torch.tensor([1.0, -1.0]).double())


BAD_ROWS = [
    (lambda: _fake(4, 8, device="cpu"), "CUDA"),
    (lambda: _fake(4, 8, dtype=torch.float64), "bf16, fp16 or fp32"),
    (lambda: _fake(4, 8, dtype=torch.int8), "bf16, fp16 or fp32"),
    (lambda: _fake(()), "at least one"),
    (lambda: _fake(4, 0), "at least one"),
]


@pytest.mark.parametrize("make,words", BAD_ROWS)
def test_rows_refused(make, words):
    with FakeTensorMode():
        x = make()
        with pytest.raises(ValueError, match=words):
            mrsa.quantize_rows(x)
        with pytest.raises(ValueError, match=words):
            mrsa.swiglu_int8(x)
        with pytest.raises(ValueError, match=words):
            mrsa.add_rms_norm_int8(x, None, x, 1e-6)


def test_norm_refused():
    with FakeTensorMode():
        x, w = _fake(4, 8), _fake(8)
        for res in (_fake(3, 8), _fake(4, 8, dtype=torch.float16), _fake(4, 8, device="cpu")):
            with pytest.raises(ValueError, match="residual"):
                mrsa.add_rms_norm_int8(x, res, w, 1e-6)
        for bad in (_fake(4), _fake(8, dtype=torch.float32), _fake(8, device="cpu"), _fake(1, 8)):
            with pytest.raises(ValueError, match="weight"):
                mrsa.add_rms_norm_int8(x, None, bad, 1e-6)
        for eps in (0.0, -1e-6, 1e-25, 1e25, float("nan"), float("inf")):
            with pytest.raises(ValueError, match="eps"):
                mrsa.add_rms_norm_int8(x, None, w, eps)
        with pytest.raises(ValueError, match="even"):
            mrsa.swiglu_int8(_fake(4, 7))


def test_dequantize_refused():
    with FakeTensorMode():
        v, s = _fake(4, 8, dtype=torch.int8), _fake(4, dtype=torch.float32)
        for bad in (_fake(4, 8), _fake(4, 8, dtype=torch.uint8),
                    _fake(4, 8, dtype=torch.int8, device="cpu")):
            with pytest.raises(ValueError, match="int8"):
                mrsa.dequantize_rows(bad, s)
        for bad in (_fake(3, dtype=torch.float32), _fake(4, 1, dtype=torch.float32), _fake(4)):
            with pytest.raises(ValueError, match="scales"):
                mrsa.dequantize_rows(v, bad)
        with pytest.raises(ValueError, match="one device"):
            mrsa.dequantize_rows(v, _fake(4, dtype=torch.float32, device="cpu"))
        with pytest.raises(ValueError, match="dtype"):
            mrsa.dequantize_rows(v, s, torch.int32)
        with pytest.raises(ValueError, match="at least one"):
            mrsa.dequantize_rows(v[:, :0], s)


def test_linear_refused():
    with FakeTensorMode():
        x, sx = _fake(4, 32, dtype=torch.int8), _fake(4, dtype=torch.float32)
        w, sw = _fake(6, 32, dtype=torch.int8), _fake(6, dtype=torch.float32)
        assert mrsa.int8_linear(x, sx, w, sw).shape == (4, 6)
        for bad in (_fake(6, 31, dtype=torch.int8), _fake(2, 6, 32, dtype=torch.int8)):
            with pytest.raises(ValueError, match="weight"):
                mrsa.int8_linear(x, sx, bad, _fake(*bad.shape[:-1], dtype=torch.float32))
        with pytest.raises(ValueError, match="int8"):
            mrsa.int8_linear(_fake(4, 32), sx, w, sw)
        with pytest.raises(ValueError, match="int8"):
            mrsa.int8_linear(x, sx, _fake(6, 32), sw)
        with pytest.raises(ValueError, match="scales"):
            mrsa.int8_linear(x, sw, w, sw)
        with pytest.raises(ValueError, match="scales"):
            mrsa.int8_linear(x, sx, w, _fake(6))
        for bias in (_fake(5), _fake(6, dtype=torch.float32), _fake(6, device="cpu"),
                     _fake(1, 6)):
            with pytest.raises(ValueError, match="bias"):
                mrsa.int8_linear(x, sx, w, sw, bias)
        mrsa.int8_linear(x, sx, w, sw, _fake(6, dtype=torch.float32), dtype=torch.float32)
        with pytest.raises(ValueError, match="dtype"):
            mrsa.int8_linear(x, sx, w, sw, dtype=torch.int8)
        for dim in (0, 131072):
            a, b = _fake(4, dim, dtype=torch.int8), _fake(6, dim, dtype=torch.int8)
            with pytest.raises(ValueError, match="131071"):
                mrsa.int8_linear(a, sx, b, sw)


def test_tensors_that_ask_for_a_derivative_are_refused():
    with FakeTensorMode():
        x = _fake(4, 8).requires_grad_()
        w = _fake(8)
        v, s = _fake(4, 8, dtype=torch.int8), _fake(4, dtype=torch.float32).requires_grad_()
        b = _fake(4).requires_grad_()
        calls = (lambda: mrsa.quantize_rows(x), lambda: mrsa.swiglu_int8(x),
                 lambda: mrsa.add_rms_norm_int8(x, None, w, 1e-6),
                 lambda: mrsa.add_rms_norm_int8(x.detach(), x, w, 1e-6),
                 lambda: mrsa.add_rms_norm_int8(x.detach(), None, x[0], 1e-6),
                 lambda: mrsa.dequantize_rows(v, s), lambda: mrsa.int8_linear(v, s, v, s.detach()),
                 lambda: mrsa.int8_linear(v, s.detach(), v, s),
                 lambda: mrsa.int8_linear(v, s.detach(), v, s.detach(), b))
        for call in calls:
            with pytest.raises(ValueError, match="no gradient"):
                call()
            with torch.no_grad():
                call()


def test_dual_tensors_are_refused():
    from torch.autograd import forward_ad

    x = torch.zeros(4, 8)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        from mrsa import int8

        with pytest.raises(ValueError, match="forward-mode"):
            int8._no_gradient("quantize_rows", dual)
        int8._no_gradient("quantize_rows", x)


def test_a_missing_library_is_an_error_of_the_call():
    error = mrsa.ops._load_native("/nonexistent/libmrsa_torch.so")
    assert isinstance(error, mrsa.MrsaLibraryError) and "build" in str(error)
    assert mrsa.ops._native_error is None   # (built for these tests)


def test_fake_results():
    with FakeTensorMode():
        x = _fake(2, 3, 64, dtype=torch.float16)
        total, v, s = mrsa.add_rms_norm_int8(x, x, _fake(64, dtype=torch.float16), 1e-5)
        assert total.shape == x.shape and total.dtype == torch.float16
        assert v.shape == x.shape and v.dtype == torch.int8
        assert s.shape == (2, 3) and s.dtype == torch.float32
        none, _, _ = mrsa.add_rms_norm_int8(x, None, _fake(64, dtype=torch.float16), 1e-5)
        assert none is None
        v, s = mrsa.swiglu_int8(x)
        assert v.shape == (2, 3, 32) and s.shape == (2, 3)
        w, sw = mrsa.quantize_rows(_fake(10, 32))
        out = mrsa.int8_linear(v, s, w, sw, _fake(10, dtype=torch.float16), dtype=torch.float16)
        assert out.shape == (2, 3, 10) and out.dtype == torch.float16
        back = mrsa.dequantize_rows(v, s, torch.float32)
        assert back.shape == v.shape and back.dtype == torch.float32
        row = mrsa.quantize_rows(_fake(7))
        assert row[0].shape == (7,) and row[1].shape == ()


class _Mlp(torch.nn.Module):
    def forward(self, x, res, norm_w, gu, sgu, down, sdown):
        total, v, s = mrsa.add_rms_norm_int8(x, res, norm_w, 1e-6)
        v, s = mrsa.swiglu_int8(mrsa.int8_linear(v, s, gu, sgu))
        return total, mrsa.int8_linear(v, s, down, sdown), mrsa.dequantize_rows(v, s)


def test_an_8_bit_mlp_exports_as_one_graph():
    with FakeTensorMode(allow_non_fake_inputs=True):
        args = (_fake(40, 64), _fake(40, 64), _fake(64), _fake(192, 64, dtype=torch.int8),
                _fake(192, dtype=torch.float32), _fake(64, 96, dtype=torch.int8),
                _fake(64, dtype=torch.float32))
        with torch.no_grad():
            ep = torch.export.export(_Mlp(), args, strict=True)
    names = [str(n.target) for n in ep.graph.nodes if n.op == "call_function"]
    assert names.count("mrsa.int8_linear.default") == 2
    for op in ("add_rms_norm_int8", "swiglu_int8", "dequantize_rows"):
        assert f"mrsa.{op}.default" in names


def test_c_entry_points_check_before_they_launch():
    call = _lib.call
    p = 64  # (an address that is never followed)
    bf16, fp32 = 0, 2
    assert call("mrsa_quantize_rows_fwd", None, 8, 0, 8, bf16, None, None, None) == 0
    assert call("mrsa_quantize_rows_fwd", None, 8, 2, 8, bf16, p, p, None) == 1
    assert call("mrsa_quantize_rows_fwd", p, 8, -1, 8, bf16, p, p, None) == 1
    assert call("mrsa_quantize_rows_fwd", p, -8, 2, 8, bf16, p, p, None) == 1
    assert call("mrsa_quantize_rows_fwd", p, 8, 2, 8, 3, p, p, None) == 2
    assert call("mrsa_quantize_rows_fwd", p, 8, 2, 0, bf16, p, p, None) == 2
    assert call("mrsa_quantize_rows_fwd", p + 1, 8, 2, 8, bf16, p, p, None) == 1
    assert call("mrsa_quantize_rows_fwd", p + 2, 8, 2, 8, fp32, p, p, None) == 1
    assert call("mrsa_quantize_rows_fwd", p, 8, 2, 8, bf16, p, p + 2, None) == 1
    assert call("mrsa_quantize_rows_fwd", p, 8, 2, (1 << 31) + 1, bf16, p, p, None) == 2
    assert call("mrsa_quantize_rows_fwd", p, 1 << 50, 1 << 10, 8, bf16, p, p, None) == 2
    assert call("mrsa_swiglu_int8_fwd", None, 16, 0, 8, bf16, None, None, None) == 0
    assert call("mrsa_swiglu_int8_fwd", p, 16, 2, 8, bf16, None, p, None) == 1
    assert call("mrsa_swiglu_int8_fwd", p, 16, 2, 8, 7, p, p, None) == 2
    for dim in (0, (1 << 30) + 1, 1 << 62, (1 << 63) - 1):   # (twice it may pass 63 bits)
        assert call("mrsa_swiglu_int8_fwd", p, 16, 2, dim, bf16, p, p, None) == 2
    norm = "mrsa_add_rms_norm_int8_fwd"
    assert call(norm, None, 8, None, 0, None, 0, 8, 1e-6, bf16, None, None, None, None) == 0
    assert call(norm, p, 8, p, 8, p, 2, 8, 1e-6, bf16, None, p, p, None) == 1   # sum nowhere
    assert call(norm, p, 8, None, 0, p, 2, 8, 1e-6, bf16, p, p, p, None) == 1   # of nothing
    assert call(norm, p, 8, None, 0, p, 2, 8, 0.0, bf16, None, p, p, None) == 1
    assert call(norm, p, 8, None, 0, p, 2, 8, float("nan"), bf16, None, p, p, None) == 1
    assert call(norm, p, 8, None, 0, None, 2, 8, 1e-6, bf16, None, p, p, None) == 1
    assert call("mrsa_dequantize_rows_fwd", None, 8, None, 0, 8, bf16, None, None) == 0
    assert call("mrsa_dequantize_rows_fwd", None, 8, None, 4, 0, bf16, None, None) == 0
    assert call("mrsa_dequantize_rows_fwd", p, 8, p, 4, 8, bf16, None, None) == 1
    assert call("mrsa_dequantize_rows_fwd", p, 8, p, 4, 8, fp32, p + 2, None) == 1

    def linear(x=p, xs=64, sx=p, w=p, ws=64, sw=p, bias=None, m=4, n=6, k=64, dtype=bf16,
               space=None, size=0, out=p):
        return call("mrsa_int8_linear_fwd", x, xs, sx, w, ws, sw, bias, m, n, k, dtype, space,
                    size, out, None)

    assert linear(m=0) == 0 and linear(n=0) == 0
    for bad in (dict(m=-1), dict(n=-1), dict(k=-1), dict(xs=-1), dict(ws=-1), dict(x=None),
                dict(w=None), dict(sx=None), dict(sw=None), dict(out=None), dict(sx=p + 2),
                dict(out=p + 1), dict(bias=p + 1), dict(out=p + 2, dtype=fp32)):
        assert linear(**bad) == 1, bad
    for bad in (dict(k=131072), dict(m=1 << 31), dict(n=1 << 31), dict(dtype=3),
                dict(xs=1 << 31), dict(ws=1 << 31), dict(n=(1 << 31) - 1, m=1 << 20)):
        assert linear(**bad) == 2, bad
    # a workspace that is needed
    sizes = (256, 3584, 18944)
    need = call("mrsa_int8_linear_workspace_bytes", *sizes)
    assert need > 0
    m, n, k = sizes
    assert linear(m=m, n=n, k=k, xs=k, ws=k) == 1
    assert linear(m=m, n=n, k=k, xs=k, ws=k, space=p, size=16) == 1
    assert linear(m=m, n=n, k=k, xs=k, ws=k, space=p + 8, size=need) == 1
    # one for copies of rows
    m, n, k = 2000, 2000, 7999
    need = call("mrsa_int8_linear_workspace_bytes", m, n, k)
    assert need >= (m + n) * 8064
    assert linear(m=m, n=n, k=k, xs=k, ws=k) == 1
    assert linear(m=m, n=n, k=k, xs=k, ws=k, space=p, size=need - 1) == 1
    assert call("mrsa_int8_linear_workspace_bytes", -1, 1, 1) == -1
    assert call("mrsa_int8_linear_workspace_bytes", 1, 1, 131072) == -1
    assert call("mrsa_int8_linear_workspace_bytes", 1, 37888, 3584) == 0


@pytest.mark.parametrize("rows", (1, 16, 64, 65, 130, 1003, 16384, 70000))
@pytest.mark.parametrize("out_dim", (1, 64, 1001, 3584, 37888, 152064))
def test_workspaces_stay_small(rows, out_dim):
    for dim in (1, 16, 1003, 3584, 18944, 131071):
        need = _lib.call("mrsa_int8_linear_workspace_bytes", rows, out_dim, dim)
        # partial sums only of as many tiles as the CUs hold at once; copies only of rows that no
        # stride aligns
        copies = (rows + out_dim) * (dim + 127) if dim % 16 and rows > 32 else 0
        assert 0 <= need <= 256 * 256 * 256 * 4 + copies


def test_int8_form_of_a_model_keeps_what_stays():
    shape = DreamShape(layers=2, hidden=64, intermediate=96, q_heads=7, kv_heads=1, vocab=128,
                       interleave=2, mask_token_id=127)
    with FakeTensorMode():
        def layer(route):
            return DreamLayerWeights(
                input_norm=_fake(64), qkv_weight=_fake(9 * 128, 64), qkv_bias=_fake(9 * 128),
                o_weight=_fake(64, 7 * 128), post_norm=_fake(64), gate_up_weight=_fake(192, 64),
                down_weight=_fake(64, 96), qcal_down=_fake(16, 64) if route else None,
                qcal_up=_fake(7 * 128, 16) if route else None)

        w = DreamWeights(shape=shape, embed=_fake(128, 64), lmk_type=_fake(64),
                         final_norm=_fake(64), lm_head=_fake(128, 64),
                         layers=[layer(False), layer(True)])
        w8 = w.int8()
    assert w8.embed is w.embed and w8.lm_head is w.lm_head and w8.final_norm is w.final_norm
    for a, b in zip(w.layers, w8.layers):
        assert b.is_int8 and not a.is_int8
        assert b.input_norm is a.input_norm and b.qkv_bias is a.qkv_bias
        assert b.qkv_weight.values.shape == a.qkv_weight.shape
        assert b.qkv_weight.scales.shape == a.qkv_weight.shape[:1]
        assert b.qcal_up is a.qcal_up
    assert w8.layers[0].qcal_down is None and w8.layers[1].qcal_down.values.dtype == torch.int8
