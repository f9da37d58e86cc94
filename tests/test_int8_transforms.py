"""The 8-bit operators under torch.func's transforms, on fake tensors: what asks for a derivative is
refused in every nesting (a gradient of zeros never comes back), vmap alone passes."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.func import functional_call, grad, hessian, jacfwd, jacrev, jvp, vjp, vmap

import mrsa


def _operands():
    def fake(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    return fake(4, 8), fake(8), fake(4, 8, dtype=torch.int8), fake(4)


# of each differentiable operand of each operator: (which, a function of it)
def _functions(ops, x, w, v, s):
    linear = lambda a, b, c: ops.int8_linear(v, a, v, b, c, **ops.f32)  # noqa: E731
    norm = lambda a, b, c: ops.add_rms_norm_int8(a, b, c, 1e-6)         # noqa: E731
    return {
        "quantize x": (x, lambda t: ops.quantize_rows(t)[1]),
        "dequantize scales": (s, lambda t: ops.dequantize_rows(v, t, torch.float32)),
        "norm x, its sum": (x, lambda t: norm(t, x, w)[0]),
        "norm x": (x, lambda t: norm(t, None, w)[2]),
        "norm residual": (x, lambda t: norm(x, t, w)[0]),
        "norm weight": (w, lambda t: norm(x, None, t)[2]),
        "swiglu": (x, lambda t: ops.swiglu_int8(t)[1]),
        "linear x scales": (s, lambda t: linear(t, s, None)),
        "linear weight scales": (s, lambda t: linear(s, t, None)),
        "linear bias": (s, lambda t: linear(s, s, t)),
    }


class _Public:
    f32 = {"dtype": torch.float32}

    def __getattr__(self, name):
        return getattr(mrsa, name)


class _Direct:   # as a compiler's traces call them
    f32 = {"dtype": torch.float32}

    def __getattr__(self, name):
        return getattr(torch.ops.mrsa, name)


NAMES = tuple(_functions(_Public(), None, None, None, None))


@pytest.mark.parametrize("ops", (_Public(), _Direct()), ids=("public", "direct"))
@pytest.mark.parametrize("name", NAMES)
def test_derivatives_are_refused(name, ops):
    with FakeTensorMode():
        t, f = _functions(ops, *_operands())[name]
        total = lambda t: f(t).sum()   # noqa: E731
        for call in (lambda: grad(total)(t), lambda: vjp(f, t), lambda: jacrev(f)(t),
                     lambda: hessian(total)(t), lambda: grad(lambda a: grad(total)(a).sum())(t)):
            with pytest.raises(ValueError, match="no gradient|forward-mode"):
                call()
        for call in (lambda: jvp(f, (t,), (t,)), lambda: jacfwd(f)(t)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()


def test_derivatives_of_and_in_vmap_are_refused():
    with FakeTensorMode():
        x, w, v, s = _operands()
        rows = lambda r: mrsa.quantize_rows(r)[1]   # noqa: E731
        for call in (lambda: grad(lambda a: vmap(rows)(a).sum())(x), lambda: vmap(grad(rows))(x),
                     lambda: vmap(grad(lambda b: mrsa.int8_linear(
                         v, s, v, s, b, dtype=torch.float32).sum()))(torch.stack((s, s)))):
            with pytest.raises(ValueError, match="no gradient"):
                call()
        assert vmap(rows)(x).shape == (4,)


class _Layer(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.bias = torch.nn.Parameter(torch.empty(4, device="cuda"))

    def forward(self, v, s):
        return mrsa.int8_linear(v, s, v, s, self.bias, dtype=torch.float32)


def test_a_module_s_gradient_is_refused():
    with FakeTensorMode():
        _, _, v, s = _operands()
        layer = _Layer()
        with pytest.raises(ValueError, match="no gradient"):
            grad(lambda p: functional_call(layer, p, (v, s)).sum())(dict(layer.named_parameters()))
