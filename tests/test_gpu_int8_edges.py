"""8-bit rows at the ends of their inputs' range, against their definitions in 64 bits.

Tolerances as in tests/test_gpu_int8_linear.py, u = 2^-24 (half a step of fp32).  A gate g below
-87, whose exp(-g) nears the end of fp32, gives ((g h) up) h with h = exp(g / 2): h twice, within 2
steps (4 u) each, and three products: 11 u of y, and half of the smallest step, 2^-150, where y is
that small.  Both count twice for a value: in y and in the row's top.
"""

import pytest
import torch

import mrsa
from oracle import int8_oracle as O8
from test_gpu_int8_linear import DEV, DTYPES, U, _rows, check_rows

pytestmark = pytest.mark.gpu
DIMS = (6, 9, 700, 1001, 3584, 18944, 21000)


def check_swiglu(x, slack):
    values, scales = mrsa.swiglu_int8(x)
    y = O8.swiglu_rows(x.double())
    for i in range(x.shape[0]):
        top = float(y[i].abs().max())
        small = 0.0 if top == 0 else 2.0 ** -149 * 127 / top
        check_rows(values[i], scales[i], y[i], 127 * 2 * slack + small, 2 * slack)
    return values, scales


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_swiglu_int8_of_masked_gates(dim, dtype):
    """Gates of the type's lowest value among ordinary ones are zeros."""

    x = _rows(6, 2 * dim, dtype, dim, 2.0)
    assert x[:, :dim].max() <= 16
    low = torch.finfo(dtype).min
    x[1, dim - 1] = low
    x[2, ::2] = low         # (the other factor, too: of ordinary and of masked gates)
    x[2, dim:] = 1.0
    x[3, : dim // 2] = low
    x[4, 0], x[4, dim] = low, 1e4
    x[5, 1], x[5, dim + 1] = -1e4, -1e4
    values, _ = check_swiglu(x, (1.5 * 16 + 8) * U)
    assert not values[2, ::2][: dim // 2].any() and not values[3, : dim // 2].any()
    assert values[4, 0] == 0 and values[5, 1] == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_swiglu_int8_of_gates_that_are_all_very_negative(dim, dtype):
    g = torch.Generator(device=DEV).manual_seed(dim)
    big = 6e4 if dtype == torch.float16 else 1e20
    gate = torch.rand(8, dim, generator=g, device=DEV) * 33 - 120        # -120 .. -87
    gate[1], gate[2], gate[3], gate[4] = -88.0, -100.0, -87.0, -110.0
    gate[5] = torch.rand(dim, generator=g, device=DEV) * 4 - 89          # on both sides of -87
    gate[6] = torch.rand(dim, generator=g, device=DEV) * 10 - 100
    up = torch.rand(8, dim, generator=g, device=DEV) * 2 - 1
    up[:6] *= big                                      # (the others: near the smallest numbers)
    x = torch.cat((gate, up), dim=1).to(dtype)
    # (gates above -87 as others: 1.5 |g| + 8; below: 11)
    values, scales = check_swiglu(x, (1.5 * 89 + 8) * U)
    assert (values.abs().amax(dim=1) == 127).all() and (scales > 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_swiglu_int8_of_gates_that_leave_nothing(dim, dtype):
    low = torch.finfo(dtype).min
    gates = [-1e3, -1e4, low] + ([] if dtype == torch.float16 else [-1e30])
    x = torch.ones(len(gates) + 1, 2 * dim, dtype=dtype, device=DEV) * 1e4
    for i, g in enumerate(gates):
        x[i, :dim] = g
    x[-1, :dim] = low
    x[-1, dim // 2] = float("-inf")                    # -inf * 0
    values, scales = mrsa.swiglu_int8(x)
    assert not values.any() and not scales[:-1].any() and scales[-1].isnan()


def test_transforms_of_real_tensors():
    """Derivatives by torch.func are refused (tests/test_int8_transforms.py has all of them); of
    other tensors, beside the operators, they are right; vmap alone gives the rows' own results."""

    from torch.func import grad, jacrev, jvp, vmap

    x, w = _rows(4, 32, torch.float32, 1), _rows(1, 32, torch.float32, 2)[0]
    v, s = mrsa.quantize_rows(x)
    product = lambda b: mrsa.int8_linear(v, s, v, s, b, dtype=torch.float32)   # noqa: E731
    for call in (lambda: grad(lambda b: product(b).sum())(s), lambda: jacrev(product)(s),
                 lambda: grad(lambda t: mrsa.add_rms_norm_int8(t, x, w, 1e-6)[0].sum())(x),
                 lambda: grad(lambda t: torch.ops.mrsa.quantize_rows(t)[1].sum())(x),
                 lambda: vmap(grad(lambda t: mrsa.swiglu_int8(t)[1]))(x),
                 lambda: grad(lambda t: vmap(lambda r: mrsa.quantize_rows(r)[1])(t).sum())(x),
                 lambda: jvp(lambda t: mrsa.dequantize_rows(v, t), (s,), (s,)),
                 lambda: jvp(lambda t: torch.ops.mrsa.quantize_rows(t)[1], (x,), (x,))):
        with pytest.raises(ValueError, match="no gradient|forward-mode"):
            call()

    def beside(b):
        with torch.no_grad():
            rows = mrsa.quantize_rows(b[:, None] * x)[1]
        return (rows * b * mrsa.quantize_rows(x)[1] * mrsa.swiglu_int8(b.detach()[:, None] * x)[1]
                ).sum()

    b = torch.tensor([1.0, 2.0, 0.5, 3.0], device=DEV)
    rows = b[:, None] * x
    want = mrsa.quantize_rows(rows)[1] * mrsa.quantize_rows(x)[1] * mrsa.swiglu_int8(rows)[1]
    torch.testing.assert_close(grad(beside)(b), want, rtol=4 * U, atol=0.0)
    batch = torch.stack((x, 2 * x, x.flip(0)))
    for got, one in zip(vmap(mrsa.quantize_rows)(batch), zip(*map(mrsa.quantize_rows, batch))):
        assert torch.equal(got, torch.stack(one))


def test_gradients_of_a_graph_around_the_operators():
    """Ordinary autograd: what runs under no_grad inside a recorded graph stays a constant of it."""

    x = _rows(4, 32, torch.float32, 3).requires_grad_()
    with torch.no_grad():
        v, s = mrsa.quantize_rows(x)
        back = mrsa.dequantize_rows(v, s, torch.float32)
    (x * back).sum().backward()
    assert torch.equal(x.grad, back)
    with torch.inference_mode():
        again = mrsa.quantize_rows(x)
    assert torch.equal(again[0], v) and torch.equal(again[1], s)


@pytest.mark.parametrize("rows,dim", [((1 << 22) + 5, 9), ((1 << 22) + 5, 3),
                                      ((1 << 20) + 3, 1025)])
def test_more_rows_than_blocks(rows, dim):
    """Blocks that take several rows each (rows that fit a wave: four a block)."""

    x = _rows(257, dim, torch.bfloat16, dim)
    x = x.repeat(rows // 257 + 1, 1)[:rows]
    n = torch.arange(rows, device=DEV) % 257
    for call in (mrsa.quantize_rows,
                 lambda t: mrsa.add_rms_norm_int8(t, None, torch.ones_like(t[0]), 1e-6)[1:],
                 lambda t: mrsa.swiglu_int8(t[:, : dim // 2 * 2])):
        values, scales = call(x)
        first, its = call(x[:257])
        assert torch.equal(values, first[n]) and torch.equal(scales, its[n])
    values, scales = mrsa.quantize_rows(x)
    check_rows(values[:257], scales[:257], x[:257].double(), 127 * 3 * U, U)
    back = mrsa.dequantize_rows(values, scales)
    assert torch.equal(back, (values.float() * scales[:, None]).bfloat16())


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("dim", DIMS)
def test_norm_beside_weights_near_the_end_of_fp32(dim, dtype):
    """t * weight leaves fp32 where the normed t times the weight does not (rows 0 and 1), or the
    other way round (row 2: counted as infinite); ordinary rows beside them."""

    x = torch.where(_rows(6, dim, torch.float32, dim) < 0, -1.9, 1.9)
    x[0] *= 64.0
    x[1] *= 2.0 ** 126
    x[2] = 0.0
    x[2, dim // 2] = 0.5
    x[3:] = 0.0                                # small weights alone meet these
    x[3:, :2] = _rows(3, 2, torch.float32, 9)
    g = torch.Generator(device=DEV).manual_seed(dim)
    w = (torch.rand(dim, generator=g, device=DEV) * 2 - 1) * 2.5e38
    w[:2] = 1.0
    w[dim // 2] = 2.5e38
    x, w = x.to(dtype), w.to(dtype)
    total, values, scales = mrsa.add_rms_norm_int8(x, None, w, 1e-6)
    y = O8.norm_rows(x.double(), w.double(), 1e-6)
    assert y[:2].abs().max() < 3e38 and y[2].abs().max() > 3.5e38
    assert scales[2].isnan() and not values[2].any()
    rest = [0, 1, 3, 4, 5]
    check_rows(values[rest], scales[rest], y[rest], 127 * 5 * U, ((dim / 64 + 24) / 2 + 8) * U)
    assert (values[rest].abs().amax(dim=1) == 127).all()


@pytest.mark.parametrize("dim", DIMS)
def test_rows_of_the_largest_numbers_come_back_finite(dim):
    """top / 127 may round up, and 127 of it past fp32: the scale is then one step (2 u) less."""

    x = _rows(4, dim, torch.float32, dim)
    most = torch.finfo(torch.float32).max
    x[0, dim - 1], x[1, 0] = most, -most
    x[2] = most
    gated = torch.cat((x, torch.ones_like(x)), dim=1)      # silu(most) is most
    ones = torch.ones(dim, device=DEV)
    heavy = torch.where(torch.arange(dim, device=DEV) % 2 == 0, most, 1.0)
    for y, (values, scales) in ((x, mrsa.quantize_rows(x)), (None, mrsa.swiglu_int8(gated)),
                                (None, mrsa.add_rms_norm_int8(ones[None], None, heavy, 1e-24)[1:])):
        if y is not None:
            check_rows(values, scales, y.double(), 127 * 3 * U, 2 * U)
        back = mrsa.dequantize_rows(values, scales, torch.float32)
        assert torch.isfinite(back).all() and torch.isfinite(scales).all()
        assert back[0].abs().max() > 0.999 * most and values[0].abs().max() == 127


def test_product_of_rows_that_lie_gigabytes_apart():
    K, apart = 144, (1 << 31) + 16
    memory = torch.empty(2 * apart + K, dtype=torch.int8, device=DEV)
    far = memory.as_strided((3, K), (apart, 1))
    near = torch.randint(-127, 128, (3, K), device=DEV).to(torch.int8)
    far.copy_(near)
    s, many = torch.rand(3, device=DEV), torch.randint(-127, 128, (70, K), device=DEV)
    many, its = many.to(torch.int8), torch.rand(70, device=DEV)
    for got, want in ((mrsa.int8_linear(far, s, many, its), mrsa.int8_linear(near, s, many, its)),
                      (mrsa.int8_linear(many, its, far, s), mrsa.int8_linear(many, its, near, s))):
        assert torch.equal(got, want)
    assert torch.equal(mrsa.dequantize_rows(far, s), mrsa.dequantize_rows(near, s))
