"""Linear layers in 8 bits on the GPU against their definitions in 64 bits.

Tolerances, u = 2^-24 (half a step of fp32):
  * 8-bit values: v is the whole number nearest to the fp32 product f * up, where
    up = (1 / top) * 127 is off by 2 u, the product by u and, behind the norm, f = t * w and top
    by u each: |v - 127 y / a| <= 1/2 + 127 * 3 u, 1/2 + 127 * 5 u (norm).  The gated activation:
    exp within 2 steps (4 u), a sum, a quotient and a product: below (1.5 |g| + 8) u of y and as
    much of the top.
  * scales: top / 127 off by u; the norm's also by its mean: a sum of squares along a chain of n
    additions is off by n u, and enters with its square root; six more roundings (the square, the
    mean, eps, rsqrt's 2 u, the two products).
  * sums in int32 are exact; out = fma(fl(fl(sum) sx), sw, bias) is off by 3 u of the product and
    u of the result, then by half a step of the output's type.
"""

import pytest
import torch

import mrsa
from mrsa import _lib
from oracle import int8_oracle as O8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
DIMS = (1, 3, 7, 8, 9, 15, 64, 100, 511, 512, 513, 1001, 1024, 1025, 2047, 2056, 3584, 4096, 4097,
        8192, 8200, 12288, 12289, 18944, 20480, 20481, 30001)


def _rows(rows, dim, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, dim, generator=g, device=DEV) * scale
    return x.to(dtype)


def check_rows(values, scales, y, value_slack, scale_slack):
    """8-bit rows against the real rows y (fp64)."""

    real, scale = O8.quantized(y)
    assert values.dtype == torch.int8 and scales.dtype == torch.float32
    assert values.shape == y.shape and scales.shape == y.shape[:-1]
    off = (values.double() - real).abs()
    bad = off > 0.5 + value_slack
    assert not bad.any(), (bad.nonzero()[:4].tolist(), off.max().item())
    nan = torch.isnan(scale)
    assert torch.equal(torch.isnan(scales), nan)
    err = (scales.double() - scale).abs()[~nan]
    # (2^-149: one step of the smallest numbers)
    assert (err <= scale_slack * scale[~nan] + 2.0 ** -149).all(), (err / scale[~nan]).max().item()
    assert int(values.abs().max()) <= 127 if values.numel() else True


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_quantize_rows(dim, dtype):
    x = _rows(5, dim, dtype, dim)
    values, scales = mrsa.quantize_rows(x)
    check_rows(values, scales, x.double(), 127 * 3 * U, U)
    # the largest magnitude stands for 127
    top = x.double().abs().amax(dim=-1, keepdim=True) == x.double().abs()
    assert (values.abs()[top] == 127).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", (5, 700, 3584, 21000))
def test_quantize_rows_without_a_scale(dim, dtype):
    x = _rows(7, dim, dtype, 3)
    x[0] = 0
    x[1, dim // 2] = float("inf")
    x[2, dim - 1] = float("-inf")
    x[3, 0] = float("nan")
    x[4] = -x[4].abs()
    x[5] = 0
    x[5, dim - 1] = -1.5
    values, scales = mrsa.quantize_rows(x)
    y = x.double()
    check_rows(values, scales, y, 127 * 3 * U, U)
    assert scales[0] == 0 and not values[:4].any() and scales[1:4].isnan().all()
    assert values[5, dim - 1] == -127 and values[5].abs().sum() == 127
    back = mrsa.dequantize_rows(values, scales, dtype)
    assert back[1:4].isnan().all() and not back[0].any()


@pytest.mark.parametrize("value", (3e38, 1e-30, 1e-37, 1e-39, 3e-44))
@pytest.mark.parametrize("dim", (6, 64, 5000))
def test_quantize_rows_at_the_ends_of_fp32(dim, value):
    g = torch.Generator(device=DEV).manual_seed(4)
    x = (torch.rand(3, dim, generator=g, device=DEV) * 2 - 1).float() * value
    x[:, dim - 1] = value
    values, scales = mrsa.quantize_rows(x)
    check_rows(values, scales, x.double(), 127 * 3 * U, U)


def test_rounding_takes_ties_to_even():
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5]], device=DEV)
    values, scales = mrsa.quantize_rows(x)
    assert values[0].tolist() == [127, 0, 2, 2, 0, -2, -2, 126] and scales[0] == 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", (False, True))
@pytest.mark.parametrize("dim", DIMS)
def test_add_rms_norm_int8(dim, residual, dtype):
    x = _rows(5, dim, dtype, dim, 3.0)
    r = _rows(5, dim, dtype, dim + 1) if residual else None
    w = (1 + 0.2 * _rows(1, dim, torch.float32, 7)[0]).to(dtype)
    x[3] = 0
    if residual:
        r[3] = 0
    total, values, scales = mrsa.add_rms_norm_int8(x, r, w, 1e-6)
    t = x
    if residual:
        t = (x.float() + r.float()).to(dtype)
        assert torch.equal(total, t)
    else:
        assert total is None
    y = O8.norm_rows(t.double(), w.double(), 1e-6)
    chain = dim / 64 + 24
    check_rows(values, scales, y, 127 * 5 * U, (chain / 2 + 8) * U)


@pytest.mark.parametrize("dtype,big", [(torch.bfloat16, 2e38), (torch.float32, 3e38),
                                       (torch.bfloat16, 1e20), (torch.float32, 1e-18)])
@pytest.mark.parametrize("dim", (5, 600, 3584, 18944, 21000))
def test_norm_of_values_whose_squares_leave_fp32(dim, dtype, big):
    g = torch.Generator(device=DEV).manual_seed(6)
    x = ((torch.rand(6, dim, generator=g, device=DEV) * 2 - 1).double() * big).to(dtype)
    x[1] = _rows(1, dim, dtype, 5)[0]        # a neighbour of ordinary size
    x[2] = 0
    x[3, dim - 1] = float("inf")
    x[4, 0] = float("nan")
    w = (1 + 0.2 * _rows(1, dim, torch.float32, 7)[0]).to(dtype)
    _, values, scales = mrsa.add_rms_norm_int8(x, None, w, 1e-6)
    y = O8.norm_rows(x.double(), w.double(), 1e-6)
    check_rows(values, scales, y, 127 * 5 * U, ((dim / 64 + 24) / 2 + 8) * U)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_swiglu_int8(dim, dtype):
    x = _rows(5, 2 * dim, dtype, dim, 2.0)
    x[2] = 0
    if dim > 1:
        x[3, 1] = -300.0     # exp passes fp32
    values, scales = mrsa.swiglu_int8(x)
    y = O8.swiglu_rows(x.double())
    # (only magnitudes near the top matter to a value: |g| of the largest product)
    slack = (1.5 * 16 + 8) * U
    assert x[:, :dim].max() <= 16
    check_rows(values, scales, y, 127 * 2 * slack, 2 * slack)


def test_swiglu_int8_not_finite():
    x = _rows(5, 2 * 900, torch.float32, 1)
    x[0, 3] = float("nan")
    x[1, 4] = float("-inf")    # -inf * 0
    x[2, 900 + 5] = float("inf")
    x[3, 6], x[3, 906] = 1e30, 1e30
    values, scales = mrsa.swiglu_int8(x)
    assert scales[:4].isnan().all() and not values[:4].any()
    assert torch.isfinite(scales[4]) and values[4].abs().max() == 127


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 15), (300, 16), (70000, 17), (5, 3584),
                                      (1000, 1001), (2, 70000)])
def test_dequantize_rows(rows, dim, dtype):
    g = torch.Generator(device=DEV).manual_seed(2)
    v = torch.randint(-128, 128, (rows, dim), generator=g, device=DEV).to(torch.int8)
    s = torch.rand(rows, generator=g, device=DEV)
    out = mrsa.dequantize_rows(v, s, dtype)
    exact = v.double() * s.double()[:, None]
    half = torch.finfo(dtype).eps / 2
    assert out.dtype == dtype
    # (2^-25: half a step of fp16's smallest numbers)
    assert ((out.double() - exact).abs() <= exact.abs() * (half + 2 * U) + 2.0 ** -25).all()


def test_rows_of_any_strides():
    wide = _rows(40, 3001, torch.bfloat16, 1)
    for x in (wide[:, 3:1003], wide[::2, :1000], wide[:1].expand(6, 3001), wide.t()[5:50],
              wide[:36, :24].reshape(3, 2, 6, 24).transpose(0, 2), wide[7, 5:900]):
        values, scales = mrsa.quantize_rows(x)
        again = mrsa.quantize_rows(x.contiguous())
        assert values.is_contiguous() and values.shape == x.shape
        assert torch.equal(values, again[0]) and torch.equal(scales, again[1])
        check_rows(values, scales, x.double(), 127 * 3 * U, U)
        w = torch.ones(2 * x.shape[-1], dtype=x.dtype, device=DEV)[::2]
        res = torch.ones_like(x).expand(x.shape)
        got = mrsa.add_rms_norm_int8(x, res, w, 1e-5)
        want = mrsa.add_rms_norm_int8(x.contiguous(), res.contiguous(), w.contiguous(), 1e-5)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        if x.shape[-1] % 2 == 0:
            got, want = mrsa.swiglu_int8(x), mrsa.swiglu_int8(x.contiguous())
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        spread = torch.zeros((*values.shape, 2), dtype=torch.int8, device=DEV)
        spread[..., 0] = values
        back = mrsa.dequantize_rows(spread[..., 0], scales, torch.float32)
        assert torch.equal(back, mrsa.dequantize_rows(values, scales, torch.float32))


def test_no_rows():
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    values, scales = mrsa.quantize_rows(x.reshape(3, 0, 64))
    assert values.shape == (3, 0, 64) and scales.shape == (3, 0)
    assert mrsa.dequantize_rows(values, scales).shape == (3, 0, 64)
    total, values, scales = mrsa.add_rms_norm_int8(x, x, x.new_ones(64), 1e-6)
    assert total.shape == (0, 64) and values.shape == (0, 64)
    assert mrsa.swiglu_int8(x)[0].shape == (0, 32)
    w, sw = torch.ones(5, 64, dtype=torch.int8, device=DEV), torch.ones(5, device=DEV)
    assert mrsa.int8_linear(values, scales, w, sw).shape == (0, 5)
    one = torch.ones(2, 64, dtype=torch.int8, device=DEV)
    assert mrsa.int8_linear(one, one[:, 0].float(), w[:0], sw[:0]).shape == (2, 0)


# ---- the matrix product -----------------------------------------------------------------

def _operands(M, N, K, seed, full=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    lo = -128 if full else -127
    x = torch.randint(lo, 128, (M, K), generator=g, device=DEV).to(torch.int8)
    w = torch.randint(lo, 128, (N, K), generator=g, device=DEV).to(torch.int8)
    sx = torch.rand(M, generator=g, device=DEV) * 0.05 + 1e-3
    sw = torch.rand(N, generator=g, device=DEV) * 1e-3 + 1e-5
    bias = torch.randn(N, generator=g, device=DEV)
    return x, sx, w, sw, bias


def check_linear(out, x, sx, w, sw, bias=None):
    exact, product = O8.linear(x, sx, w, sw, bias)
    assert out.shape == exact.shape
    half = torch.finfo(out.dtype).eps / 2
    bound = (3 * U * product.abs() + U * exact.abs()) * 1.001
    bound = bound + half * (exact.abs() + bound) + 2.0 ** -25
    bad = (out.double() - exact).abs() > bound
    assert not bad.any(), (bad.nonzero()[:4].tolist(), int(bad.sum()))


SHAPES = [(1, 1, 1), (2, 3, 15), (70, 90, 9), (1, 5, 16), (1, 4608, 3584), (3, 17, 16),
          (16, 33, 64), (17, 64, 80), (2, 100, 1003), (32, 3584, 1003), (33, 129, 1000),
          (48, 20, 31), (64, 48, 4096), (64, 1, 18944), (65, 1, 16), (65, 129, 17),
          (100, 300, 48), (128, 128, 64), (129, 257, 1008), (200, 130, 18944), (257, 511, 255),
          (1000, 64, 3584), (517, 1001, 1003), (1, 37888, 3584), (300, 4608, 3584),
          (513, 8192, 1040), (4097, 4097, 16), (4097, 4097, 64), (4090, 4100, 96),
          (4097, 4096, 112), (3900, 4300, 336), (2000, 9000, 1600)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_int8_linear(M, N, K):
    print(f"[gpu-case] int8_linear {M} {N} {K}", flush=True)
    x, sx, w, sw, bias = _operands(M, N, K, M + N + K)
    for dtype in DTYPES:
        check_linear(mrsa.int8_linear(x, sx, w, sw, dtype=dtype), x, sx, w, sw)
        b = bias.to(dtype)
        check_linear(mrsa.int8_linear(x, sx, w, sw, b, dtype=dtype), x, sx, w, sw, b)


@pytest.mark.parametrize("M,N", [(1, 3), (20, 40), (60, 16), (70, 130)])
def test_the_longest_sum_of_the_largest_products(M, N):
    K = 131071
    x = torch.full((M, K), -128, dtype=torch.int8, device=DEV)
    w = x[:1].expand(N, K).contiguous()
    one = torch.ones(max(M, N), device=DEV)
    out = mrsa.int8_linear(x, one[:M], w, one[:N], dtype=torch.float32)
    assert (out.double() == float(torch.tensor(K * 2.0 ** 14).float())).all()
    w[:, 1::2] = 127
    out = mrsa.int8_linear(x, one[:M], w, one[:N], dtype=torch.float32)
    exact = 2 ** 14 * ((K + 1) // 2) - 128 * 127 * (K // 2)
    assert (out.double() == exact).all()


@pytest.mark.parametrize("M,N,K", [(1, 300, 208), (30, 300, 208), (64, 300, 208), (150, 300, 208),
                                   (1500, 1404, 400), (4200, 4100, 80)])
def test_int8_linear_of_any_strides(M, N, K):
    x, sx, w, sw, bias = _operands(M, N, K, 5, full=True)
    want = mrsa.int8_linear(x, sx, w, sw, bias, dtype=torch.float32)
    check_linear(want, x, sx, w, sw, bias)

    def placed(t, left, right, up=0):   # inside wider rows of other values
        big = torch.full((t.shape[0] + up, t.shape[1] + left + right), 77, dtype=torch.int8,
                         device=DEV)
        big[up:, left:left + t.shape[1]] = t
        return big[up:, left:left + t.shape[1]]

    for xs, ws in ((placed(x, 16, 32), w), (x, placed(w, 32, 16, 1)), (placed(x, 3, 0), w),
                   (x, placed(w, 0, 1)), (placed(x, 5, 6), placed(w, 7, 2)),
                   (x.t().contiguous().t(), w.t().contiguous().t())):
        assert torch.equal(mrsa.int8_linear(xs, sx, ws, sw, bias, dtype=torch.float32), want)
    strided = torch.stack((sx, sx), 1)[:, 0], torch.stack((sw, sw), 1)[:, 1]
    double = torch.stack((bias, bias), 1)[:, 1]
    assert torch.equal(mrsa.int8_linear(x, strided[0], w, strided[1], double,
                                        dtype=torch.float32), want)
    if M % 2 == 0:
        got = mrsa.int8_linear(x.reshape(2, M // 2, K), sx.reshape(2, M // 2), w, sw, bias,
                               dtype=torch.float32)
        assert torch.equal(got.reshape(M, N), want)
    one = mrsa.int8_linear(x[0], sx[0], w, sw, bias, dtype=torch.float32)
    assert one.shape == (N,) and torch.equal(one, want[0])
    same = mrsa.int8_linear(x[:1].expand(M, K), sx[:1].expand(M), w, sw, bias, dtype=torch.float32)
    assert torch.equal(same, want[:1].expand(M, N))


@pytest.mark.parametrize("M,N,K", [(65, 3584, 3583), (128, 3584, 3584), (577, 33, 130),
                                   (130, 30, 17), (4100, 20, 100), (193, 40, 2048),
                                   (4194240, 3, 16), (4194305, 3, 16)])
def test_many_rows_of_few_results(M, N, K):
    """Row groups of 64 (at most 65535 of them): the last one's rows, and those behind it."""

    x, sx, w, sw, bias = _operands(M, N, K, 11, full=True)
    out = mrsa.int8_linear(x, sx, w, sw, bias, dtype=torch.float32)
    check_linear(out, x, sx, w, sw, bias)
    part = mrsa.int8_linear(x[-70:], sx[-70:], w, sw, bias, dtype=torch.float32)
    assert torch.equal(out[-70:], part)


@pytest.mark.parametrize("more", range(1, 16))
def test_rows_that_are_copied_to_aligned_ones(more):
    """Lengths that no stride aligns, at sizes where the copies pay: their last bytes, and what
    lies behind the rows."""

    M, N, K = 1301, 1403, 2032 + more
    need = _lib.call("mrsa_int8_linear_workspace_bytes", M, N, K)
    assert need >= (M + N) * 2048   # copied
    x, sx, w, sw, bias = _operands(M, N, K, more, full=True)
    want = mrsa.int8_linear(x, sx, w, sw, bias, dtype=torch.float32)
    check_linear(want, x, sx, w, sw, bias)
    wide = torch.full((M, K + 5 + more), 127, dtype=torch.int8, device=DEV)
    wide[:, 2:K + 2] = x
    heavy = torch.full((N, K + 48 - more), -128, dtype=torch.int8, device=DEV)
    heavy[:, 1:K + 1] = w
    got = mrsa.int8_linear(wide[:, 2:K + 2], sx, heavy[:, 1:K + 1], sw, bias, dtype=torch.float32)
    assert torch.equal(got, want)


@pytest.mark.parametrize("M,N,K", [(3, 70, 96), (40, 70, 96), (200, 70, 96), (1500, 1404, 400),
                                   (256, 512, 9000), (1301, 1403, 2033)])
def test_rows_without_a_scale_stay_alone(M, N, K):
    x, sx, w, sw, bias = _operands(M, N, K, 8)
    sx[1], sx[2] = float("nan"), 0.0
    out = mrsa.int8_linear(x, sx, w, sw, bias, dtype=torch.float32)
    assert out[1].isnan().all() and torch.equal(out[2], bias)
    rest = [i for i in range(M) if i != 1]
    check_linear(out[rest], x[rest], sx[rest], w, sw, bias)


def test_a_linear_layer_of_floats():
    """Activations and a weight matrix made 8-bit and multiplied: within the 8 bits' own error of
    the product in 64 bits.  Every value is off by half a step of its row, so a sum of K products
    by at most K/2 (|x| sw + |w| sx) on each side; here the sum of those bounds itself."""

    x, w = _rows(100, 3584, torch.bfloat16, 1), _rows(256, 3584, torch.bfloat16, 2, 0.02)
    xv, xs = mrsa.quantize_rows(x)
    wv, ws = mrsa.quantize_rows(w)
    out = mrsa.int8_linear(xv, xs, wv, ws, dtype=torch.float32).double()
    exact = x.double() @ w.double().T
    half_x, half_w = 0.5001 * xs.double()[:, None], 0.5001 * ws.double()
    bound = (half_x * w.double().abs().sum(1) + half_w * x.double().abs().sum(1)[:, None]
             + 3584 * half_x * half_w)
    assert ((out - exact).abs() <= bound + 1e-5).all()
    assert float((out - exact).norm() / exact.norm()) < 0.02


# ---- how calls run ----------------------------------------------------------------------

def _chain(x, res, norm_w, gate_up, down, eps=1e-6):
    total, v, s = mrsa.add_rms_norm_int8(x, res, norm_w, eps)
    m = mrsa.int8_linear(v, s, *gate_up)
    v, s = mrsa.swiglu_int8(m)
    return total, mrsa.int8_linear(v, s, *down)


def _chain_operands(rows, hidden=256, inner=704, seed=0):
    x, res = (_rows(rows, hidden, torch.bfloat16, seed + i) for i in (1, 2))
    norm_w = (1 + 0.1 * _rows(1, hidden, torch.float32, 3)[0]).bfloat16()
    gate_up = mrsa.quantize_rows(_rows(2 * inner, hidden, torch.bfloat16, 4, 0.05))
    down = mrsa.quantize_rows(_rows(hidden, inner, torch.bfloat16, 5, 0.05))
    return x, res, norm_w, gate_up, down


@pytest.mark.parametrize("rows", (1, 40, 300))
def test_a_chain_captured_and_replayed(rows):
    x, res, norm_w, gate_up, down = _chain_operands(rows)
    x0, res0 = x.clone(), res.clone()
    _chain(x, res, norm_w, gate_up, down)
    torch.cuda.synchronize()
    graphs, outs = [], []
    pool = torch.cuda.graph_pool_handle()
    for _ in range(2):   # two graphs whose workspaces come from one pool
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            out = _chain(x, res, norm_w, gate_up, down)
        graphs.append(g)
        outs.append(out)
    for i in range(4):
        x.copy_(x0 * (i + 1))
        res.copy_(res0 - i)
        want = _chain(x, res, norm_w, gate_up, down)
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[i % 2], want))


@pytest.mark.parametrize("M,N,K", [(256, 512, 9000), (1301, 1403, 2033), (1003, 3584, 18943)])
def test_products_with_a_workspace_captured_and_replayed(M, N, K):
    """Partial sums, copies of rows, or both, in two graphs of one pool."""

    assert _lib.call("mrsa_int8_linear_workspace_bytes", M, N, K) > 0
    x, sx, w, sw, bias = _operands(M, N, K, 9)
    x0, w0 = x.clone(), w.clone()
    mrsa.int8_linear(x, sx, w, sw, bias, dtype=torch.float32)
    torch.cuda.synchronize()
    graphs, outs = [], []
    pool = torch.cuda.graph_pool_handle()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            out = mrsa.int8_linear(x, sx, w, sw, bias, dtype=torch.float32)
        graphs.append(g)
        outs.append(out)
    for i in range(4):
        x.copy_(x0.roll(i, 0))
        w.copy_(w0.roll(i, 1))
        want = mrsa.int8_linear(x, sx, w, sw, bias, dtype=torch.float32)
        if i == 0:
            check_linear(want, x, sx, w, sw, bias)
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want)


def test_products_with_a_workspace_on_other_streams():
    ops = [_operands(*s, 3) for s in ((256, 512, 9000), (1301, 1403, 2033), (257, 511, 9001))]
    want = [mrsa.int8_linear(*o, dtype=torch.float32) for o in ops]
    torch.cuda.synchronize()
    got = []
    for o, st in zip(ops, [torch.cuda.Stream() for _ in ops]):
        with torch.cuda.stream(st):
            for _ in range(5):
                out = mrsa.int8_linear(*o, dtype=torch.float32)
            got.append(out)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_on_other_streams():
    ops = [_chain_operands(rows, seed=rows) for rows in (200, 131, 33)]
    want = [_chain(*o) for o in ops]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ops]
    got = []
    for o, st in zip(ops, streams):
        with torch.cuda.stream(st):
            for _ in range(5):
                out = _chain(*o)
            got.append(out)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_compiled_chain_gives_the_same_bits():
    x, res, norm_w, gate_up, down = _chain_operands(70)
    want = _chain(x, res, norm_w, gate_up, down)
    traced = torch.compile(_chain, fullgraph=True, backend="aot_eager")
    got = traced(x, res, norm_w, gate_up, down)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_direct_calls_refuse_tangents():
    """What a compiler has traced reaches the operators past the public functions."""

    from torch.autograd import forward_ad

    x = torch.zeros(4, 32, device=DEV)
    v, s = mrsa.quantize_rows(x)
    ops = torch.ops.mrsa
    with forward_ad.dual_level(), torch.no_grad():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        ds = forward_ad.make_dual(s, torch.ones_like(s))
        for call in (lambda: ops.quantize_rows(dual), lambda: ops.swiglu_int8(dual),
                     lambda: ops.add_rms_norm_int8(x, dual, x[0], 1e-6),
                     lambda: ops.add_rms_norm_int8(dual, None, x[0], 1e-6),
                     lambda: ops.add_rms_norm_int8(x, None, dual[0], 1e-6),
                     lambda: ops.dequantize_rows(v, ds, torch.float32),
                     lambda: ops.int8_linear(v, ds, v, s, None, torch.float32),
                     lambda: ops.int8_linear(v, s, v, ds, None, torch.float32),
                     lambda: ops.int8_linear(v, s, v, s, ds, torch.float32)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        ops.quantize_rows(x)


def test_direct_calls_map_errors_as_the_others():
    """The C entry points' checks behind the operators: ValueError, as through ctypes."""

    x = torch.zeros(4, 32, device=DEV)
    v, s = mrsa.quantize_rows(x)
    ops = torch.ops.mrsa
    with pytest.raises(ValueError):
        ops.add_rms_norm_int8(x, None, x[0].contiguous(), 0.0)
    with pytest.raises(ValueError):
        ops.quantize_rows(x.double())
    with pytest.raises(ValueError):
        ops.dequantize_rows(v, s, torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.quantize_rows(x.cpu())


def test_calls_that_ask_for_a_derivative():
    """Refused on the GPU as for fake tensors; without gradients the same tensors pass."""

    x = torch.ones(4, 32, device=DEV).requires_grad_()
    v, s = mrsa.quantize_rows(x.detach())
    s.requires_grad_()
    for call in (lambda: mrsa.quantize_rows(x), lambda: mrsa.swiglu_int8(x),
                 lambda: mrsa.add_rms_norm_int8(x, None, x[0].detach(), 1e-6),
                 lambda: mrsa.add_rms_norm_int8(x.detach(), x, x[0].detach(), 1e-6),
                 lambda: mrsa.add_rms_norm_int8(x.detach(), None, x[0], 1e-6),
                 lambda: mrsa.dequantize_rows(v, s),
                 lambda: mrsa.int8_linear(v, s, v, s.detach()),
                 lambda: mrsa.int8_linear(v, s.detach(), v, s),
                 lambda: mrsa.int8_linear(v, s.detach(), v, s.detach(), s, dtype=torch.float32)):
        with pytest.raises(ValueError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    with torch.no_grad(), pytest.raises(Exception, match="forward-mode"):
        torch.func.jvp(lambda t: mrsa.quantize_rows(t)[1], (x.detach(),), (torch.ones_like(x),))


def test_refusals_of_real_tensors():
    """The words of the fake tensors' refusals (tests/test_int8_linear.py)."""

    x = torch.zeros(4, 32, device=DEV)
    v, s = mrsa.quantize_rows(x)
    for call, words in (
            (lambda: mrsa.quantize_rows(x.cpu()), "CUDA"),
            (lambda: mrsa.quantize_rows(x.double()), "bf16, fp16 or fp32"),
            (lambda: mrsa.quantize_rows(x[0, 0]), "at least one"),
            (lambda: mrsa.quantize_rows(x[:, :0]), "at least one"),
            (lambda: mrsa.swiglu_int8(x[:, :7]), "even"),
            (lambda: mrsa.add_rms_norm_int8(x, x[:3], x[0], 1e-6), "residual"),
            (lambda: mrsa.add_rms_norm_int8(x, x.cpu(), x[0], 1e-6), "residual"),
            (lambda: mrsa.add_rms_norm_int8(x, None, x[:1], 1e-6), "weight"),
            (lambda: mrsa.add_rms_norm_int8(x, None, x[0].half(), 1e-6), "weight"),
            (lambda: mrsa.add_rms_norm_int8(x, None, x[0], float("nan")), "eps"),
            (lambda: mrsa.dequantize_rows(x, s), "int8"),
            (lambda: mrsa.dequantize_rows(v, s[:, None]), "scales"),
            (lambda: mrsa.dequantize_rows(v, s.cpu()), "one device"),
            (lambda: mrsa.dequantize_rows(v, s, torch.int32), "dtype"),
            (lambda: mrsa.dequantize_rows(v[:, :0], s), "at least one"),
            (lambda: mrsa.int8_linear(v, s, v[:, :31], s), "weight"),
            (lambda: mrsa.int8_linear(v, s, v[None], s[None]), "weight"),
            (lambda: mrsa.int8_linear(v, s, x, s), "int8"),
            (lambda: mrsa.int8_linear(v, s[:3], v, s), "scales"),
            (lambda: mrsa.int8_linear(v, s, v, s, s), "bias"),
            (lambda: mrsa.int8_linear(v, s, v, s, dtype=torch.int8), "dtype"),
            (lambda: mrsa.int8_linear(v[:, :0], s, v[:, :0], s), "131071")):
        with pytest.raises(ValueError, match=words):
            call()


def test_direct_calls_refuse_what_would_pass_their_memory():
    x = torch.zeros(4, 32, device=DEV)
    v, s = mrsa.quantize_rows(x)
    ops = torch.ops.mrsa
    f32, bf16 = torch.float32, torch.bfloat16
    for call in (lambda: ops.dequantize_rows(v, s[:3], f32),
                 lambda: ops.dequantize_rows(v, s.double(), f32),
                 lambda: ops.dequantize_rows(v, s.cpu(), f32),
                 lambda: ops.dequantize_rows(x, s, f32),
                 lambda: ops.dequantize_rows(v.cpu(), s, f32),
                 lambda: ops.add_rms_norm_int8(x.cpu(), x, x[0], 1e-6),
                 lambda: ops.int8_linear(v.cpu(), s, v, s, None, f32),
                 lambda: ops.add_rms_norm_int8(x, None, x[0, :31], 1e-6),
                 lambda: ops.add_rms_norm_int8(x, None, x[0].bfloat16(), 1e-6),
                 lambda: ops.add_rms_norm_int8(x, x[:3], x[0], 1e-6),
                 lambda: ops.add_rms_norm_int8(x, x.view(8, 16), x[0], 1e-6),
                 lambda: ops.add_rms_norm_int8(x, x.bfloat16(), x[0], 1e-6),
                 lambda: ops.swiglu_int8(x[:, :31]),
                 lambda: ops.int8_linear(v, s[:3], v, s, None, f32),
                 lambda: ops.int8_linear(v, s, v, s[:3], None, f32),
                 lambda: ops.int8_linear(v, s, v[:, :16], s, None, f32),
                 lambda: ops.int8_linear(v, s, v.float(), s, None, f32),
                 lambda: ops.int8_linear(x, s, v, s, None, f32),
                 lambda: ops.int8_linear(v, s, v.cpu(), s, None, f32),
                 lambda: ops.int8_linear(v, s, v, s, x[0, :3], f32),
                 lambda: ops.int8_linear(v, s, v, s, x[0, :4], bf16)):
        with pytest.raises((ValueError, NotImplementedError)):
            call()


def test_offsets_past_32_bits():
    """The last rows of matrices of more than 2^32 elements."""

    K, rows = 16384, (1 << 32) // 16384 + 40
    w = torch.empty(rows, K, dtype=torch.int8, device=DEV)
    w[-40:] = _operands(40, 1, K, 3)[0]
    x, sx, _, _, _ = _operands(8, 1, K, 4)
    sw = torch.full((rows,), 1e-3, device=DEV)
    out = mrsa.int8_linear(x, sx, w[rows - 40 - 600:], sw[:640])
    check_linear(out[:, -40:], x, sx, w[-40:], sw[:40])
    out = mrsa.int8_linear(w, sw, x, sx)     # as activations: 2^18 rows
    check_linear(out[-40:], w[-40:], sw[:40], x, sx)
    del w
    f = torch.zeros(rows, K, dtype=torch.bfloat16, device=DEV)
    f[-3:] = _rows(3, K, torch.bfloat16, 9)
    values, scales = mrsa.quantize_rows(f)
    check_rows(values[-3:], scales[-3:], f[-3:].double(), 127 * 3 * U, U)
    back = mrsa.dequantize_rows(values, scales)
    assert torch.equal(back[-3:], (values[-3:].float() * scales[-3:, None]).bfloat16())
