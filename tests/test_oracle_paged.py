"""The rotary and paged-cache oracle against closed forms and torch's own ops."""

import math

import pytest
import torch

import mrsa
from mrsa import dream
from oracle import paged_oracle as P


def test_rotary_is_a_complex_product_and_its_transpose_the_inverse():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 5, 3, 8, generator=g, dtype=torch.float64)
    cos, sin = mrsa.rotary_tables(9, mrsa.rotary_frequencies(6)[0], device="cpu")
    pos = torch.randint(0, 9, (2, 5), generator=g)
    y = P.rotary(x, cos, sin, pos, interleaved=True)
    z = torch.view_as_complex(x[..., :6].reshape(2, 5, 3, 3, 2))
    w = torch.complex(cos.double(), sin.double())[pos][:, :, None]
    assert torch.allclose(torch.view_as_real(z * w).reshape(2, 5, 3, 6), y[..., :6], atol=1e-14)
    assert torch.equal(y[..., 6:], x[..., 6:])
    # the half layout is the interleaved one with its dims in another order
    order = [0, 2, 4, 1, 3, 5, 6, 7]
    half = P.rotary(x[..., order], cos, sin, pos)
    assert torch.allclose(half, y[..., order], atol=1e-14)
    for inter in (False, True):
        leaf = x.clone().requires_grad_()
        grad = torch.randn(x.shape, generator=g, dtype=torch.float64)
        (P.rotary(leaf, cos, sin, pos, inter) * grad).sum().backward()
        assert torch.allclose(leaf.grad, P.rotary(grad, cos, sin, pos, inter, inverse=True),
                              atol=1e-13)


def test_rotary_positions_outside_the_tables_are_nan():
    x = torch.ones(1, 3, 1, 4)
    cos, sin = torch.ones(5, 1), torch.zeros(5, 1)
    y = P.rotary(x, cos, sin, torch.tensor([[-1, 4, 5]]))
    assert torch.isnan(y[0, 0, 0, :2]).all() and torch.isnan(y[0, 2, 0, :2]).all()
    assert torch.equal(y[0, 1], x[0, 1].double()) and torch.equal(y[0, 0, 0, 2:],
                                                                  x[0, 0, 0, 2:].double())


def test_frequencies_of_each_scaling():
    R, base = 64, 1.0e6
    plain, one = mrsa.rotary_frequencies(R, base)
    assert one == 1.0
    assert torch.allclose(plain, torch.tensor([base ** (-2 * i / R) for i in range(R // 2)],
                                              dtype=torch.float64), rtol=1e-14)
    linear, _ = mrsa.rotary_frequencies(R, base, "linear", 4.0)
    assert torch.allclose(linear * 4, plain, rtol=1e-15)
    ntk, _ = mrsa.rotary_frequencies(R, base, "ntk", 4.0)
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]) * 4, float(plain[-1]), rel_tol=1e-12)
    shape = dream.DreamShape()
    want, factor = dream.yarn_inv_freq(shape)
    got, f2 = mrsa.rotary_frequencies(128, shape.rope_theta, "yarn", shape.yarn_factor,
                                      shape.yarn_original_max)
    assert f2 == factor
    # (dream's are these, rounded to fp32)
    assert torch.equal(got.float(), want)


def test_tables_of_far_positions_keep_their_angles():
    inv, _ = mrsa.rotary_frequencies(4, 10000.0)
    cos, sin = mrsa.rotary_tables(200001, inv, device="cpu")
    # half a step of fp32 around the true value
    assert abs(float(cos[200000, 0]) - math.cos(200000.0)) <= 2 ** -24
    assert abs(float(sin[131071, 1]) - math.sin(131071.0 / 100.0)) <= 2 ** -24


@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (False, 3), (True, 2)])
def test_attention_against_a_dense_softmax(causal, window):
    g = torch.Generator().manual_seed(2)
    n, Lq, Hq, Hkv, D, page = 21, 4, 6, 2, 8, 4
    k, v = (torch.randn(n, Hkv, D, generator=g) for _ in range(2))
    q = torch.randn(1, Lq, Hq, D, generator=g)
    order = torch.randperm(9, generator=g)[:6]
    kp, vp = torch.full((2, 9, page, Hkv, D), float("nan"))
    for j in range(n):
        kp[order[j // page], j % page] = k[j]
        vp[order[j // page], j % page] = v[j]
    out, lse, _, _ = P.attention(q, kp, vp, order[None], torch.tensor([n]), None, causal, window)
    j, p = torch.arange(n)[None], torch.arange(n - Lq, n)[:, None]
    mask = torch.zeros(Lq, n, dtype=torch.float64)
    if causal:
        mask = mask.masked_fill(j > p, float("-inf"))
    if window is not None:
        mask = mask.masked_fill((j - p).abs() > window, float("-inf"))
    qh = q[0].double().transpose(0, 1)
    kh = k.double().repeat_interleave(Hq // Hkv, 1).transpose(0, 1)
    vh = v.double().repeat_interleave(Hq // Hkv, 1).transpose(0, 1)
    s = qh @ kh.transpose(1, 2) * D ** -0.5 + mask
    assert torch.allclose(out[0], (torch.softmax(s, -1) @ vh).transpose(0, 1), atol=1e-12)
    assert torch.allclose(lse[0], torch.logsumexp(s, -1).transpose(0, 1), atol=1e-12)


def test_padding_unmapped_pages_and_empty_sequences_see_nothing():
    q = torch.ones(3, 2, 1, 8)
    pages = torch.ones(2, 4, 1, 8)
    table = torch.tensor([[0, 1], [-1, 9], [0, 1]])
    out, lse, _, _ = P.attention(q, pages, pages, table, torch.tensor([1, 8, 0]))
    assert torch.isinf(lse[0, 0]).all() and torch.isfinite(lse[0, 1]).all()
    assert torch.equal(out[0, 1], torch.ones(1, 8, dtype=torch.float64))
    assert torch.isinf(lse[1:]).all() and not out[1:].any()
