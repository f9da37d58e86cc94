"""rotary_qk on the GPU against the fp64 oracle, forward and gradient.

Tolerance of one element y = x1 c - x2 s: two fp32 products and a sum round by at
most 2^-24 each relative to |x1 c| + |x2 s| (3 x 2^-24 with the sum's), then the
result to its type, half a step of |y| (finfo.eps / 2) or of the smallest
subnormal."""

import pytest
import torch

import mrsa
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _tolerance(want, magnitude, dtype):
    info = torch.finfo(dtype)
    return (info.eps / 2 * (want.abs() + 4 * 2.0 ** -24 * magnitude) + 4 * 2.0 ** -24 * magnitude
            + info.smallest_normal * info.eps / 2)


def _check(got, x, cos, sin, pos, inter, inverse=False):
    x = x.cpu()
    want = P.rotary(x, cos, sin, pos, inter, inverse)
    tol = _tolerance(want, P.rotary_magnitude(x, cos, sin, pos, inter), x.dtype)
    R = 2 * cos.shape[1]
    err = (got.cpu().double() - want).abs()
    assert torch.equal(got.cpu()[..., R:], x[..., R:])
    assert bool((err <= tol).all()), (float((err - tol).max()), tuple(x.shape))


def _tables(rows, R):
    return mrsa.rotary_tables(rows, mrsa.rotary_frequencies(max(R, 2), 1.0e6)[0][:R // 2],
                              device="cpu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,L,Hq,Hkv,D,R", [
    (1, 1, 1, 1, 128, 128), (1, 32, 28, 4, 128, 128), (2, 7, 8, 8, 64, 32), (3, 5, 16, 1, 128, 64),
    (2, 3, 5, 2, 40, 20), (1, 4, 3, 1, 10, 6), (2, 2, 3, 0, 8, 8), (1, 9, 2, 1, 64, 0),
    (1, 2, 300, 9, 128, 96), (1, 301, 28, 4, 128, 128),
])
def test_rotary_matches_the_oracle(dtype, inter, B, L, Hq, Hkv, D, R):
    g = torch.Generator().manual_seed(B * 100 + L + D + R)
    q = torch.randn(B, L, Hq, D, generator=g).to(dtype)
    k = torch.randn(B, L, Hkv, D, generator=g).to(dtype) if Hkv else None
    cos, sin = _tables(1000, R)
    pos = torch.randint(0, 1000, (B, L), generator=g)
    out_q, out_k = mrsa.rotary_qk(q.to(DEV), None if k is None else k.to(DEV), cos.to(DEV),
                                  sin.to(DEV), pos.to(DEV), interleaved=inter)
    _check(out_q, q, cos, sin, pos, inter)
    if k is None:
        assert out_k is None
    else:
        _check(out_k, k, cos, sin, pos, inter)
    # rows at positions 0 .. L - 1 and one list of positions for every sequence
    row_q, _ = mrsa.rotary_qk(q.to(DEV), None, cos.to(DEV), sin.to(DEV), interleaved=inter)
    _check(row_q, q, cos, sin, None, inter)
    same, _ = mrsa.rotary_qk(q.to(DEV), None, cos.to(DEV), sin.to(DEV), pos[0].to(DEV),
                             interleaved=inter)
    _check(same, q, cos, sin, pos[:1], inter)


def test_many_tokens_take_the_shared_table_path():
    # 256 x 1024 units and more: a thread turns several heads with one table row
    g = torch.Generator().manual_seed(9)
    cos, sin = _tables(1100, 128)
    for Hq, Hkv in ((28, 4), (7, 2)):
        q = torch.randn(1, 1025 * 8, Hq, 128, generator=g).bfloat16().to(DEV)
        k = torch.randn(1, 1025 * 8, Hkv, 128, generator=g).bfloat16().to(DEV)
        pos = torch.randint(0, 1100, (1, 1025 * 8), generator=g).to(DEV)
        out_q, out_k = mrsa.rotary_qk(q, k, cos.to(DEV), sin.to(DEV), pos)
        assert q.shape[1] * (Hq + Hkv) * 8 >= 256 * 1024
        # rows one at a time, as short calls compute them
        for t in (0, 1, 4097, 8199):
            a, b = mrsa.rotary_qk(q[:, t:t + 1], k[:, t:t + 1], cos.to(DEV), sin.to(DEV),
                                  pos[:, t:t + 1])
            assert torch.equal(a, out_q[:, t:t + 1]) and torch.equal(b, out_k[:, t:t + 1])
        _check(out_q[:, :40], q[:, :40], cos, sin, pos[:, :40].cpu(), False)
        _check(out_k[:, -40:], k[:, -40:], cos, sin, pos[:, -40:].cpu(), False)


def test_strides_and_alignment():
    g = torch.Generator().manual_seed(3)
    cos, sin = _tables(50, 64)
    ct, st = cos.to(DEV), sin.to(DEV)
    fused = torch.randn(2, 6, (8 + 2 * 2) * 64, generator=g).bfloat16().to(DEV)
    q = fused[..., :512].view(2, 6, 8, 64)
    k = fused[..., 512:640].view(2, 6, 2, 64)
    cases = [(q, k), (q.transpose(0, 1), k.transpose(0, 1)), (q.flip(1), k.flip(1)),
             (q[:, ::2], k[:, ::2]), (q[:, :1].expand(2, 6, 8, 64), k)]
    shifted = torch.empty(2 * 6 * 8 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(2, 6, 8, 64)
    shifted.copy_(q)                                   # rows 2 bytes off 16-byte alignment
    cases.append((shifted, k))
    apart = torch.randn(2, 6, 8, 128, generator=g).bfloat16().to(DEV)[..., ::2]
    cases.append((apart, k))                           # a last dim that is not dense
    for a, b in cases:
        got, got_k = mrsa.rotary_qk(a, b, ct, st)
        _check(got, a, cos, sin, None, False)
        _check(got_k, b, cos, sin, None, False)
        assert got.is_contiguous() and got_k.is_contiguous()
    # tables and positions that are views
    wide = torch.stack((cos, sin), -1).to(DEV)
    pos = torch.randint(0, 50, (6, 2), generator=g)
    got, _ = mrsa.rotary_qk(q, k, wide[..., 0], wide[..., 1], pos.to(DEV).t())
    _check(got, q, cos, sin, pos.t(), False)


def test_positions_outside_the_tables_give_nan_rows():
    cos, sin = _tables(5, 16)
    x = torch.ones(1, 4, 2, 24, device=DEV)
    pos = torch.tensor([[-1, 4, 5, 1 << 40]], device=DEV)
    for inter in (False, True):
        y, _ = mrsa.rotary_qk(x, None, cos.to(DEV), sin.to(DEV), pos, interleaved=inter)
        assert torch.isnan(y[0, [0, 2, 3], :, :16]).all() and torch.isfinite(y[0, 1]).all()
        assert torch.equal(y[..., 16:], x[..., 16:])


def test_empty_calls():
    cos, sin = (t.to(DEV) for t in _tables(5, 16))
    for B, L, H in ((0, 3, 2), (2, 0, 2), (2, 3, 0)):
        x = torch.empty(B, L, H, 32, device=DEV, dtype=torch.bfloat16)
        q, k = mrsa.rotary_qk(x, x, cos, sin)
        assert q.shape == x.shape and k.shape == x.shape


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
def test_gradient_is_the_transpose(dtype, inter):
    g = torch.Generator().manual_seed(5)
    B, L, Hq, Hkv, D, R = 2, 5, 4, 2, 64, 32
    cos, sin = _tables(100, R)
    ct, st = cos.to(DEV), sin.to(DEV)
    pos = torch.randint(0, 100, (B, L), generator=g)
    q = torch.randn(B, L, Hq, D, generator=g).to(dtype).to(DEV).requires_grad_()
    k = torch.randn(B, L, Hkv, D, generator=g).to(dtype).to(DEV).requires_grad_()
    gq = torch.randn(B, L, Hq, D, generator=g).to(dtype).to(DEV)
    gk = torch.randn(B, L, Hkv, D, generator=g).to(dtype).to(DEV)
    out = mrsa.rotary_qk(q, k, ct, st, pos.to(DEV), interleaved=inter)
    dq, dk = torch.autograd.grad(out, (q, k), (gq, gk))
    _check(dq, gq, cos, sin, pos, inter, inverse=True)
    _check(dk, gk, cos, sin, pos, inter, inverse=True)
    # one output used, one input needing a gradient, a broadcast gradient
    out = mrsa.rotary_qk(q, k, ct, st, pos.to(DEV), interleaved=inter)
    dq, dk = torch.autograd.grad(out[1], (q, k), gk, allow_unused=True)
    assert dq is None
    _check(dk, gk, cos, sin, pos, inter, inverse=True)
    out = mrsa.rotary_qk(q, k.detach(), ct, st, pos.to(DEV), interleaved=inter)
    dq, = torch.autograd.grad(out[0].sum(), q)
    _check(dq, torch.ones_like(gq), cos, sin, pos, inter, inverse=True)
    out = mrsa.rotary_qk(q, None, ct, st, pos.to(DEV), interleaved=inter)
    dq, = torch.autograd.grad(out[0], q, gq)
    _check(dq, gq, cos, sin, pos, inter, inverse=True)


def test_gradient_against_differences_and_of_gradients():
    g = torch.Generator().manual_seed(6)
    cos, sin = _tables(20, 8)
    ct, st = cos.to(DEV), sin.to(DEV)
    x = torch.randn(1, 3, 2, 8, generator=g).to(DEV).requires_grad_()
    w = torch.randn(1, 3, 2, 8, generator=g).to(DEV).requires_grad_()
    y = mrsa.rotary_qk(x, None, ct, st)[0]
    dx, = torch.autograd.grad((y * w).sum(), x, create_graph=True)
    for i in range(x.numel()):
        e = torch.zeros(x.numel(), device=DEV)
        e[i] = 0.5                           # linear: a wide step is exact but for rounding
        hi = mrsa.rotary_qk(x.detach() + e.view(x.shape), None, ct, st)[0]
        lo = mrsa.rotary_qk(x.detach() - e.view(x.shape), None, ct, st)[0]
        slope = float(((hi - lo).double() * w.detach().double()).sum())
        # hi and lo are sums of two products of values up to 5, rounded to fp32
        assert abs(slope - float(dx.reshape(-1)[i])) <= 16 * 2 * 10 * 2.0 ** -24
    # d/dw of <v, dx> is the rotation of v
    v = torch.randn(1, 3, 2, 8, generator=g).to(DEV)
    dw, = torch.autograd.grad((dx * v).sum(), w)
    _check(dw, v, cos, sin, None, False)


def test_dream_rope_is_the_half_layout():
    # the fused projection's rotation, element for element (its products may round elsewhere)
    from mrsa import dream

    g = torch.Generator().manual_seed(7)
    shape = dream.DreamShape()
    qkv = torch.randn(96, 36 * 128, generator=g).bfloat16().to(DEV)
    cos, sin = dream.yarn_tables(96, shape, DEV)
    q, k, v, _ = dream.rope_qkv(qkv, cos, sin, shape)
    heads = qkv.view(1, 96, 36, 128)
    got_q, got_k = mrsa.rotary_qk(heads[:, :, :28], heads[:, :, 28:32], cos, sin)
    for got, fused, x in ((got_q, q, heads[:, :, :28]), (got_k, k, heads[:, :, 28:32])):
        _check(got, x, cos.cpu(), sin.cpu(), None, False)
        _check(fused, x, cos.cpu(), sin.cpu(), None, False)


def test_other_streams_and_replayed_graphs():
    g = torch.Generator().manual_seed(8)
    cos, sin = (t.to(DEV) for t in _tables(64, 128))
    q = torch.randn(2, 9, 28, 128, generator=g).bfloat16().to(DEV)
    k = torch.randn(2, 9, 4, 128, generator=g).bfloat16().to(DEV)
    want = mrsa.rotary_qk(q, k, cos, sin)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mrsa.rotary_qk(q, k, cos, sin)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    pos = torch.arange(9, device=DEV)
    with torch.cuda.graph(graph):
        out = mrsa.rotary_qk(q, k, cos, sin, pos)
    for shift in (0, 5, 40):
        pos.copy_(torch.arange(shift, shift + 9, device=DEV))
        graph.replay()
        want = mrsa.rotary_qk(q, k, cos, sin, pos)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_a_captured_backward_pass():
    g = torch.Generator().manual_seed(9)
    cos, sin = (t.to(DEV) for t in _tables(64, 64))
    q, k, gq, gk = (torch.randn(2, 9, h, 64, generator=g).half().to(DEV) for h in (6, 2, 6, 2))
    q.requires_grad_(), k.requires_grad_()

    def step():
        out = mrsa.rotary_qk(q, k, cos, sin)
        return torch.autograd.grad(out, (q, k), (gq, gk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        gq.copy_(torch.randn(gq.shape, generator=g)), gk.mul_(-2)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_forward_mode(dtype):
    from torch.autograd import forward_ad

    g = torch.Generator().manual_seed(10)
    cos, sin = (t.to(DEV) for t in _tables(16, 32))
    q, tq = torch.randn(2, 2, 9, 6, 64, generator=g).to(dtype).to(DEV)
    k, tk = torch.randn(2, 2, 9, 2, 64, generator=g).to(dtype).to(DEV)
    want = mrsa.rotary_qk(tq, tk, cos, sin, interleaved=True)
    with forward_ad.dual_level():
        out = mrsa.rotary_qk(forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk), cos, sin,
                             interleaved=True)
        got = [forward_ad.unpack_dual(t).tangent for t in out]
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    _, got = torch.func.jvp(lambda a, b: mrsa.rotary_qk(a, b, cos, sin, interleaved=True), (q, k),
                            (tq, tk))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
