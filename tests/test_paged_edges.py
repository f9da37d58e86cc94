"""The paged operators and rotary_qk at their edges, without a GPU: what the C entry points
refuse, and what the operators' own Python code does around a kernel (a stand-in here)."""

import ctypes

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad

import mrsa
from mrsa import _lib, paged_cache, rotary


def test_c_append_without_kv_heads_still_needs_its_table():
    s = (512, 512, 128)
    status = _lib.call("mrsa_paged_append_fwd", 4096, *s, None, 0, 0, 0, None, 0, 0, 0, None, None,
                       0, None, 0, 0, 4096, 1, 1, None, 4, 4, 7, 16, None, *s, None, *s, 1, 1, 4, 0,
                       128, 0, 0, 0, 4096, None)
    assert status == _lib.MRSA_ERR_INVALID_ARGUMENT


def test_c_workspace_sizes_do_not_wrap():
    def size(*args):
        return _lib.call("mrsa_paged_attention_workspace_bytes", *args)

    for batch, q_len, heads in ((1 << 9, 1 << 31, 1), (1 << 24, 1, 1 << 16), (1 << 7, 1 << 31, 1),
                                (1 << 6, 1 << 31, 2), (3, 1000003, 7)):
        for head_dim in (64, 128, 4096):
            for parts in (2, 1024):
                want = batch * q_len * heads * parts * (head_dim + 2) * 4
                assert size(batch, q_len, heads, head_dim, parts) in (
                    (want, -1) if want < 1 << 63 else (-1,))
    assert size(3, 1000003, 7, 128, 1024) == 3 * 1000003 * 7 * 1024 * 130 * 4


def _plain_rotary(q, qb, ql, qh, k, kb, kl, kh, cos, sin, rows, pos, pb, pl, B, L, Hq, Hkv, D, R,
                  dtype, interleaved, inverse, q_out, k_out, stream):
    """mrsa_rotary_fwd of fp32 host memory (half layout, every position given by its row)."""

    def array(at, shape, strides):
        size = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
        flat = np.ctypeslib.as_array((ctypes.c_float * size).from_address(at))
        return np.lib.stride_tricks.as_strided(flat, shape, [4 * s for s in strides])

    assert dtype == 2 and not interleaved and pos is None
    h = R // 2
    c = array(cos, (L, h), (h, 1))[:, None]
    s = array(sin, (L, h), (h, 1))[:, None] * (-1 if inverse else 1)
    for x, sb, sl, sh, H, y in ((q, qb, ql, qh, Hq, q_out), (k, kb, kl, kh, Hkv, k_out)):
        if H:
            x = array(x, (B, L, H, D), (sb, sl, sh, 1))
            y = array(y, (B, L, H, D), (L * H * D, H * D, D, 1))
            y[:] = x
            y[..., :h] = x[..., :h] * c - x[..., h:R] * s
            y[..., h:R] = x[..., h:R] * c + x[..., :h] * s


@pytest.fixture
def cpu_ops(monkeypatch):
    """The operators' own code on CPU tensors, with a stand-in for the library: what it was
    called with is kept, and of the kernels only the rotation is computed."""

    calls = []

    def call_on(device, name, *args):
        calls.append(name)
        if name == "mrsa_rotary_fwd":
            _plain_rotary(*args)
        return _lib.MRSA_OK

    monkeypatch.setattr(_lib, "call_on", call_on)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    monkeypatch.setattr(paged_cache, "check_heads", lambda t, name: None)
    monkeypatch.setattr(rotary, "check_heads", lambda t, name: None)
    lib = torch.library.Library("mrsa", "IMPL")
    lib.impl("rotary", rotary._rotary_impl, "CPU")
    lib.impl("paged_append_", paged_cache._paged_append_impl, "CPU")
    lib.impl("paged_attention", paged_cache._paged_attention_impl, "CPU")
    lib.impl("copy_pages_", paged_cache._copy_pages_impl, "CPU")
    yield calls
    lib._destroy()


def _pools(**kw):
    return torch.zeros(2, 5, 16, 2, 64, **kw), torch.zeros(2, 5, 16, 2, 64, **kw)


def _append(kp, vp, **kw):
    k = torch.zeros(1, 3, 2, 64)
    mrsa.paged_cache_append(k, k, kp, vp, torch.zeros(1, 5, dtype=torch.int32),
                            torch.arange(3)[None], **kw)


def test_in_place_operators_raise_the_pools_version_counters(cpu_ops):
    # (what torch itself goes by to refuse a stale backward pass, and kv_fragments_cached to lay
    # a changed K / V out again)
    kp, vp = _pools()
    view = kp[0].view(1, 80, 2, 64)
    before = kp._version, vp._version, view._version
    _append(kp[0], vp[0])
    after = kp._version, vp._version, view._version
    assert all(b > a for a, b in zip(before, after))
    torch.ops.mrsa.copy_pages_(kp, vp, [0], [1])
    assert kp._version > after[0] and vp._version > after[1] and view._version > after[2]
    w = torch.ones(2, 5, 16, 2, 64, requires_grad=True)
    loss = (w * kp).sum()
    _append(kp[1], vp[1])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():       # those tensors have no counter
        kp, vp = _pools()
    _append(kp[0], vp[0])
    torch.ops.mrsa.copy_pages_(kp, vp, [0], [1])
    mixed, _ = _pools()
    _append(kp[0], mixed[0]), _append(mixed[0], vp[0])
    assert mixed._version == 2
    assert cpu_ops[:5] == ["mrsa_paged_append_fwd", "mrsa_copy_pages",
                            "mrsa_paged_append_fwd", "mrsa_paged_append_fwd", "mrsa_copy_pages"]


def test_batches_and_attention_with_room_to_grow(cpu_ops, monkeypatch):
    c = mrsa.PagedKVCache(1, 12, 16, 2, 64, device="cpu")
    a, b = c.add(20), c.add(3)
    now, room = c.batch([a, b]), c.batch([a, b], max_len=70)
    assert now.max_len == 20 and now.page_table.shape == (2, 2)
    assert room.max_len == 70 and room.page_table.shape == (2, 5)
    assert room.page_table.tolist() == [c.pages(a) + [-1] * 3, c.pages(b) + [-1] * 4]
    for x, y in ((room.slots, now.slots), (room.cache_lens, now.cache_lens),
                 (room.positions, now.positions), (room.query_starts, now.query_starts)):
        assert torch.equal(x, y)
    c.batch([a, b], max_len=20)
    c.batch([], max_len=0)
    for bad in (19, 0, -1):
        with pytest.raises(ValueError, match="max_len"):
            c.batch([a, b], max_len=bad)
    seen = []
    monkeypatch.setattr(paged_cache, "paged_cached_attention",
                        lambda *args, **kw: seen.append(kw["max_len"]))
    q = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16)
    c.attend(0, now, q)
    c.attend(0, room, q, causal=True)
    c.attend(0, now, q, max_len=500, parts=2)
    assert seen == [20, 70, 500]
    with pytest.raises(ValueError, match="max_len"):
        c.attend(0, room, q, max_len=69)


def _paged_calls():
    """Append and attention as functions of one of their float tensors, and that tensor."""

    kp, vp = _pools(dtype=torch.bfloat16)
    k = torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16)
    table, slots = torch.zeros(1, 5, dtype=torch.int32), torch.arange(3)[None]
    lens = torch.tensor([3], dtype=torch.int32)
    append = lambda **kw: mrsa.paged_cache_append(  # noqa: E731
        **{**dict(k=k, v=k, q=k, k_pages=kp[0], v_pages=vp[0], page_table=table, slots=slots),
           **kw})
    attend = lambda **kw: mrsa.paged_cached_attention(  # noqa: E731
        **{**dict(q=k, k_pages=kp[0], v_pages=vp[0], page_table=table, cache_lens=lens), **kw})
    for name in ("q", "k", "v"):
        yield (lambda t, name=name: append(**{name: t})), k
    for name in ("k_pages", "v_pages"):
        yield (lambda t, name=name: append(**{name: t})), kp[0]
        yield (lambda t, name=name: attend(**{name: t})), kp[0]
    yield (lambda t: attend(q=t)), k


@pytest.mark.parametrize("i", range(8))
def test_paged_operators_refuse_what_they_have_no_derivative_of(cpu_ops, i):
    call, t = list(_paged_calls())[i]
    call(t)
    with pytest.raises(ValueError, match="no gradient"):
        call(t.clone().requires_grad_())
    with torch.no_grad():
        call(t.clone().requires_grad_())
    n = len(cpu_ops)
    for grads in (False, True):          # (no_grad leaves forward mode on)
        with torch.set_grad_enabled(grads):
            with forward_ad.dual_level():
                with pytest.raises(ValueError, match="forward-mode"):
                    call(forward_ad.make_dual(t, torch.ones_like(t)))
            with pytest.raises(ValueError, match="forward-mode"):
                torch.func.jvp(call, (t,), (torch.ones_like(t),))
            assert len(cpu_ops) == n
            with forward_ad.dual_level():
                call(t)              # nothing dual
            n = len(cpu_ops)


def test_page_copies_refuse_what_they_have_no_derivative_of():
    with FakeTensorMode():
        kp, vp = _pools(device="cuda")
        for call, t in ((lambda t: mrsa.copy_cache_pages(t, vp, [0], [1]), kp),
                        (lambda t: mrsa.copy_cache_pages(kp, t, [0], [1]), vp)):
            call(t)
            with pytest.raises(ValueError, match="no gradient"):
                call(t.clone().requires_grad_())
            with torch.no_grad():
                call(t.clone().requires_grad_())
            with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))


def _rope(seed=0):
    g = torch.Generator().manual_seed(seed)
    q, tq, gq = torch.randn(3, 2, 5, 3, 8, generator=g)
    k, tk, gk = torch.randn(3, 2, 5, 1, 8, generator=g)
    cos, sin = mrsa.rotary_tables(9, mrsa.rotary_frequencies(6)[0], device="cpu")
    return q, k, tq, tk, gq, gk, lambda q, k: mrsa.rotary_qk(q, k, cos, sin)


def test_rotary_forward_mode(cpu_ops):
    # the rotation is linear: its derivative along a tangent is the tangent, turned
    q, k, tq, tk, gq, gk, f = _rope()
    want_q, want_k = f(tq, tk)
    assert not torch.equal(want_q, tq)

    def tangents(a, b):
        with forward_ad.dual_level():
            return [forward_ad.unpack_dual(t).tangent
                    for t in f(*(forward_ad.make_dual(x, t) if t is not None else x
                                 for x, t in ((q, a), (k, b))))]

    for grads in (False, True):          # (no_grad leaves forward mode on)
        with torch.set_grad_enabled(grads):
            got = tangents(tq, tk)
            assert torch.equal(got[0], want_q) and torch.equal(got[1], want_k)
            got = tangents(tq, None)
            assert torch.equal(got[0], want_q) and not got[1].any()
            got = tangents(None, tk)
            assert not got[0].any() and torch.equal(got[1], want_k)
            with forward_ad.dual_level():
                out = f(forward_ad.make_dual(q, tq), None)[0]
                assert torch.equal(forward_ad.unpack_dual(out).tangent, want_q)
                out = f(q, k)            # nothing dual in a dual level
                assert torch.equal(out[0], f(q, k)[0])
    # forward over reverse: the gradient of sum(f(q)^2) / 2 is f'(f(q)), its derivative along t
    # f'(f(t)) = t, off by two rotations, each by at most 3 x 2^-24 (|x1| + |x2|), of values up to 4
    x = q.clone().requires_grad_()
    with forward_ad.dual_level():
        y = f(forward_ad.make_dual(x, tq), None)[0]
        dx, = torch.autograd.grad((y * y).sum() / 2, x)
        assert (forward_ad.unpack_dual(dx).tangent - tq).abs().max() <= 2 * 3 * 8 * 2.0 ** -24


@pytest.mark.filterwarnings("ignore:There is a performance drop")
def test_rotary_under_function_transforms(cpu_ops):
    q, k, tq, tk, gq, gk, f = _rope(1)
    want = f(tq, tk)
    out, got = torch.func.jvp(f, (q, k), (tq, tk))
    assert all(torch.equal(a, b) for a, b in zip((*out, *got), (*f(q, k), *want)))
    x, y = q.clone().requires_grad_(), k.clone().requires_grad_()
    grads = torch.autograd.grad(f(x, y), (x, y), (gq, gk))
    got = torch.func.grad(lambda a, b: sum((o * w).sum() for o, w in zip(f(a, b), (gq, gk))),
                          argnums=(0, 1))(q, k)
    assert all(torch.equal(a, b) for a, b in zip(got, grads))
    got = torch.func.vjp(f, q, k)[1]((gq, gk))
    assert all(torch.equal(a, b) for a, b in zip(got, grads))
    two, tangents = torch.stack((q, gq)), torch.stack((tq, q))
    one = lambda a, t: torch.func.jvp(lambda x: f(x, None)[0], (a,), (t,))[1]  # noqa: E731
    got = torch.func.vmap(one)(two, tangents)
    assert torch.equal(got, torch.stack([f(t, None)[0] for t in tangents]))
    got = torch.func.vmap(torch.func.grad(lambda a: f(a, None)[0].square().sum() / 2))(two)
    assert (got - two).abs().max() <= 2 * 3 * 8 * 2.0 ** -24


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_rotary_and_its_gradient_trace_without_a_graph_break(cpu_ops, backend):
    q, k, tq, tk, gq, gk, f = _rope(2)
    compiled = torch.compile(f, backend=backend, fullgraph=True)
    assert all(torch.equal(a, b) for a, b in zip(compiled(q, k), f(q, k)))
    x, y = q.clone().requires_grad_(), k.clone().requires_grad_()
    want = torch.autograd.grad(f(x, y), (x, y), (gq, gk))
    got = torch.autograd.grad(compiled(x, y), (x, y), (gq, gk))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("backend", [None, "eager", "aot_eager"])
def test_traced_and_direct_calls_refuse_tangents(cpu_ops, backend):
    q, _, tq, _, _, _, _ = _rope(3)
    cos, sin = torch.zeros(5, 3), torch.zeros(5, 3)
    kp, vp = _pools()
    k = torch.zeros(1, 3, 2, 64)
    table, slots = torch.zeros(1, 5, dtype=torch.int32), torch.arange(3)[None]
    lens = torch.tensor([3], dtype=torch.int32)
    ops, rest = torch.ops.mrsa, (None, None, None, None, False)
    calls = [
        (lambda t: ops.rotary(t, None, cos, sin, None, False, False), q),
        (lambda t: ops.paged_append_(t, k, kp[0], vp[0], table, slots, *rest), k),
        (lambda t: ops.paged_append_(k, k, t, vp[0], table, slots, *rest), kp[0]),
        (lambda t: ops.paged_attention(t, kp[0], vp[0], table, lens, None, 3, False, -1, 0.1, 1),
         k),
        (lambda t: ops.copy_pages_(kp, t, [0], [1]), vp),
    ]
    for call, t in calls:
        torch._dynamo.reset()
        f = call if backend is None else torch.compile(call, backend=backend)
        f(t)
        n = len(cpu_ops)
        with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
            f(forward_ad.make_dual(t, torch.ones_like(t)))
        assert len(cpu_ops) == n
