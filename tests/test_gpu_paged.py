"""The paged cache's operators on the GPU against the fp64 oracle.

Attention's tolerance for one output, with u half a step of the type, A = sum_j p_j |v_j|
and r = scale max_j sum_d |q_d k_jd|:
  scores   fp32 sums of D exact products: off by at most D 2^-24 r, the product with
           the scale by 2 x 2^-24 r more, so e_s = (D + 2) 2^-24 r
  exp2     2 x 2^-24 of its argument's rounding per unit of exponent (at most r and
           the maximum's, 2 r) and 2^-22 of its own: e_p = e_s + (4 r + 4) 2^-24
  P        rounded as an operand: u per term (fp16: or half its smallest subnormal)
  sums     n terms in fp32, rescaled and joined: (n + 64) 2^-24
  out      u of itself
so |error| <= A (u + 2 e_p + 2 (n + 64) 2^-24) + u |out| (fp16: + n 2^-25 max|v|), and
the LSE's is e_p + (n + 64) 2^-24 + 2^-22 (1 + |lse|)."""

import pytest
import torch

import mrsa
from mrsa import _lib
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F24 = 2.0 ** -24


def _case(B, Lq, lens, Hq, Hkv, D, page, dtype, seed=0, spare=2, poison=True, unmap=()):
    """Pools whose unused rows are NaN and infinite, pages in random order."""

    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    N = sum(need) + spare
    k = torch.randn(N, page, Hkv, D, generator=g).to(dtype)
    v = torch.randn(N, page, Hkv, D, generator=g).to(dtype)
    table = torch.full((B, max(need, default=0) + 1), -1, dtype=torch.int32)
    order, at = torch.randperm(N, generator=g), 0
    used = torch.zeros(N, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        pages = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = pages.int()
        for j in range(n):
            used[pages[j // page], j % page] = True
    if poison:
        bad = torch.tensor([float("nan"), float("inf"), float("-inf")])
        k[~used] = bad[torch.randint(0, 3, k[~used].shape, generator=g)].to(dtype)
        v[~used] = bad[torch.randint(0, 3, v[~used].shape, generator=g)].to(dtype)
    for b, e, to in unmap:  # mapped entries that hold no keys
        table[b, e] = to if to < 0 else N + to
    q = torch.randn(B, Lq, Hq, D, generator=g).to(dtype)
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32)


def _check(got, q, k, v, table, lens, **kw):
    out, lse = (t.cpu() for t in got)
    starts = kw.get("query_starts")
    want, wlse, size, reach = P.attention(q.cpu(), k.cpu(), v.cpu(), table.cpu(), lens.cpu(),
                                          None if starts is None else starts.cpu(),
                                          kw.get("causal", False), kw.get("window"),
                                          kw.get("sm_scale"))
    n = float(lens.max()) if lens.numel() else 0.0
    D, u = q.shape[-1], torch.finfo(q.dtype).eps / 2
    e_p = (D + 2) * F24 * reach + (4 * reach + 4) * F24
    sums = (n + 64) * F24
    tol = size * (u + 2 * e_p[..., None] + 2 * sums) * (1 + u) + u * want.abs()
    if q.dtype == torch.float16:
        big = v.cpu()[torch.isfinite(v.cpu())].abs().max() if v.numel() else 0.0
        tol = tol + n * 2.0 ** -25 * float(big) + 2.0 ** -25
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), (float((err - tol).max()), float(err.max()))
    seen = torch.isfinite(wlse)
    assert torch.equal(torch.isfinite(lse), seen) and bool((lse[~seen] == float("-inf")).all())
    assert not out[~seen].any()
    ltol = e_p + sums + 2.0 ** -22 * (1 + wlse.abs())
    assert bool(((lse.double() - wlse).abs() <= ltol)[seen].all())


def _run(q, k, v, table, lens, **kw):
    move = lambda t: t.to(DEV) if isinstance(t, torch.Tensor) else t  # noqa: E731
    return mrsa.paged_cached_attention(move(q), move(k), move(v), move(table), move(lens),
                                       **{n: move(t) for n, t in kw.items()})


SHAPES = [
    # B, Lq, lens, Hq, Hkv, D, page
    (1, 1, [1], 1, 1, 128, 16),
    (1, 1, [1000], 28, 4, 128, 64),
    (3, 1, [0, 17, 33], 28, 4, 128, 16),
    (4, 1, [31, 32, 127, 129], 14, 2, 64, 32),
    (2, 1, [256, 255], 16, 1, 128, 128),
    (2, 1, [300, 64], 8, 8, 64, 256),
    (2, 3, [70, 2], 20, 1, 128, 16),
    (2, 5, [5, 131], 28, 4, 128, 32),
    (1, 32, [200], 28, 4, 128, 64),
    (2, 33, [40, 160], 14, 2, 64, 16),
    (1, 64, [64], 4, 4, 128, 64),
    (2, 100, [250, 90], 16, 4, 128, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(x) for x in s))
def test_attention_matches_the_oracle(shape, dtype):
    B, Lq, lens, Hq, Hkv, D, page = shape
    args = _case(B, Lq, lens, Hq, Hkv, D, page, dtype, seed=len(lens) + Lq + D)
    _check(_run(*args), *args)
    _check(_run(*args, causal=True), *args, causal=True)
    for parts in (1, 2, 7):
        _check(_run(*args, window=40, parts=parts, max_len=max(lens)), *args, window=40)


# Columns of two to ten waves, over tiles that fill the ring more than once: rows of one KV
# head, whole tiles and one key more or less.
@pytest.mark.parametrize("Lq", [17, 40, 128, 129, 160, 225, 256, 257, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_blocks_over_many_tiles(Lq, D):
    for lens, page in (([64, 65], 64), ([191, 0, 192], 16), ([321, 449], 32), ([1000, 703], 128)):
        args = _case(len(lens), Lq, lens, 2, 2, D, page, torch.bfloat16, seed=Lq + D)
        starts = torch.tensor([n // 2 for n in lens], dtype=torch.int32)
        for kw in (dict(parts=1), dict(parts=2, causal=True), dict(window=200, parts=1),
                   dict(query_starts=starts, window=130, parts=3),
                   dict(query_starts=starts, causal=True)):
            _check(_run(*args, **kw), *args, **kw)


def test_holes_and_values_not_finite_among_many_tiles():
    args = _case(1, 200, [900], 2, 1, 128, 32, torch.bfloat16, seed=3, unmap=[(0, 9, -1), (0, 20, 3)])
    for kw in (dict(parts=1), dict(parts=2, causal=True)):
        _check(_run(*args, **kw), *args, **kw)
    q, k, v, table, lens = _case(1, 200, [900], 2, 1, 128, 32, torch.bfloat16, seed=4)
    v[P.place(table, 0, 850, 32, k.shape[0])] = float("inf")
    out, lse = (t.cpu() for t in _run(q, k, v, table, lens, causal=True))
    want, wlse, _, _ = P.attention(q, k, v, table, lens, causal=True)
    assert torch.equal(torch.isposinf(out), torch.isposinf(want)) and not torch.isnan(out).any()
    assert bool(torch.isposinf(out[0, 150:]).all()) and bool(torch.isfinite(out[0, :150]).all())


@pytest.mark.parametrize("window", [0, 1, 5, 31, 64, 100000])
@pytest.mark.parametrize("causal", [False, True])
def test_windows_and_blocks_inside_a_sequence(window, causal):
    args = _case(3, 6, [90, 7, 150], 14, 2, 128, 16, torch.bfloat16, seed=window)
    # inside, over the end (padding behind), before the start (padding in front)
    for starts in ([40, 0, 100], [87, 5, 149], [-3, -6, -1], [90, 1 << 30, -(1 << 30)]):
        kw = dict(query_starts=torch.tensor(starts, dtype=torch.int32), causal=causal,
                  window=window)
        _check(_run(*args, **kw), *args, **kw)
        _check(_run(*args, parts=3, **kw), *args, **kw)


def test_unmapped_pages_hold_no_keys():
    for unmap in ([(0, 0, -1)], [(0, 2, 0), (1, 0, 5)], [(0, e, -7) for e in range(7)]):
        args = _case(2, 3, [100, 20], 7, 1, 128, 16, torch.bfloat16, seed=4, unmap=unmap)
        _check(_run(*args), *args)
        _check(_run(*args, parts=4, causal=True), *args, causal=True)


def test_values_that_are_not_finite_stay_with_the_rows_that_see_them():
    # V rows of the block itself, which causal and windowed rows see or do not
    for dtype in (torch.bfloat16, torch.float16):
        for page, Hq, Hkv in ((16, 14, 2), (64, 8, 8)):
            q, k, v, table, lens = _case(1, 20, [75], Hq, Hkv, 128, page, dtype, seed=5)
            for j, x in ((60, float("inf")), (66, float("nan")), (70, float("-inf"))):
                at = P.place(table, 0, j, page, k.shape[0])
                v[at[0], at[1], 0, 3::7] = x
            k[P.place(table, 0, 72, page, k.shape[0])] = float("nan")
            for kw in (dict(causal=True), dict(window=4), dict(causal=True, window=3)):
                out, lse = (t.cpu().double() for t in _run(q, k, v, table, lens, **kw))
                want, wlse, size, reach = P.attention(q, k, v, table, lens, **kw)
                assert torch.equal(torch.isnan(out), torch.isnan(want))
                assert torch.equal(torch.isinf(out), torch.isinf(want))
                assert torch.equal(out[torch.isinf(out)], want[torch.isinf(want)])
                fine = torch.isfinite(want)
                e_p = (130 * F24 * reach + (4 * reach + 4) * F24)[..., None]
                u = torch.finfo(dtype).eps / 2
                tol = size * (u + 2 * e_p + 300 * F24) * (1 + u) + u * want.abs() + 2.0 ** -18
                assert bool(((out - want).abs() <= tol)[fine].all())


def test_scales_and_large_scores():
    q, k, v, table, lens = _case(2, 2, [300, 40], 14, 2, 128, 64, torch.bfloat16, seed=6)
    for scale in (1.0, 0.01, 3.0):
        _check(_run(q, k, v, table, lens, sm_scale=scale), q, k, v, table, lens, sm_scale=scale)
    # scores that rise along the cache: the maximum moves in every tile
    at = torch.arange(300)
    page = table[0].long()[at // 64]
    k[page, at % 64] = (q[0, 0, 0] * (at[:, None, None] / 300.0)).to(k.dtype)
    _check(_run(q, k, v, table, lens), q, k, v, table, lens)


def test_layouts_strides_and_bounds():
    q, k, v, table, lens = _case(2, 3, [100, 33], 8, 2, 64, 16, torch.bfloat16, seed=7)
    want = [t.clone() for t in _run(q, k, v, table, lens)]
    # [pages, Hkv, page_size, D] pools, K and V of one tensor, layers between pages
    kh = k.transpose(1, 2).contiguous().transpose(1, 2)
    both = torch.stack((k, v), 1)
    layers = torch.stack((torch.zeros_like(k), k), 1)
    fused = torch.randn(2, 3, 8 * 64 + 9 * 8).to(q.dtype)
    fused[..., 8:8 + 512] = q.reshape(2, 3, 512)
    wide = torch.full((2, 20), -1, dtype=torch.int32)
    wide[:, 3:3 + table.shape[1]] = table
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape)
    odd.copy_(q)
    d = lambda t: t.to(DEV)  # noqa: E731
    tries = [
        (q, kh, kh.transpose(1, 2).transpose(1, 2), table), (q, k, v.transpose(1, 2).contiguous()
                                                             .transpose(1, 2), table),
        (q, d(both)[:, 0], d(both)[:, 1], table), (q, d(layers)[:, 1], v, table),
        (d(fused)[..., 8:520].view(2, 3, 8, 64), k, v, table), (odd, k, v, table),
        (q.transpose(1, 2).contiguous().transpose(1, 2), k, v, table),
        (q, k, v, d(wide)[:, 3:3 + table.shape[1]]), (q, k, v, table.t().contiguous().t()),
    ]
    for n, (q2, k2, v2, t2) in enumerate(tries):
        got = _run(q2, k2, v2, t2, lens)
        if n == 0:
            _check(got, q, k, k, table, lens)
            continue
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), n
    # max_len as told, and lengths past it or past the table cut to it
    for max_len, cut in ((100, [100, 33]), (64, [64, 33]), (0, [0, 0]), (10 ** 6, [100, 33])):
        _check(_run(q, k, v, table, lens, max_len=max_len), q, k, v, table,
               torch.tensor(cut, dtype=torch.int32))
    q, k, v, table, lens = _case(2, 3, [100, 33], 8, 2, 64, 16, torch.bfloat16, poison=False)
    for over in ([10 ** 6, -5], [table.shape[1] * 16, 33]):
        cut = [min(max(n, 0), table.shape[1] * 16) for n in over]
        _check(_run(q, k, v, table, torch.tensor(over, dtype=torch.int32)), q, k, v, table,
               torch.tensor(cut, dtype=torch.int32))
    # misaligned pools are refused, not copied
    shifted = torch.empty(k.numel() + 1, dtype=k.dtype, device=DEV)[1:].view(k.shape)
    with pytest.raises(ValueError):
        _run(q, shifted, v, table, lens)


def test_empty_calls():
    q, k, v, table, lens = _case(2, 3, [20, 3], 8, 2, 64, 16, torch.bfloat16)
    out, lse = _run(q[:0], k, v, table[:0], lens[:0])
    assert out.shape == (0, 3, 8, 64) and lse.shape == (0, 3, 8)
    out, lse = _run(q[:, :0], k, v, table, lens)
    assert out.shape == (2, 0, 8, 64)
    for t, p in ((table[:, :0], k), (table, k[:0])):
        out, lse = _run(q, p, v[:p.shape[0]], t, lens)
        assert not out.any() and bool((lse == float("-inf")).all())


def test_offsets_past_32_bits():
    # 70 000 pages of 32768 values: 2.3e9 in each pool, the pages in use at the end
    N, page, Hkv, D = 70000, 64, 4, 128
    kp = torch.empty(N, page, Hkv, D, dtype=torch.bfloat16, device=DEV)
    vp = torch.empty(N, page, Hkv, D, dtype=torch.bfloat16, device=DEV)
    q, k, v, table, lens = _case(2, 2, [130, 90], 28, Hkv, D, page, torch.bfloat16, seed=8)
    n = k.shape[0]
    far = torch.where(table >= 0, N - 1 - table * 13, -1).int()
    kp[N - 1 - torch.arange(n, device=DEV) * 13] = k.to(DEV)
    vp[N - 1 - torch.arange(n, device=DEV) * 13] = v.to(DEV)
    got = _run(q, kp, vp, far, lens)
    _check(got, q, k, v, table, lens)
    # and an append and a copy there
    rows = torch.randn(2, 1, Hkv, D).bfloat16().to(DEV)
    slots = torch.tensor([[129], [89]], device=DEV)
    mrsa.paged_cache_append(rows, rows * 2, kp, vp, far.to(DEV), slots)
    for b, s in ((0, 129), (1, 89)):
        p = int(far[b, s // page])
        assert torch.equal(kp[p, s % page], rows[b, 0]) and torch.equal(vp[p, s % page],
                                                                       rows[b, 0] * 2)
    mrsa.copy_cache_pages(kp, vp, [N - 1], [1])
    assert torch.equal(kp[1].view(torch.int16), kp[N - 1].view(torch.int16))


# ---- append

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,Hq,Hkv,D,R,page", [
    (1, 1, 28, 4, 128, 128, 64), (3, 5, 8, 2, 64, 32, 16), (2, 40, 4, 4, 128, 0, 32),
    (2, 3, 2, 1, 40, 12, 16), (16, 1, 28, 4, 128, 128, 16),
])
def test_append_writes_its_rows_and_no_others(dtype, B, L, Hq, Hkv, D, R, page):
    g = torch.Generator().manual_seed(B + L + D)
    N, width = 3 * B + 4, 3
    kp, vp = torch.randn(2, N, page, Hkv, D, generator=g).to(dtype)
    table = torch.randperm(N, generator=g)[:B * width].view(B, width).int()
    table[0, 2] = -1
    table[-1, 2] = N
    k, v = torch.randn(2, B, L, Hkv, D, generator=g).to(dtype)
    q = torch.randn(B, L, Hq, D, generator=g).to(dtype)
    # distinct slots, some past the mapped pages and past the table (0 and page kept apart)
    free = torch.tensor([s for s in range(1, 4 * page) if s not in (page, 3 * page + 2)])
    slots = torch.stack([free[torch.randperm(len(free), generator=g)[:L]] for _ in range(B)])
    slots[:, -1] = torch.tensor([-1, 3 * page + 2, 0])[torch.arange(B) % 3]
    if L > 1:
        slots[:, 0] = page
    cos = sin = pos = None
    kr = k
    for inter in (False, True):
        kd, vd = kp.to(DEV), vp.to(DEV)
        kw = dict(interleaved=inter)
        want_q = q
        if R:
            inv = mrsa.rotary_frequencies(R)[0]
            cos, sin = mrsa.rotary_tables(500, inv, device=DEV)
            pos = torch.randint(0, 500, (B, L), generator=g)
            kw.update(cos=cos, sin=sin, positions=pos.to(DEV))
            rot_q, rot_k = mrsa.rotary_qk(q.to(DEV), k.to(DEV), cos, sin, pos.to(DEV),
                                          interleaved=inter)
            want_q, kr = rot_q.cpu(), rot_k.cpu()
        got = mrsa.paged_cache_append(k.to(DEV), v.to(DEV), kd, vd, table.to(DEV), slots.to(DEV),
                                      q=q.to(DEV), **kw)
        assert torch.equal(got.cpu(), want_q)          # the same bits as rotary_qk
        assert torch.equal(kd.cpu(), P.append(kr, kp, table, slots))
        assert torch.equal(vd.cpu(), P.append(v, vp, table, slots))
        if R:  # without q, at the slots' own places
            kd, vd = kp.to(DEV), vp.to(DEV)
            assert mrsa.paged_cache_append(k.to(DEV), v.to(DEV), kd, vd, table.to(DEV),
                                           slots.to(DEV), cos=cos, sin=sin,
                                           interleaved=inter) is None
            at, _ = mrsa.rotary_qk(k.to(DEV), None, cos, sin, slots.to(DEV), interleaved=inter)
            assert torch.equal(kd.cpu(), P.append(at.cpu(), kp, table, slots))


def test_append_strides_and_empty_calls():
    g = torch.Generator().manual_seed(1)
    table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32)
    slots = torch.tensor([[3, 4, 17], [0, 31, 30]])
    fused = torch.randn(2, 3, (4 + 2 + 2) * 64, generator=g).half().to(DEV)
    k = fused[..., 256:384].view(2, 3, 2, 64)
    v = fused[..., 384:].view(2, 3, 2, 64)
    base_k, base_v = torch.randn(2, 4, 16, 2, 64, generator=g).half()
    want = [P.append(r.cpu(), p, table, slots) for r, p in ((k, base_k), (v, base_v))]
    pools = [
        (base_k.to(DEV), base_v.to(DEV)),
        tuple(t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for t in (base_k, base_v)),
        tuple(torch.stack((base_k, base_v), 1).to(DEV).unbind(1)),
    ]
    shifted = [torch.empty(base_k.numel() + 1, dtype=torch.float16, device=DEV)[1:].view(
        base_k.shape) for _ in range(2)]
    shifted[0].copy_(base_k)
    shifted[1].copy_(base_v)
    pools.append(tuple(shifted))                       # unaligned: one value at a time
    for kd, vd in pools:
        mrsa.paged_cache_append(k, v, kd, vd, table.to(DEV), slots.to(DEV))
        assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1])
    before = pools[0][0].clone()
    mrsa.paged_cache_append(k[:0], v[:0], *pools[0], table[:0].to(DEV), slots[:0].to(DEV))
    mrsa.paged_cache_append(k[:, :0], v[:, :0], *pools[0], table.to(DEV), slots[:, :0].to(DEV))
    mrsa.paged_cache_append(k, v, *pools[0], table[:, :0].to(DEV), slots.to(DEV))
    assert torch.equal(before, pools[0][0])
    with pytest.raises(ValueError):                    # K and V in one memory
        mrsa.paged_cache_append(k, v, pools[0][0], pools[0][0], table.to(DEV), slots.to(DEV))


# ---- pages

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_page_copies(dtype):
    g = torch.Generator().manual_seed(2)
    for layers, N, page, Hkv, D, n in ((3, 20, 16, 2, 64, 7), (1, 5, 64, 4, 128, 2),
                                       (2, 1200, 16, 1, 8, 500), (28, 9, 16, 1, 24, 4)):
        k, v = torch.randn(2, layers, N, page, Hkv, D, generator=g).to(dtype)
        order = torch.randperm(N, generator=g).tolist()
        src, dst = order[:n], order[n:2 * n]
        src[-1] = src[0]                               # one page to two places
        want_k, want_v = k.clone(), v.clone()
        want_k[:, dst], want_v[:, dst] = k[:, src], v[:, src]
        kd, vd = k.to(DEV), v.to(DEV)
        mrsa.copy_cache_pages(kd, vd, src, dst)
        assert torch.equal(kd.cpu(), want_k) and torch.equal(vd.cpu(), want_v)
        # one layer; K and V of one tensor, every second page
        kd = k.to(DEV)
        mrsa.copy_cache_pages(kd[0], vd[0], src, dst)
        assert torch.equal(kd[0].cpu(), want_k[0]) and torch.equal(kd[1:].cpu(), k[1:])
        both = torch.stack((k, v), 2).to(DEV)
        mrsa.copy_cache_pages(both[:, :, 0], both[:, :, 1], src, dst)
        assert torch.equal(both[:, :, 0].cpu(), want_k) and torch.equal(both[:, :, 1].cpu(), want_v)


def test_page_copies_that_are_refused_copy_nothing():
    k = torch.arange(4 * 16 * 8.0, device=DEV).view(4, 16, 1, 8)
    v, before = -k, k.clone()
    for src, dst in (([4], [0]), ([0], [4]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 2], [2, 3]),
                     ([1], [1]), ([0, 2 ** 40], [2, 3])):
        with pytest.raises(ValueError):
            mrsa.copy_cache_pages(k, v, src, dst)
    mrsa.copy_cache_pages(k, v, [], [])
    torch.cuda.synchronize()
    assert torch.equal(k, before) and torch.equal(v, -before)


# ---- beside the framework's own cached attention, together, on streams and in graphs

def test_agrees_with_the_dense_cached_window_attention():
    g = torch.Generator().manual_seed(3)
    L, Lq, W, page = 1024, 32, 256, 64
    k, v = torch.randn(2, 1, L, 4, 128, generator=g).bfloat16().to(DEV)
    q = torch.randn(1, Lq, 28, 128, generator=g).bfloat16().to(DEV)
    for start in (0, 480, L - Lq):
        pos = torch.arange(start, start + Lq, device=DEV)
        want, wlse = mrsa.cached_local_attention(q, k, v, torch.ones(1, L, dtype=torch.bool,
                                                                    device=DEV), pos, W, 64)
        order = torch.randperm(L // page, generator=g).int()
        kp, vp = (torch.empty(L // page, page, 4, 128, dtype=torch.bfloat16, device=DEV)
                  for _ in range(2))
        kp[order.long().to(DEV)] = k[0].view(-1, page, 4, 128)
        vp[order.long().to(DEV)] = v[0].view(-1, page, 4, 128)
        out, lse = mrsa.paged_cached_attention(
            q, kp, vp, order[None].to(DEV), torch.tensor([L], dtype=torch.int32, device=DEV),
            query_starts=torch.tensor([start], dtype=torch.int32, device=DEV), window=W)
        # each is within its own rounding of the exact value: half a step of P per term and
        # of the result, of weighted sums of |v| below 4
        assert (out.float() - want.float()).abs().max() <= 2 * 2 * 4 * 2.0 ** -8
        # and of scores up to 12: 2 ((128 + 6) 12 + 1024 + 64) 2^-24
        assert (lse - wlse).abs().max() <= 2.0 ** -11


class _Dense:
    """What a sequence's cache must hold: rotated keys and values of one layer."""

    def __init__(self, Hkv, D):
        self.k = torch.zeros(0, Hkv, D)
        self.v = torch.zeros(0, Hkv, D)


def test_prompts_blocks_forks_and_compaction_together():
    layers, Hq, Hkv, D, page = 2, 14, 2, 64, 16
    g = torch.Generator().manual_seed(4)
    c = mrsa.PagedKVCache(layers, 24, page, Hkv, D, device=DEV)
    for pool in (c.k_pages, c.v_pages):
        pool.fill_(float("nan"))
    cos, sin = mrsa.rotary_tables(400, mrsa.rotary_frequencies(D, 1e6, "yarn", 8.0)[0], device=DEV)
    model = {}

    def step(seqs, rows, rewrite=False, **kw):
        """New (or rewritten) rows of some sequences through every layer, checked."""
        L = max(rows)
        bat = c.batch(seqs, rows=rows)
        for layer in range(layers):
            q = torch.randn(len(seqs), L, Hq, D, generator=g).bfloat16()
            k, v = torch.randn(2, len(seqs), L, Hkv, D, generator=g).bfloat16()
            rq = c.append(layer, bat, k.to(DEV), v.to(DEV), q=q.to(DEV), cos=cos, sin=sin)
            out, lse = c.attend(layer, bat, rq, **kw)
            turned = P.rotary(k, cos.cpu(), sin.cpu(), bat.positions.cpu()).bfloat16()
            for i, (s, r) in enumerate(zip(seqs, rows)):
                held = model.setdefault((s, layer), _Dense(Hkv, D))
                keep = c.length(s) - r
                held.k = torch.cat((held.k[:keep], turned[i, :r].float()))
                held.v = torch.cat((held.v[:keep], v[i, :r].float()))
                n = c.length(s)
                assert held.k.shape[0] == n
                # the cache's own rows (their rotation may round the other way) give the check
                pages = torch.tensor(c.pages(s))
                kk = c.k_pages[layer].cpu()[pages].reshape(-1, Hkv, D)[:n]
                vv = c.v_pages[layer].cpu()[pages].reshape(-1, Hkv, D)[:n]
                assert torch.equal(vv.float(), held.v)
                assert ((kk.float() - held.k).abs() <= 2.0 ** -7 * held.k.abs() + 1e-6).all()
                pad = -(-n // 16) * 16
                kk, vv = (torch.cat((t, t.new_zeros(pad - n, Hkv, D))) for t in (kk, vv))
                _check((out[i:i + 1, :r], lse[i:i + 1, :r]), rq[i:i + 1, :r],
                       kk.view(-1, 16, Hkv, D), vv.view(-1, 16, Hkv, D),
                       torch.arange(pad // 16)[None], torch.tensor([n]),
                       query_starts=torch.tensor([n - r]), **kw)
                assert bool((lse[i, r:] == float("-inf")).all()) and not out[i, r:].any()

    a, b = c.add(37), c.add(20)
    step([a, b], [37, 20], causal=True)                # ragged prompts, the shorter padded
    for n in (1, 1, 5):                                # single tokens and a block
        for s in (a, b):
            c.extend(s, n)
        step([b, a], [n, n])
    twin = c.fork(a)
    for layer in range(layers):
        model[twin, layer] = _Dense(Hkv, D)
        model[twin, layer].k, model[twin, layer].v = model[a, layer].k, model[a, layer].v
    for s in (twin, a):                                # they part ways
        c.extend(s, 3)
    step([a, twin, b], [3, 3, 4], window=9)
    c.make_writable(a, c.length(a) - 8, c.length(a))
    step([a], [8])                                     # a block denoised again
    c.truncate(twin, 30)
    c.free(b)
    live = c.compact()
    assert live == c.num_pages - c.free_pages
    assert all(p < live for s in c.sequences() for p in c.pages(s))
    for layer in range(layers):
        model[twin, layer].k, model[twin, layer].v = (model[twin, layer].k[:30],
                                                      model[twin, layer].v[:30])
    for s in (a, twin):
        c.extend(s, 1)
    step([twin, a], [1, 1])
    c.free(a)
    c.free(twin)
    assert c.free_pages == 24


def test_other_streams():
    args = [t.to(DEV) for t in _case(2, 4, [200, 90], 28, 4, 128, 64, torch.bfloat16, seed=9)]
    want = mrsa.paged_cached_attention(*args, parts=3)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:                                  # two calls at once, a workspace each
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(mrsa.paged_cached_attention(*args, parts=3))
    for s in streams:
        s.synchronize()
    for o, l in got:
        assert torch.equal(o, want[0]) and torch.equal(l, want[1])


def test_graphs_of_a_decode_step_replay_with_new_inputs():
    # append and attention of single tokens, captured once; two graphs in turn
    B, Hq, Hkv, D, page = 3, 28, 4, 128, 16
    g = torch.Generator().manual_seed(10)
    q0, k0, v0, table, lens = _case(B, 1, [40, 100, 7], Hq, Hkv, D, page, torch.bfloat16, seed=11)
    spare = [t for t in range(k0.shape[0]) if t not in set(table.flatten().tolist())]
    for b in range(B):                                 # one page ahead, mapped before the capture
        e = int((table[b] >= 0).sum())
        if e < table.shape[1] and spare:
            table[b, e] = spare.pop()
    kp, vp, tab = k0.to(DEV), v0.to(DEV), table.to(DEV)
    cos, sin = mrsa.rotary_tables(300, mrsa.rotary_frequencies(D)[0], device=DEV)
    q = torch.zeros(B, 1, Hq, D, dtype=torch.bfloat16, device=DEV)
    k, v = torch.zeros(2, B, 1, Hkv, D, dtype=torch.bfloat16, device=DEV)
    n = lens.to(DEV)

    def step(parts):
        slots = n.long()[:, None]
        rq = mrsa.paged_cache_append(k, v, kp, vp, tab, slots, q=q, cos=cos, sin=sin)
        n.add_(1)
        return (rq, *mrsa.paged_cached_attention(rq, kp, vp, tab, n, parts=parts))

    step(1)                                            # (once outside, as torch asks)
    n.copy_(lens)
    graphs = []
    for parts in (1, 3):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(parts)
        graphs.append((graph, out, parts))
    n.copy_(lens)
    for i in range(4):
        graph, out, parts = graphs[i % 2]
        q.copy_(torch.randn(q.shape, generator=g))
        k.copy_(torch.randn(k.shape, generator=g))
        v.copy_(torch.randn(v.shape, generator=g))
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert n.tolist() == [x + i + 1 for x in lens.tolist()]
        _check(got[1:], got[0].cpu(), kp.cpu(), vp.cpu(), table, n.cpu())
        want = mrsa.paged_cached_attention(got[0], kp, vp, tab, n, parts=parts)
        assert torch.equal(got[1], want[0]) and torch.equal(got[2], want[1])
        where = [P.place(table, b, int(n[b]) - 1, page, kp.shape[0]) for b in range(B)]
        for b, at in enumerate(where):
            if at is not None:
                assert torch.equal(vp[at[0], at[1]], v[b, 0])


def test_long_tables_with_a_hole_past_their_first_entries():
    # 130 pages of 16: a hole among the first 64 entries, past them, and none
    for unmap in ([(0, 20, -1)], [(0, 100, -1)], [(0, 129, 7)], []):
        for Lq in (1, 40):
            args = _case(1, Lq, [2075], 8, 2, 128, 16, torch.bfloat16, seed=Lq, unmap=unmap)
            for kw in (dict(parts=1), dict(parts=3, causal=True)):
                _check(_run(*args, **kw), *args, **kw)


def test_blocks_at_offsets_past_32_bits():
    # 70 000 pages of 32768 values, as above, by more columns than a tile of tokens has
    N, page, Hkv, D = 70000, 64, 4, 128
    kp = torch.empty(N, page, Hkv, D, dtype=torch.bfloat16, device=DEV)
    vp = torch.empty(N, page, Hkv, D, dtype=torch.bfloat16, device=DEV)
    q, k, v, table, lens = _case(2, 40, [330, 190], 28, Hkv, D, page, torch.bfloat16, seed=9)
    far = torch.where(table >= 0, N - 1 - table * 13, -1).int()
    where = N - 1 - torch.arange(k.shape[0], device=DEV) * 13
    kp[where], vp[where] = k.to(DEV), v.to(DEV)
    for kw in (dict(), dict(causal=True, parts=2)):
        _check(_run(q, kp, vp, far, lens, **kw), q, k, v, table, lens, **kw)


def test_padding_queries_may_hold_anything():
    for Lq, n in ((2, 70), (40, 300), (200, 500)):
        q, k, v, table, lens = _case(2, Lq, [n, n - 30], 14, 2, 128, 16, torch.bfloat16, seed=Lq)
        for starts in (lens - Lq + 1, torch.full_like(lens, -(Lq // 2))):  # past the end, before 0
            pos = starts[:, None] + torch.arange(Lq)
            pad = (pos < 0) | (pos >= lens[:, None])
            assert pad.any() and not pad.all()
            bad = q.clone()
            bad[pad] = torch.tensor([float("nan"), float("inf")]).repeat(64).to(q.dtype)
            clean = torch.where(pad[..., None, None], 0, q)
            for kw in (dict(), dict(causal=True), dict(window=50, parts=3)):
                got = _run(bad, k, v, table, lens, query_starts=starts, **kw)
                _check(got, clean, k, v, table, lens, query_starts=starts, **kw)


def test_graphs_that_share_a_pool_replay_in_turn():
    # blocks (more than 16 columns) and tokens, in pieces, whose workspaces may be the same memory
    cases = [_case(2, Lq, lens, 14, 2, 128, 32, torch.bfloat16, seed=20 + Lq)
             for Lq, lens in ((1, [500, 90]), (32, [700, 333]), (90, [640, 90]))]
    dev = [[t.to(DEV) for t in c] for c in cases]
    calls = [lambda c=c, parts=parts: mrsa.paged_cached_attention(*c, parts=parts)
             for c, parts in zip(dev, (4, 5, 9))]
    for call in calls:
        call()
    graphs, pool = [], None
    for call in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = call()
        pool = graph.pool()
        graphs.append((graph, out))
    for i in (0, 1, 2, 1, 0, 2, 2, 0):
        dev[i][0].mul_(-1)
        graphs[i][0].replay()
        got = [t.clone() for t in graphs[i][1]]
        want = calls[i]()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_the_operators_trace_without_a_graph_break():
    args = [t.to(DEV) for t in _case(2, 4, [50, 20], 8, 2, 64, 16, torch.bfloat16, seed=12)]
    cos, sin = mrsa.rotary_tables(90, mrsa.rotary_frequencies(64)[0], device=DEV)

    def layer(q, kp, vp, table, lens):
        r, _ = mrsa.rotary_qk(q, None, cos, sin)
        return mrsa.paged_cached_attention(r, kp, vp, table, lens)

    want = layer(*args)
    got = torch.compile(layer, backend="eager", fullgraph=True)(*args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_the_library_is_the_one_that_ran():
    assert _lib.call("mrsa_abi_version") >= 9
