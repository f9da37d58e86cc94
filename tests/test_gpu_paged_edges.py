"""Paged attention at its edges: nothing to join, weights under the operands' smallest value,
a maximum that moves.  Tolerances as in test_gpu_paged."""

import pytest
import torch

import mrsa
from test_gpu_paged import DEV, F24, _case, _check, _run

pytestmark = pytest.mark.gpu


def test_no_keys_in_several_parts():
    # no rows, no table, no pool: every row is empty, whatever number of parts joins it
    for Lq, Hq in ((1, 8), (40, 8), (200, 14)):
        q, k, v, table, lens = _case(2, Lq, [20, 0], Hq, 2, 64, 16, torch.bfloat16)
        for t, pool, n, kw in ((table, k, lens, dict(max_len=0)), (table[:, :0], k, lens, {}),
                               (table, k[:0], lens, {}), (table, k, lens * 0, {}),
                               (table, k, lens, dict(max_len=0, window=3, causal=True))):
            for parts in (1, 2, 7, 1024):
                out, lse = _run(q, pool, v[:pool.shape[0]], t, n, parts=parts, **kw)
                assert not out.any() and bool((lse == float("-inf")).all())


def test_a_view_of_the_pool_is_laid_out_again_after_a_write():
    # a sequence whose pages follow each other, read by a dense operator through a view
    g = torch.Generator().manual_seed(30)
    kp, vp = torch.randn(2, 6, 32, 2, 128, generator=g).bfloat16().to(DEV)
    k, v = kp[:4].view(1, 128, 2, 128), vp[:4].view(1, 128, 2, 128)
    q = torch.randn(1, 128, 4, 128, generator=g).bfloat16().to(DEV)
    table = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    valid = torch.ones(1, 128, dtype=torch.bool, device=DEV)

    def check():
        got = mrsa.bidir_local_attention(q, k, v, valid, 64, 64)
        want = mrsa.bidir_local_attention(q, k.clone(), v.clone(), valid, 64, 64)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        return got[0]

    first = check()
    new = torch.randn(2, 1, 50, 2, 128, generator=g).bfloat16().to(DEV)
    mrsa.paged_cache_append(new[0], new[1], kp, vp, table, torch.arange(60, 110, device=DEV)[None])
    second = check()
    mrsa.copy_cache_pages(kp, vp, [0, 5], [3, 1])
    third = check()
    assert not torch.equal(first, second) and not torch.equal(second, third)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_a_traced_step_writes_the_pools_it_was_given(backend):
    g = torch.Generator().manual_seed(31)
    args = [t.to(DEV) for t in _case(2, 3, [50, 20], 8, 2, 64, 16, torch.bfloat16, seed=12,
                                     poison=False)]
    k, v = torch.randn(2, 2, 3, 2, 64, generator=g).bfloat16().to(DEV)
    slots = torch.tensor([[47, 48, 49], [17, 18, 19]], device=DEV)
    cos, sin = mrsa.rotary_tables(90, mrsa.rotary_frequencies(64)[0], device=DEV)
    table = args[3]
    src, dst = [int(table[0, 0])], [int(table[1, 0])]

    def step(q, kp, vp, table, lens):
        before = mrsa.paged_cached_attention(q, kp, vp, table, lens)
        rq = mrsa.paged_cache_append(k, v, kp, vp, table, slots, q=q, cos=cos, sin=sin)
        mid = mrsa.paged_cached_attention(rq, kp, vp, table, lens)
        mrsa.copy_cache_pages(kp, vp, src, dst)
        return *before, rq, *mid, *mrsa.paged_cached_attention(rq, kp, vp, table, lens)

    mine, theirs = ([t.clone() for t in args] for _ in range(2))
    want = step(*mine)
    traced = torch.compile(step, backend=backend, fullgraph=True)
    versions = theirs[1]._version, theirs[2]._version
    got = traced(*theirs)
    for a, b in zip((*got, *theirs), (*want, *mine)):
        assert torch.equal(a, b)
    assert not torch.equal(theirs[1], args[1]) and not torch.equal(want[0], want[3])
    assert theirs[1]._version > versions[0] and theirs[2]._version > versions[1]


def test_a_captured_step_of_the_cache_serves_sequences_that_grow():
    # captured at 20 and 7 rows, replayed up to 170 and 157: the bound and the table's width
    # are the capture's, everything else is read anew
    Hq, Hkv, D, page, L, most = 14, 2, 128, 16, 5, 200
    g = torch.Generator().manual_seed(32)
    c = mrsa.PagedKVCache(1, 30, page, Hkv, D, device=DEV)
    c.k_pages.fill_(float("nan")), c.v_pages.fill_(float("nan"))
    cos, sin = mrsa.rotary_tables(most, mrsa.rotary_frequencies(D)[0], device=DEV)
    seqs = [c.add(20), c.add(7)]
    rows = torch.randn(2, 2, 20, Hkv, D, generator=g).bfloat16().to(DEV)
    c.append(0, c.batch(seqs, rows=[20, 7]), rows[0], rows[1], cos=cos, sin=sin)
    q = torch.zeros(2, L, Hq, D, dtype=torch.bfloat16, device=DEV)
    k, v = torch.zeros(2, 2, L, Hkv, D, dtype=torch.bfloat16, device=DEV)
    held = c.batch(seqs, rows=L, max_len=most)

    def step():
        rq = c.append(0, held, k, v, q=q, cos=cos, sin=sin)
        return (rq, *c.attend(0, held, rq, causal=True))

    saved = c.k_pages.clone(), c.v_pages.clone()
    step()                                             # (once outside, as torch asks)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    c.k_pages.copy_(saved[0]), c.v_pages.copy_(saved[1])
    for i in range(30):
        for s in seqs:
            c.extend(s, L)
        now = c.batch(seqs, rows=L, max_len=most)
        for name in ("page_table", "cache_lens", "query_starts", "slots", "positions"):
            getattr(held, name).copy_(getattr(now, name))
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        got = [t.clone() for t in out]
        exact = c.batch(seqs, rows=L)                  # no wider than needed
        rq = c.append(0, exact, k, v, q=q, cos=cos, sin=sin)
        torch.cuda.synchronize()
        assert torch.equal(rq, got[0])
        if i % 7 == 0 or i > 27:
            _check(got[1:], rq.cpu(), c.k_pages[0].cpu(), c.v_pages[0].cpu(),
                   now.page_table.cpu(), now.cache_lens.cpu(), causal=True)
        assert bool(torch.isfinite(got[2]).all())
    assert c.length(seqs[0]) == 170


# Columns of four waves (a ring of two slots), of five and of eight (three slots).
BLOCKS = [(20, 2, 1), (150, 2, 1), (64, 4, 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Lq,Hq,Hkv", BLOCKS)
@pytest.mark.parametrize("rise", [4.0, 5.0, 6.5, 9.0, 30.0, -9.0])
def test_the_maximum_of_a_block_moves(Lq, Hq, Hkv, dtype, rise):
    # Scores of row i are c_i (j // 96) rise, c_i in 0, 1/4, 1/2, 1, -1: of a wave's columns some
    # rise past what a running maximum allows, some just below it, some fall and some stay.
    D, n = 64, 430
    q, k, v, table, lens = _case(1, Lq, [n], Hq, Hkv, D, 32, dtype, seed=Lq)
    c = torch.tensor([0.0, 0.25, 0.5, 1.0, -1.0])[torch.arange(Lq) * 7 % 5]
    q.mul_(0.125)
    q[..., 0] = c[None, :, None].to(dtype)
    at = torch.arange(n)
    page = table[0].long()[at // 32]
    k[page, at % 32, :, 0] = ((at // 96) * rise)[:, None].to(dtype)
    for kw in (dict(parts=1), dict(parts=3), dict(parts=1, causal=True), dict(window=130, parts=2)):
        _check(_run(q, k, v, table, lens, sm_scale=1.0, **kw), q, k, v, table, lens, sm_scale=1.0,
               **{x: y for x, y in kw.items() if x != "parts"})


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Lq,Hq,Hkv", BLOCKS)
def test_one_key_of_a_block_just_past_the_others(Lq, Hq, Hkv, dtype):
    # one weight of e^d over a tile's others: below 1024 (d < 6.93) the maximum stays, and the
    # operand holds up to that
    for d in (6.0, 6.9, 6.95, 7.5, 11.0):
        q, k, v, table, lens = _case(1, Lq, [300], Hq, Hkv, 128, 64, dtype, seed=int(d))
        q.zero_()
        q[..., 5] = 1
        k[table[0, :5].long(), :, :, 5] = 0
        k[table[0, 3].long(), 11, :, 5] = d     # key 203
        k[table[0, 4].long(), 40:, :, 5] = d    # keys 296 ..
        for kw in (dict(parts=1), dict(parts=1, causal=True)):
            _check(_run(q, k, v, table, lens, sm_scale=1.0, **kw), q, k, v, table, lens,
                   sm_scale=1.0, causal=kw.get("causal", False))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_of_blocks(dtype):
    for Lq, Hq, Hkv in BLOCKS:
        q, k, v, table, lens = _case(1, Lq, [250], Hq, Hkv, 128, 16, dtype, seed=Lq)
        for scale in (0.01, 1.0, 3.0):
            _check(_run(q, k, v, table, lens, sm_scale=scale), q, k, v, table, lens,
                   sm_scale=scale)


@pytest.mark.parametrize("Lq,Hq", [(1, 8), (20, 2), (150, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_fp16_weights_far_below_the_largest_still_count(Lq, Hq, D):
    # One key of score 17.5 with value 0 and n keys of score 0 with value 1: weights of
    # 2^-25.2, below half of fp16's smallest, are together n w / (1 + n w) of the output.
    # As operands they are multiplied by 2^5 at least, so each is off by 2^-25 / 2^5 at most.
    n, page = 20000, 64
    pages = -(-n // page)
    k = torch.zeros(pages, page, 1, D, dtype=torch.float16)
    v = torch.ones_like(k)
    q = torch.zeros(1, Lq, Hq, D, dtype=torch.float16)
    q[..., 0] = 1
    table = torch.arange(pages, dtype=torch.int32)[None]
    lens = torch.tensor([n], dtype=torch.int32)
    w = (n - 1) * torch.tensor(-17.5, dtype=torch.float64).exp()
    want, wlse = w / (1 + w), 17.5 + torch.log1p(w)
    e_p = (D + 2) * F24 * 17.5 + (4 * 17.5 + 4) * F24
    sums = (n + 64) * F24
    for first in (0, 130, n - 1):           # where the large one is
        kk, vv = k.clone(), v.clone()
        kk[first // page, first % page, 0, 0] = 17.5
        vv[first // page, first % page] = 0
        for parts in (1, 2):
            out, lse = (t.cpu().double() for t in _run(q, kk, vv, table, lens, sm_scale=1.0,
                                                       parts=parts))
            tol = want * (2.0 ** -11 + 2 * e_p + 2 * sums) + n * 2.0 ** -30
            assert bool(((out - want).abs() <= tol).all()), (first, parts, float(out.min()),
                                                             float(out.max()), float(want))
            assert bool(((lse - wlse).abs() <= e_p + sums + 2.0 ** -22 * (1 + wlse)).all())
