"""The paged cache's book-keeping against a plain model of it, and the refusals of
its operators and of rotary_qk, all before anything is launched (no GPU)."""

import random

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mrsa
from mrsa import _lib, paged_cache


@pytest.fixture
def cpu_copies(monkeypatch):
    """copy_cache_pages on CPU pools, with its own checks."""

    def copy(k_pages, v_pages, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for pool in (k_pages, v_pages):
            pool[:, dst] = pool[:, src]

    monkeypatch.setattr(paged_cache, "copy_cache_pages", copy)


def _cache(pages=12, P=16):
    return mrsa.PagedKVCache(2, pages, P, 1, 1, dtype=torch.float32, device="cpu")


def _write(c, seq, slots, rows):
    """Rows (a number each) written through the pages, as an append would."""
    held = c.pages(seq)
    for s, x in zip(slots, rows):
        assert c._refs[held[s // c.page_size]] == 1
        for layer in range(2):
            c.k_pages[layer, held[s // c.page_size], s % c.page_size] = x + layer
            c.v_pages[layer, held[s // c.page_size], s % c.page_size] = -x - layer


def _read(c, seq, layer=1):
    held, P = c.pages(seq), c.page_size
    return [float(c.k_pages[layer, held[s // P], s % P]) - layer for s in range(c.length(seq))]


@pytest.mark.parametrize("seed", range(6))
def test_bookkeeping_follows_a_plain_model(cpu_copies, seed):
    rng = random.Random(seed)
    c, model, count = _cache(), {}, 0
    for _ in range(300):
        op = rng.choice(["add", "extend", "extend", "rewrite", "fork", "truncate", "free", "compact"])
        before = (c.sequences(), c.free_pages, [c.pages(s) for s in c.sequences()])
        try:
            if op == "add":
                n = rng.choice([0, 1, 15, 16, 17, 40])
                seq = c.add(n)
                rows = [float(count + i) for i in range(n)]
                count += n
                _write(c, seq, range(n), rows)
                model[seq] = rows
            elif op == "compact":
                live = c.compact()
                used = {p for s in model for p in c.pages(s)}
                assert live == len(used) and used == set(range(live))
                assert sorted(c._free) == list(range(live, c.num_pages))
            elif model:
                seq = rng.choice(sorted(model))
                rows = model[seq]
                if op == "extend":
                    n = rng.choice([0, 1, 3, 16, 33])
                    slots = c.extend(seq, n)
                    assert list(slots) == list(range(len(rows), len(rows) + n))
                    new = [float(count + i) for i in range(n)]
                    count += n
                    _write(c, seq, slots, new)
                    model[seq] = rows + new
                elif op == "rewrite" and rows:
                    a = rng.randrange(len(rows))
                    b = rng.randint(a, len(rows))
                    c.make_writable(seq, a, b)
                    new = [float(count + i) for i in range(b - a)]
                    count += b - a
                    _write(c, seq, range(a, b), new)
                    model[seq] = rows[:a] + new + rows[b:]
                elif op == "fork":
                    model[c.fork(seq)] = list(rows)
                elif op == "truncate":
                    n = rng.randint(0, len(rows))
                    c.truncate(seq, n)
                    model[seq] = rows[:n]
                elif op == "free":
                    c.free(seq)
                    del model[seq]
        except mrsa.PagesExhausted:
            assert before == (c.sequences(), c.free_pages, [c.pages(s) for s in c.sequences()])
        assert c.sequences() == sorted(model)
        held = [p for s in model for p in c.pages(s)]
        assert [held.count(p) for p in range(c.num_pages)] == c._refs
        assert sorted(c._free) == [p for p in range(c.num_pages) if c._refs[p] == 0]
        for s, rows in model.items():
            assert len(c.pages(s)) == -(-len(rows) // c.page_size)
            assert _read(c, s) == rows
    for s in list(model):
        c.free(s)
    assert c.free_pages == c.num_pages


def test_forks_share_pages_until_written(cpu_copies):
    c = _cache()
    a = c.add(20)
    _write(c, a, range(20), [float(i) for i in range(20)])
    b = c.fork(a)
    assert c.pages(a) == c.pages(b) and c.free_pages == 10
    c.extend(b, 1)                       # the partly filled page is copied, the full one shared
    assert c.pages(a)[0] == c.pages(b)[0] and c.pages(a)[1] != c.pages(b)[1]
    _write(c, b, [20], [99.0])
    assert _read(c, b) == [float(i) for i in range(20)] + [99.0]
    assert c.make_writable(a, 16, 20) == 0 and c.make_writable(a, 3, 4) == 1
    full = c.add(32)
    twin = c.fork(full)
    v = c.version
    c.extend(twin, 4)                    # a full shared page is never written: no copy
    assert c.version == v and c.pages(twin)[:2] == c.pages(full)


def test_a_failed_copy_changes_nothing(monkeypatch):
    def fail(*_):
        raise RuntimeError("no launch")

    monkeypatch.setattr(paged_cache, "copy_cache_pages", fail)
    c = _cache()
    a = c.add(20)
    b = c.fork(a)
    state = (c.pages(a), c.pages(b), list(c._refs), sorted(c._free), c.version)
    with pytest.raises(RuntimeError):
        c.extend(b, 1)
    assert state == (c.pages(a), c.pages(b), list(c._refs), sorted(c._free), c.version)
    assert c.length(b) == 20


def test_batches_hold_what_the_operators_take(cpu_copies):
    c = _cache()
    a, b, e = c.add(20), c.add(3), c.add(0)
    bat = c.batch([b, a, e], rows=[3, 2, 0])
    assert bat.page_table.dtype == bat.cache_lens.dtype == bat.query_starts.dtype == torch.int32
    assert bat.page_table.tolist() == [c.pages(b) + [-1], c.pages(a), [-1, -1]]
    assert bat.cache_lens.tolist() == [3, 20, 0] and bat.query_starts.tolist() == [0, 18, 0]
    assert bat.slots.tolist() == [[0, 1, 2], [18, 19, -1], [-1, -1, -1]]
    assert bat.positions.tolist() == [[0, 1, 2], [18, 19, 20], [0, 1, 2]]
    assert bat.max_len == 20
    empty = c.batch([e], rows=0)
    assert empty.page_table.shape == (1, 0) and empty.slots.shape == (1, 0)
    none = c.batch([])
    assert none.page_table.shape == (0, 0) and none.max_len == 0
    for bad in ([a, a], [77]):
        with pytest.raises(ValueError):
            c.batch(bad)
    for rows in (21, -1, [1], [1, 21]):
        with pytest.raises(ValueError):
            c.batch([a, b], rows=rows)


def test_out_of_date_batches_and_shared_rows_are_refused(cpu_copies):
    c = _cache()
    a, b = c.add(20), c.add(5)
    bat = c.batch([a], rows=4)
    k = torch.zeros(1, 4, 1, 1)
    c.extend(b, 1)
    c._current(bat)                      # other rows grew: still true
    c.free(b)
    with pytest.raises(ValueError, match="out of date"):
        c.append(0, bat, k, k)
    with pytest.raises(ValueError, match="out of date"):
        c.attend(0, bat, k)
    bat = c.batch([a], rows=4)
    twin = c.fork(a)
    with pytest.raises(ValueError, match="shared page"):
        c.append(0, bat, k, k)
    c.make_writable(twin, 0, 20)
    bat = c.batch([a], rows=4)
    c.truncate(a, 19)
    with pytest.raises(ValueError, match="out of date"):
        c.attend(0, bat, k)


def test_cache_argument_errors(cpu_copies):
    for bad in (dict(page_size=8), dict(page_size=24), dict(layers=0), dict(dtype=torch.int8)):
        args = dict(layers=1, num_pages=2, page_size=16, kv_heads=1, head_dim=64, device="cpu")
        args.update(bad)
        with pytest.raises(ValueError):
            mrsa.PagedKVCache(**args)
    c = _cache()
    a = c.add(3)
    for call in (lambda: c.add(-1), lambda: c.extend(a, -1), lambda: c.truncate(a, 4),
                 lambda: c.make_writable(a, 2, 5), lambda: c.free(9), lambda: c.length(9)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(mrsa.PagesExhausted):
        c.add(16 * 12)


# ---- refusals of the operators (fake CUDA tensors: checks run, kernels cannot)

def _rope_args():
    q = torch.empty(2, 5, 8, 128, dtype=torch.bfloat16, device="cuda")
    k = torch.empty(2, 5, 2, 128, dtype=torch.bfloat16, device="cuda")
    cos = torch.empty(9, 64, device="cuda")
    return dict(q=q, k=k, cos=cos, sin=torch.empty_like(cos))


def test_rotary_shapes_and_refusals():
    with FakeTensorMode():
        a = _rope_args()
        q, k = mrsa.rotary_qk(**a)
        assert q.shape == a["q"].shape and k.shape == a["k"].shape and k.dtype == torch.bfloat16
        assert mrsa.rotary_qk(**{**a, "k": None})[1] is None
        long = torch.empty(2, 5, dtype=torch.long, device="cuda")
        mrsa.rotary_qk(**a, positions=long)
        mrsa.rotary_qk(**a, positions=long[0])
        cpu = torch.empty(2, 5, 8, 128)
        bad = [
            dict(q=a["q"][0]), dict(q=cpu), dict(q=a["q"].double()), dict(k=a["k"][:, :4]),
            dict(k=a["k"].float()), dict(k=a["k"][..., :64]), dict(cos=a["cos"][:4]),
            dict(cos=a["cos"].double()), dict(cos=a["cos"].cpu()), dict(positions=long.int()),
            dict(positions=long[:1]), dict(positions=long.cpu()),
            dict(cos=torch.empty(9, 65, device="cuda"), sin=torch.empty(9, 65, device="cuda")),
            dict(cos=a["cos"][:4], sin=a["sin"][:4]),  # 5 rows do not fit 4 positions
        ]
        for change in bad:
            with pytest.raises(ValueError):
                mrsa.rotary_qk(**{**a, **change})
        with pytest.raises(ValueError, match="no gradient"):
            mrsa.rotary_qk(**{**a, "cos": a["cos"].requires_grad_()})


@pytest.mark.parametrize("kwargs", [
    dict(rotary_dim=5), dict(rotary_dim=0), dict(rotary_dim=8, scaling="other"),
    dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, factor=0.0),
    dict(rotary_dim=2, scaling="ntk", factor=2.0),
    dict(rotary_dim=8, scaling="yarn", factor=2.0, beta_fast=1.0),
])
def test_frequency_refusals(kwargs):
    with pytest.raises(ValueError):
        mrsa.rotary_frequencies(**kwargs)


def _paged_args():
    pool = torch.empty(7, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
    return dict(q=torch.empty(3, 4, 8, 128, dtype=torch.bfloat16, device="cuda"), k_pages=pool,
                v_pages=torch.empty_like(pool),
                page_table=torch.empty(3, 5, dtype=torch.int32, device="cuda"),
                cache_lens=torch.empty(3, dtype=torch.int32, device="cuda"))


def test_paged_attention_shapes_and_refusals():
    with FakeTensorMode():
        a = _paged_args()
        out, lse = mrsa.paged_cached_attention(**a, query_starts=a["cache_lens"], window=3)
        assert out.shape == a["q"].shape and out.dtype == torch.bfloat16
        assert lse.shape == (3, 4, 8) and lse.dtype == torch.float32
        p, t = a["k_pages"], a["page_table"]
        bad = [
            dict(q=a["q"].float(), k_pages=p.float(), v_pages=p.float()), dict(q=a["q"].half()),
            dict(q=a["q"][0]), dict(q=a["q"][:, :, :7]), dict(q=a["q"][..., :96]),
            dict(v_pages=p[:6]), dict(v_pages=p.half()), dict(k_pages=p.cpu()),
            dict(k_pages=p[:, :8], v_pages=p[:, :8]),
            dict(k_pages=p.transpose(2, 3).contiguous().transpose(2, 3)),
            dict(page_table=t.long()), dict(page_table=t[:2]), dict(page_table=t.cpu()),
            dict(cache_lens=a["cache_lens"].long()), dict(cache_lens=a["cache_lens"][:2]),
            dict(query_starts=a["cache_lens"].long()), dict(window=-1), dict(max_len=-1),
            dict(q=a["q"].clone().requires_grad_()),
        ]
        for change in bad:
            with pytest.raises(ValueError):
                mrsa.paged_cached_attention(**{**a, **change})


def test_paged_append_shapes_and_refusals():
    with FakeTensorMode():
        p = _paged_args()
        k = torch.empty(3, 4, 2, 128, dtype=torch.bfloat16, device="cuda")
        cos = torch.empty(9, 32, device="cuda")
        slots = torch.empty(3, 4, dtype=torch.long, device="cuda")
        a = dict(k=k, v=torch.empty_like(k), k_pages=p["k_pages"], v_pages=p["v_pages"],
                 page_table=p["page_table"], slots=slots)
        assert mrsa.paged_cache_append(**a) is None
        assert mrsa.paged_cache_append(**a, q=p["q"], cos=cos, sin=cos).shape == p["q"].shape
        bad = [
            dict(v=k[:, :3]), dict(v=k.half()), dict(k=k.cpu()), dict(slots=slots.int()),
            dict(slots=slots[:2]), dict(cos=cos), dict(positions=slots),
            dict(k=k[:, :, :1], v=k[:, :, :1]),
            dict(k_pages=p["k_pages"][:1].expand(7, 16, 2, 128)), dict(q=p["q"][:, :3]),
            dict(q=p["q"].half()), dict(page_table=p["page_table"][:1]),
            dict(k=k.clone().requires_grad_()),
        ]
        for change in bad:
            with pytest.raises(ValueError):
                mrsa.paged_cache_append(**{**a, **change})


def test_copy_refusals():
    with FakeTensorMode():
        p = torch.empty(2, 7, 16, 2, 64, device="cuda")
        v = torch.empty_like(p)
        mrsa.copy_cache_pages(p, v, [0], [1])
        for args in [(p, v[:1], [0], [1]), (p, v.half(), [0], [1]), (p[0, 0], v[0, 0], [0], [1]),
                     (p, v, [0, 1], [2]), (p.cpu(), v, [0], [1]),
                     (p[:, :1].expand(2, 7, 16, 2, 64), v, [0], [1]),
                     (p.transpose(2, 3), v.transpose(2, 3), [0], [1])]:
            with pytest.raises(ValueError):
                mrsa.copy_cache_pages(*args)


def _c_copy(src, dst, pages=7, page_bytes=4096, layers=2, align=0, count=None):
    """mrsa_copy_pages up to its launch: with page_bytes 0 a good call copies nothing."""
    import ctypes

    n = len(src)
    a, b = (ctypes.c_int64 * max(n, 1))(*src), (ctypes.c_int64 * max(n, 1))(*dst)
    return _lib.call("mrsa_copy_pages", 4096 + align, 4096 * pages, 4096, 8192, 4096 * pages, 4096,
                     layers, pages, page_bytes, n if count is None else count,
                     ctypes.addressof(a), ctypes.addressof(b), None)


def test_c_copy_pages_refuses_bad_pages_before_any_launch():
    assert _c_copy([0, 1], [2, 3], page_bytes=0) == _lib.MRSA_OK
    assert _c_copy([0, 0], [2, 3], page_bytes=0) == _lib.MRSA_OK
    for src, dst in [([7], [0]), ([-1], [0]), ([0], [7]), ([0], [-1]), ([0, 1], [2, 2]),
                     ([0, 2], [2, 3]), ([0], [0]), ([2 ** 32], [1])]:
        for page_bytes in (0, 4096):
            assert _c_copy(src, dst, page_bytes=page_bytes) == _lib.MRSA_ERR_INVALID_ARGUMENT
    assert _c_copy([0], [1], page_bytes=-1) == _lib.MRSA_ERR_INVALID_ARGUMENT
    assert _c_copy([0], [1], count=-1) == _lib.MRSA_ERR_INVALID_ARGUMENT
    assert _c_copy([0], [1], pages=0) == _lib.MRSA_ERR_INVALID_ARGUMENT
    assert _c_copy([0], [1], align=8) == _lib.MRSA_ERR_UNSUPPORTED
    assert _c_copy([0], [1], page_bytes=24) == _lib.MRSA_ERR_UNSUPPORTED
    assert _c_copy([], []) == _lib.MRSA_OK


def _c_attend(**change):
    a = dict(B=1, Lq=1, Hq=4, Hkv=2, D=128, dtype=0, P=16, width=4, pages=7, max_len=64, window=-1,
             scale=1.0, parts=1, ws=None, bytes=0, q=4096, k=4096, sr=256)
    a.update(change)
    s = (512, 512, 128)
    return _lib.call("mrsa_paged_attention_fwd", a["q"], *s, a["k"], 8192, a["sr"], 128, 4096, 8192,
                     256, 128, 4096, 4, a["width"], a["pages"], a["P"], 4096, None, a["max_len"],
                     a["B"], a["Lq"], a["Hq"], a["Hkv"], a["D"], a["dtype"], 0, a["window"],
                     a["scale"], a["parts"], a["ws"], a["bytes"], 4096, 4096, None)


def test_c_paged_attention_refusals():
    for change in (dict(B=0), dict(Lq=0)):
        assert _c_attend(**change) == _lib.MRSA_OK
    for change in (dict(B=-1), dict(Lq=-1), dict(Hq=5), dict(Hkv=0), dict(max_len=-1),
                   dict(parts=0), dict(parts=1025), dict(scale=0.0), dict(scale=float("nan")),
                   dict(scale=float("inf")), dict(q=None), dict(k=None), dict(P=0),
                   dict(parts=2), dict(parts=2, ws=4096, bytes=8)):
        assert _c_attend(**change) == _lib.MRSA_ERR_INVALID_ARGUMENT, change
    for change in (dict(D=96), dict(dtype=2), dict(P=8), dict(P=48), dict(q=4104), dict(sr=260),
                   dict(max_len=1 << 29), dict(Lq=1 << 29)):
        assert _c_attend(**change) == _lib.MRSA_ERR_UNSUPPORTED, change
    size = lambda *a: _lib.call("mrsa_paged_attention_workspace_bytes", *a)  # noqa: E731
    assert size(2, 3, 8, 128, 1) == 0 and size(2, 3, 8, 128, 4) == 2 * 3 * 8 * 4 * 130 * 4
    assert size(2, 3, 8, 128, 0) == -1 and size(-1, 3, 8, 128, 2) == -1
    assert size(1 << 31, 1 << 31, 65536, 128, 1024) == -1


def test_c_rotary_and_append_refusals():
    def rotary(B=1, L=1, D=128, R=128, dtype=0, q=4096, cos=4096, rows=4):
        return _lib.call("mrsa_rotary_fwd", q, 512, 512, 128, None, 0, 0, 0, cos, 4096, rows, None,
                         0, 0, B, L, 4, 0, D, R, dtype, 0, 0, 4096, None, None)

    assert rotary(B=0) == rotary(L=0) == _lib.MRSA_OK
    for change in (dict(B=-1), dict(R=7), dict(R=130), dict(dtype=3), dict(dtype=-1), dict(q=None),
                   dict(cos=None), dict(D=0)):
        assert rotary(**change) == _lib.MRSA_ERR_INVALID_ARGUMENT, change
    assert rotary(B=1 << 20, L=1 << 20) == _lib.MRSA_ERR_UNSUPPORTED
    assert rotary(D=8192) == _lib.MRSA_ERR_UNSUPPORTED

    def append(L=1, P=16, slots=4096, table=4096, pool=4096, vpool=8192, v=4096, R=0, width=4):
        s = (512, 512, 128)
        return _lib.call("mrsa_paged_append_fwd", None, 0, 0, 0, 4096, *s, v, *s, None, None, 0,
                         None, 0, 0, slots, 1, 1, table, 4, width, 7, P, pool, *s, vpool, *s, 1, L,
                         0, 4, 128, R, 0, 0, None, None)

    assert append(L=0) == _lib.MRSA_OK
    for change in (dict(slots=None), dict(table=None), dict(pool=None), dict(vpool=None), dict(vpool=4096),
                   dict(v=None), dict(P=0),
                   dict(L=-1), dict(R=3), dict(width=-1)):
        assert append(**change) == _lib.MRSA_ERR_INVALID_ARGUMENT, change
    assert append(P=24) == _lib.MRSA_ERR_UNSUPPORTED


def test_c_refusals_of_sizes_past_a_launch():
    # strides of rows that the DMA's 32-bit offsets do not span, scales that leave fp32
    assert _c_attend(sr=1 << 26) == _lib.MRSA_ERR_UNSUPPORTED
    assert _c_attend(scale=3e38) == _lib.MRSA_ERR_INVALID_ARGUMENT
    # more threads than a launch holds
    for B in (1 << 26, 1 << 30):
        assert _c_attend(B=B) == _lib.MRSA_ERR_UNSUPPORTED
    big = 1 << 24
    assert _lib.call("mrsa_rotary_fwd", 4096, 512, 512, 33, None, 0, 0, 0, 4096, 4096, 4, None, 0,
                     0, big, 1, 64, 0, 33, 32, 0, 0, 0, 8192, None, None) == _lib.MRSA_ERR_UNSUPPORTED


def test_parts_are_refused_outside_their_range():
    with FakeTensorMode():
        a = _paged_args()
        for parts in (0, -1, 1025):
            with pytest.raises(ValueError):
                mrsa.paged_cached_attention(**a, parts=parts)
        mrsa.paged_cached_attention(**a, parts=1024)
