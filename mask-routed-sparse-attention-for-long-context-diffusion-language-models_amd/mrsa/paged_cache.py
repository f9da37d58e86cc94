"""A K/V cache of several sequences in pages, and the operators on it.

Beside ``LayerKVCache`` (one dense sequence of one layer): a pool of pages of
``page_size`` rows that sequences of different lengths share.  A page table row lists
the pages of a sequence in order; row s of a sequence (its "slot") is row
s % page_size of page table[s // page_size].

    paged_cache_append      new K/V rows into their pages, rotated on the way
    paged_cached_attention  a block of rows of each sequence against its pages
    copy_cache_pages        pages copied inside the pool, all layers at once
    PagedKVCache            the host's book-keeping: add, extend, fork (pages shared until
                            written), truncate, free, compact

The operators have no derivative and refuse tensors that ask for one.
"""

from __future__ import annotations

import ctypes
import functools
import heapq
from dataclasses import dataclass, field
from typing import List, Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .rotary import (DTYPES, check_heads, check_tables, check_token_ints, dense_rows,
                     refuse_tangents)

MAX_PARTS = 1024


def _check_pool(k_pages, v_pages, heads) -> Tuple[int, int]:
    """(page_size, KV heads) of a layer's pages."""

    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError(f"k_pages and v_pages must have one shape [pages, page_size, Hkv, D], got "
                         f"{tuple(shape)} and {tuple(v_pages.shape)}")
    _, P, Hkv, D = shape
    if P < 16 or P & (P - 1):
        raise ValueError(f"page_size must be a power of two from 16 on, got {P}")
    device, dtype = heads.device, heads.dtype
    if (k_pages.device != device or v_pages.device != device or k_pages.dtype != dtype
            or v_pages.dtype != dtype):
        raise ValueError("k_pages and v_pages must have the device and dtype of the heads")
    if (k_pages.stride(3) != 1 or v_pages.stride(3) != 1) and D > 1:
        raise ValueError("k_pages and v_pages must have a dense last dim")
    if D != heads.shape[3]:
        raise ValueError(f"pages of head_dim {D} do not fit heads of {heads.shape[3]}")
    return P, Hkv


def _check_writable(pool, name: str) -> None:
    if 0 in pool.stride() and any(s == 0 and n > 1 for s, n in zip(pool.stride(), pool.shape)):
        raise ValueError(f"{name} must not be an expanded tensor")


def _check_table(page_table, batch: int, device) -> torch.Tensor:
    if page_table.ndim != 2 or page_table.shape[0] != batch:
        raise ValueError(f"page_table must have shape [{batch}, pages], got "
                         f"{tuple(page_table.shape)}")
    if page_table.dtype != torch.int32 or page_table.device != device:
        raise ValueError("page_table must be int32 on the device of the heads")
    return page_table if page_table.stride(1) == 1 or page_table.shape[1] <= 1 \
        else page_table.contiguous()


def _no_gradient(name: str, *tensors) -> None:
    """Refuse tensors whose derivative a caller would wait for in vain, in either mode."""

    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no gradient: call it under torch.no_grad()")
    if forward_ad._current_level >= 0:   # (of dual tensors and of torch.func.jvp)
        wrapped = torch._C._functorch.is_functorch_wrapped_tensor
        for t in tensors:
            if t is not None and (wrapped(t) or forward_ad.unpack_dual(t).tangent is not None):
                raise ValueError(f"{name} has no forward-mode derivative")


def _written(*pools) -> None:
    """Raise the version counters of pools that a kernel has written, as torch's own in-place
    operators do: backward passes that saved them and ``kv_fragments_cached`` go by it.
    (Tensors made in inference mode have none.)"""

    if pools[0].is_inference() or pools[1].is_inference():
        pools = [t for t in pools if not t.is_inference()]
    torch.autograd.graph.increment_version(pools)


def _paged_append_impl(k, v, k_pages, v_pages, page_table, slots, q, cos, sin, positions,
                       interleaved):
    refuse_tangents("mrsa::paged_append_", q, k, v, k_pages, v_pages)
    B, L, Hkv, D = k.shape
    kc, vc = dense_rows(k), dense_rows(v)
    kb, kl, kh, _ = kc.stride()
    vb, vl, vh, _ = vc.stride()
    if q is None:
        Hq, qp, qb, ql, qh = 0, None, 0, 0, 0
    else:
        qc = dense_rows(q)
        Hq, qp = q.shape[2], qc.data_ptr()
        qb, ql, qh, _ = qc.stride()
    q_out = k.new_empty((B, L, Hq, D))
    if cos is None:
        cp = sp = pp = None
        rows = half = pb = pl = 0
    else:
        ct, st = cos.contiguous(), sin.contiguous()
        cp, sp, pp = ct.data_ptr(), st.data_ptr(), positions.data_ptr()
        rows, half = cos.shape
        pb, pl = positions.stride()
    sb, sl = slots.stride()
    kps, kss, khs, _ = k_pages.stride()
    vps, vss, vhs, _ = v_pages.stride()
    pages, page_size = k_pages.shape[:2]
    status = _lib.call_on(
        k.device, "mrsa_paged_append_fwd", qp, qb, ql, qh, kc.data_ptr(), kb, kl, kh,
        vc.data_ptr(), vb, vl, vh, cp, sp, rows, pp, pb, pl, slots.data_ptr(), sb, sl,
        page_table.data_ptr(), page_table.stride(0), page_table.shape[1], pages, page_size,
        k_pages.data_ptr(), kps, kss, khs, v_pages.data_ptr(), vps, vss, vhs, B, L, Hq, Hkv, D,
        2 * half, DTYPES[k.dtype], interleaved, q_out.data_ptr(), _lib.stream_of(k))
    _lib.check(status, "paged_cache_append")
    _written(k_pages, v_pages)
    return q_out


def paged_cache_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor,
                       v_pages: torch.Tensor, page_table: torch.Tensor, slots: torch.Tensor, *,
                       q: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                       sin: Optional[torch.Tensor] = None,
                       positions: Optional[torch.Tensor] = None,
                       interleaved: bool = False) -> Optional[torch.Tensor]:
    """Write new K/V rows into their pages, in place, in one launch.

    k, v [B, L, Hkv, D] bf16, fp16 or fp32, any strides; slots torch.long [B, L]: the
    row of its sequence that each new row becomes.  A negative slot (a padded token),
    one past the table and one whose page is outside the pool are skipped.  Two rows
    of a call must not name the same cache row, as one of them would be left (also
    through a page that two sequences share), and q, k and v must not lie in the pages.
    With cos, sin (``rotary_tables``) k rows are turned as by ``rotary_qk`` at
    ``positions`` (torch.long [B, L] or [L]; None: the slots), the same bits; q
    [B, L, Hq, D], if given, is turned too, skipped rows as well, and returned (without
    tables: copied).
    """

    check_heads(k, "k")
    B, L, Hkv, D = k.shape
    if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise ValueError(f"k and v must have one shape, dtype and device, got {tuple(k.shape)} "
                         f"{k.dtype} and {tuple(v.shape)} {v.dtype}")
    _, pool_heads = _check_pool(k_pages, v_pages, k)
    if pool_heads != Hkv:
        raise ValueError(f"pages of {pool_heads} heads do not fit rows of {Hkv}")
    _check_writable(k_pages, "k_pages")
    _check_writable(v_pages, "v_pages")
    page_table = _check_table(page_table, B, k.device)
    slots = check_token_ints(slots, "slots", B, L, k.device)
    if q is not None:
        check_heads(q, "q")
        if q.shape != (B, L, q.shape[2], D) or q.dtype != k.dtype:
            raise ValueError(f"q and k must agree in batch, length, head_dim and dtype, got "
                             f"{tuple(q.shape)} {q.dtype} and {tuple(k.shape)} {k.dtype}")
        if q.device != k.device:
            raise ValueError("q and k must be on one device")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        check_tables(cos, sin, D, k.device)
        positions = slots if positions is None else check_token_ints(positions, "positions", B, L,
                                                                     k.device)
    elif positions is not None:
        raise ValueError("positions need cos and sin")
    _no_gradient("paged_cache_append", q, k, v, k_pages, v_pages)
    q_out = torch.ops.mrsa.paged_append_.default(k, v, k_pages, v_pages, page_table, slots, q, cos,
                                                 sin, positions, bool(interleaved))
    return None if q is None else q_out


@functools.lru_cache(maxsize=4096)
def cache_parts(batch: int, q_len: int, q_heads: int, kv_heads: int, span: int, live: int) -> int:
    """Pieces that paged_cached_attention cuts the visible span into: of those that make
    whole rounds of workgroups over the 256 CUs, the one with the least work for a CU.
    ``live``: the keys of the span that there are if the rows stand at their sequence's end.

    Up to 16 columns (rows and heads of a KV head; streaming kernel) a piece costs its
    keys, about 128 more to start, the uneven ends of sequences of different lengths, and
    its part in the join, which itself costs 512.  32 sequences of 500 keys: 1 piece 13.4 us,
    2 16.6; 1 of 500: 1 piece 11.0, 5 10.9; 1 of 1000: 1 piece 15.3, 8 11.0; 64 of 1024 to
    8192: 3 pieces 128, 1 143.  More columns (block kernel; in keys of 28 ns): a round costs
    230 to start and its keys, the join 140 and its bytes, 1 KB a column and piece, written
    and read.  64 sequences of 32 rows of 2048 keys: 1 piece 78 us, 3 140; 8 of 4096: 8
    pieces 39 us, 24 64; 1 of 8192: 48 pieces 29 us, 8 42."""

    cols = q_len * (q_heads // kv_heads)
    if cols == 0 or batch == 0 or span <= 0:
        return 1
    best, least = 1, None
    if cols <= 16:
        units = batch * kv_heads
        most = min(MAX_PARTS, -(-span // 128))
        for rounds in (0, 1, 2, 3, 4, 6):
            parts = max(1, min(most, 256 * rounds // units))
            keys = -(-(span + 31) // (parts * 128)) * 128   # (with room: lengths grow)
            cost = -(-units * parts // 256) * (keys + 128) + keys // 4 + 4 * parts
            if parts > 1:
                cost += 512
            if least is None or cost < least:
                best, least = parts, cost
        return best
    groups = -(-cols // 32)
    tiles = -(-groups // 8)
    units = batch * kv_heads * tiles
    slots = 256 if -(-groups // tiles) > 4 else 512   # workgroups at a time
    most = min(MAX_PARTS, -(-span // 64))
    for quarters in (0, 2, 3, 4, 8, 12, 16, 24):
        parts = max(1, min(most, slots * quarters * span // (4 * units * live)))
        keys = -(-span // (parts * 64)) * 64
        there = min(parts, -(-live // keys))
        cost = -(-units * there // slots) * (230 + keys)
        if slots == 512 and units * there > 256:   # two on a CU slow each other
            cost = cost * 13 // 10
        if parts > 1:
            cost += 140 + batch * kv_heads * cols * there // 120
        if least is None or cost < least:
            best, least = parts, cost
    return best


def _paged_attention_impl(q, k_pages, v_pages, page_table, cache_lens, query_starts, max_len,
                          causal, window, sm_scale, parts):
    refuse_tangents("mrsa::paged_attention", q, k_pages, v_pages)
    shape = q.shape
    B, Lq, Hq, D = shape
    qc = dense_rows(q)
    qb, ql, qh, _ = qc.stride()
    if (qb | ql | qh) % 8 or qc.data_ptr() % 16:
        qc = qc.clone(memory_format=torch.contiguous_format)
        qb, ql, qh, _ = qc.stride()
    kps, kss, khs, _ = k_pages.stride()
    vps, vss, vhs, _ = v_pages.stride()
    pages, page_size, Hkv, _ = k_pages.shape
    if parts == 0:  # (here, not in the caller, which a compiler traces)
        span = live = max_len
        if window >= 0:
            right = 0 if causal else window if query_starts is not None else min(window, Lq)
            span = min(max_len, min(Lq, 256) + window + right)
            live = min(span, min(Lq, 256) + window) + 31
            span += 31   # (a window's first tile may start before it)
        parts = cache_parts(B, Lq, Hq, Hkv, span, live)
    out = q.new_empty(shape)
    lse = q.new_empty((B, Lq, Hq), dtype=torch.float32)
    nbytes, wp = 0, None
    if parts > 1:
        ws = q.new_empty(B * Lq * Hq * parts * (D + 2), dtype=torch.float32)
        nbytes, wp = ws.numel() * 4, ws.data_ptr()
    status = _lib.call_on(
        q.device, "mrsa_paged_attention_fwd", qc.data_ptr(), qb, ql, qh, k_pages.data_ptr(), kps,
        kss, khs, v_pages.data_ptr(), vps, vss, vhs, page_table.data_ptr(), page_table.stride(0),
        page_table.shape[1], pages, page_size, cache_lens.data_ptr(), _lib.ptr(query_starts),
        max_len, B, Lq, Hq, Hkv, D, DTYPES[q.dtype], causal, window, sm_scale, parts, wp, nbytes,
        out.data_ptr(), lse.data_ptr(), _lib.stream_of(q))
    _lib.check(status, "paged_cached_attention")
    return out, lse


def _check_sequence_ints(t, name: str, batch: int, device) -> torch.Tensor:
    if t.shape != (batch,) or t.dtype != torch.int32 or t.device != device:
        raise ValueError(f"{name} must be int32 [{batch}] on the device of the heads")
    return t.contiguous()


def paged_cached_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                           page_table: torch.Tensor, cache_lens: torch.Tensor, *,
                           query_starts: Optional[torch.Tensor] = None, causal: bool = False,
                           window: Optional[int] = None, sm_scale: Optional[float] = None,
                           max_len: Optional[int] = None, parts: Optional[int] = None
                           ) -> Tuple[torch.Tensor, torch.Tensor]:
    """A block of rows of each sequence against its pages: (out, natural-log LSE).

    q [B, Lq, Hq, D] bf16 or fp16, D 64 or 128, any strides; k_pages, v_pages
    [pages, page_size, Hkv, D] (any order of the first three dims in memory, so a
    [pages, Hkv, page_size, D] pool is passed as its transpose(1, 2)); page_table int32
    [B, n]; cache_lens int32 [B]: rows of each sequence in the cache, with the query rows'
    own (``paged_cache_append`` comes first).  Row i of sequence b sits at position
    p = query_starts[b] + i (int32 [B]; None: the newest rows, cache_lens - Lq + i) and
    sees the keys j of [0, cache_lens[b]) with j <= p if causal and |j - p| <= window
    if given: by default all of them, as a denoised block does.  Table entries outside
    [0, pages) hold no keys.  Rows at positions outside [0, cache_lens[b]) are padding.
    Padding, and a row that sees no key, give out = 0 and lse = -inf.

    max_len: a bound of cache_lens that the caller knows (None: the table's rows; lengths
    past it are cut to it); it sizes the launch, and a captured call keeps it.  parts: pieces
    the span is cut into, None picks them.  sm_scale: above 0, D^-0.5 if None.  Returns out
    [B, Lq, Hq, D] in q's dtype and lse fp32 [B, Lq, Hq].
    """

    check_heads(q, "q")
    if q.dtype == torch.float32:
        raise ValueError("paged_cached_attention requires bf16 or fp16")
    B, Lq, Hq, D = q.shape
    if D not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {D}")
    page_size, Hkv = _check_pool(k_pages, v_pages, q)
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"query heads ({Hq}) must be divisible by KV heads ({Hkv})")
    page_table = _check_table(page_table, B, q.device)
    cache_lens = _check_sequence_ints(cache_lens, "cache_lens", B, q.device)
    if query_starts is not None:
        query_starts = _check_sequence_ints(query_starts, "query_starts", B, q.device)
    if window is not None and window < 0:
        raise ValueError(f"window must be >= 0, got {window}")
    rows = page_table.shape[1] * page_size
    if max_len is None:
        max_len = rows
    elif max_len < 0:
        raise ValueError(f"max_len must be >= 0, got {max_len}")
    max_len = min(int(max_len), rows)
    if sm_scale is None:
        sm_scale = D ** -0.5
    _no_gradient("paged_cached_attention", q, k_pages, v_pages)
    window = -1 if window is None else int(window)
    if parts is not None and not 1 <= parts <= MAX_PARTS:
        raise ValueError(f"parts must be in [1, {MAX_PARTS}], got {parts}")
    return torch.ops.mrsa.paged_attention.default(q, k_pages, v_pages, page_table, cache_lens,
                                                  query_starts, max_len, bool(causal), window,
                                                  float(sm_scale), int(parts or 0))


def _copy_pages_impl(k_pages, v_pages, src, dst):
    refuse_tangents("mrsa::copy_pages_", k_pages, v_pages)
    n = len(src)
    layered = k_pages.ndim == 5
    shape, ks, vs = k_pages.shape, k_pages.stride(), v_pages.stride()
    if not layered:
        shape, ks, vs = (1, *shape), (0, *ks), (0, *vs)
    size = k_pages.element_size()
    arrays = (ctypes.c_int64 * max(n, 1))(*src), (ctypes.c_int64 * max(n, 1))(*dst)
    status = _lib.call_on(
        k_pages.device, "mrsa_copy_pages", k_pages.data_ptr(), ks[0] * size, ks[1] * size,
        v_pages.data_ptr(), vs[0] * size, vs[1] * size, shape[0], shape[1],
        shape[2] * shape[3] * shape[4] * size, n, ctypes.addressof(arrays[0]),
        ctypes.addressof(arrays[1]), _lib.stream_of(k_pages))
    _lib.check(status, "copy_cache_pages")
    _written(k_pages, v_pages)


def copy_cache_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src: Sequence[int],
                     dst: Sequence[int]) -> None:
    """Page src[i] copied over page dst[i], K and V, in every layer, in place.

    k_pages, v_pages [pages, page_size, Hkv, D] or [layers, pages, page_size, Hkv, D]
    on the GPU, each page dense; src, dst: host integers.  ValueError, and nothing
    copied, for a page outside the pool, a destination named twice, or a destination
    that is also a source (the copies have no order)."""

    if k_pages.ndim not in (4, 5) or v_pages.shape != k_pages.shape:
        raise ValueError(f"k_pages and v_pages must have one shape [(layers,) pages, page_size, "
                         f"Hkv, D], got {tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    if k_pages.device.type != "cuda" or v_pages.device != k_pages.device:
        raise ValueError("k_pages and v_pages must be on one CUDA device")
    if v_pages.dtype != k_pages.dtype:
        raise ValueError("k_pages and v_pages must have one dtype")
    lead = k_pages.ndim - 3
    for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if not t.is_contiguous() and t.numel() and not t[(0,) * lead].is_contiguous():
            raise ValueError(f"the pages of {name} must be dense")
        _check_writable(t, name)
    src, dst = [int(i) for i in src], [int(i) for i in dst]
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} sources for {len(dst)} destinations")
    _no_gradient("copy_cache_pages", k_pages, v_pages)
    torch.ops.mrsa.copy_pages_.default(k_pages, v_pages, src, dst)


class PagesExhausted(RuntimeError):
    """The pool has too few free pages; nothing was changed."""


@dataclass(frozen=True)
class PagedBatch:
    """Some sequences of a PagedKVCache as the operators take them (device tensors)."""

    seqs: Tuple[int, ...]
    lens: Tuple[int, ...]      # rows of each sequence,
    rows: Tuple[int, ...]      # and how many of them, the newest, the call brings
    page_table: torch.Tensor   # int32 [B, n], -1 past a sequence's pages
    cache_lens: torch.Tensor   # int32 [B]
    query_starts: torch.Tensor  # int32 [B]: position of each sequence's first new row
    slots: torch.Tensor        # int64 [B, L]: slot of each new row, -1 for padding
    positions: torch.Tensor    # int64 [B, L]: the same without the -1
    max_len: int
    version: int


@dataclass
class _Sequence:
    pages: List[int] = field(default_factory=list)
    length: int = 0


class PagedKVCache:
    """Pages of all layers and the host's book-keeping of who holds which.

    Sequences are numbered by ``add`` and ``fork``; ``extend`` makes room for new rows,
    ``batch`` uploads what the operators need, ``append`` and ``attend`` run them on a
    layer.  Forked sequences share pages; a shared page is copied before one of
    them writes to it (``extend`` for the rows it adds, ``make_writable`` for rows
    rewritten).  fp32 pools can be written and copied, but not attended.  Not for use from
    several threads at once; page copies go to the current stream, where the operators have
    to follow."""

    def __init__(self, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int,
                 *, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if min(layers, num_pages, kv_heads, head_dim) < 1:
            raise ValueError("layers, num_pages, kv_heads and head_dim must be positive")
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 on, got {page_size}")
        if dtype not in DTYPES:
            raise ValueError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
        size = (layers, num_pages, page_size, kv_heads, head_dim)
        self.k_pages = torch.empty(size, dtype=dtype, device=device)
        self.v_pages = torch.empty(size, dtype=dtype, device=device)
        self.page_size, self.num_pages = page_size, num_pages
        self.version = 0          # rises when a page in use moves or rows go
        self._free = list(range(num_pages))   # a heap: the lowest page first
        self._refs = [0] * num_pages
        self._seqs: dict[int, _Sequence] = {}
        self._next = 0

    # ---- what is there
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def sequences(self) -> List[int]:
        return sorted(self._seqs)

    def length(self, seq: int) -> int:
        return self._get(seq).length

    def pages(self, seq: int) -> List[int]:
        return list(self._get(seq).pages)

    def _get(self, seq: int) -> _Sequence:
        try:
            return self._seqs[seq]
        except KeyError:
            raise ValueError(f"no sequence {seq}") from None

    def _need(self, count: int) -> None:
        if count > len(self._free):
            raise PagesExhausted(f"{count} pages wanted, {len(self._free)} of {self.num_pages} "
                                 "free")

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._refs[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            heapq.heappush(self._free, page)

    # ---- sequences
    def add(self, length: int = 0) -> int:
        """A new sequence with room for ``length`` rows, all of them new."""

        if length < 0:
            raise ValueError(f"length must be >= 0, got {length}")
        count = -(-length // self.page_size)
        self._need(count)
        seq, self._next = self._next, self._next + 1
        self._seqs[seq] = _Sequence([self._take() for _ in range(count)], length)
        return seq

    def extend(self, seq: int, count: int) -> range:
        """Room for ``count`` more rows; their slots.  A last page that is partly
        filled and shared is copied first."""

        s = self._get(seq)
        if count < 0:
            raise ValueError(f"count must be >= 0, got {count}")
        at, P = s.length, self.page_size
        more = -(-(at + count) // P) - len(s.pages)
        shared = [len(s.pages) - 1] if count and at % P and self._refs[s.pages[-1]] > 1 else []
        self._need(more + len(shared))
        self._own(s, shared)
        s.pages += [self._take() for _ in range(more)]
        s.length = at + count
        return range(at, at + count)

    def make_writable(self, seq: int, start: int, stop: int) -> int:
        """Copies of the shared pages that hold rows [start, stop), so that they can be
        rewritten; returns how many were copied."""

        s = self._get(seq)
        if not 0 <= start <= stop <= s.length:
            raise ValueError(f"rows [{start}, {stop}) are not in a sequence of {s.length}")
        if start == stop:
            return 0
        P = self.page_size
        shared = [i for i in range(start // P, -(-stop // P)) if self._refs[s.pages[i]] > 1]
        self._need(len(shared))
        self._own(s, shared)
        return len(shared)

    def _own(self, s: _Sequence, entries: List[int]) -> None:
        if not entries:
            return
        src = [s.pages[i] for i in entries]
        dst = [self._take() for _ in entries]
        try:
            copy_cache_pages(self.k_pages, self.v_pages, src, dst)
        except Exception:
            for page in dst:
                self._drop(page)
            raise
        for i, page in zip(entries, dst):
            self._drop(s.pages[i])
            s.pages[i] = page
        self.version += 1

    def fork(self, seq: int) -> int:
        """A new sequence with the rows of ``seq``, its pages shared."""

        s = self._get(seq)
        for page in s.pages:
            self._refs[page] += 1
        new, self._next = self._next, self._next + 1
        self._seqs[new] = _Sequence(list(s.pages), s.length)
        return new

    def truncate(self, seq: int, length: int) -> None:
        """Drop the rows from ``length`` on, and the pages that only held those."""

        s = self._get(seq)
        if not 0 <= length <= s.length:
            raise ValueError(f"length must be in [0, {s.length}], got {length}")
        keep = -(-length // self.page_size)
        if length < s.length:
            self.version += 1
        for page in s.pages[keep:]:
            self._drop(page)
        del s.pages[keep:]
        s.length = length

    def free(self, seq: int) -> None:
        """Drop a sequence and the pages that nobody else holds."""

        s = self._get(seq)
        for page in s.pages:
            self._drop(page)
        del self._seqs[seq]
        self.version += 1

    def compact(self) -> int:
        """Move the live pages to the front of the pool; returns how many there are."""

        live = self.num_pages - len(self._free)
        src = [p for p in range(live, self.num_pages) if self._refs[p]]
        dst = [p for p in range(live) if not self._refs[p]]
        if not src:
            return live
        copy_cache_pages(self.k_pages, self.v_pages, src, dst)
        to = dict(zip(src, dst))
        for s in self._seqs.values():
            s.pages = [to.get(p, p) for p in s.pages]
        for a, b in to.items():
            self._refs[b], self._refs[a] = self._refs[a], 0
        self._free = list(range(live, self.num_pages))
        self.version += 1
        return live

    # ---- the operators
    def batch(self, seqs: Sequence[int], rows=1, *, max_len: Optional[int] = None) -> PagedBatch:
        """What the operators need of some sequences, in one upload.  ``rows``: how many of
        each sequence's newest rows the call brings, one number or one per sequence; rows
        of shorter ones are padding behind theirs.

        ``max_len``: a length that no sequence passes while this batch is in use (None: the
        longest one's now).  It is the table's width and attention's bound, both of which a
        captured graph keeps: capture with a max_len that covers every replay, then copy the
        tensors of ``batch(seqs, rows, max_len=...)`` into the captured batch's before each."""

        seqs = tuple(int(s) for s in seqs)
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence can be in a batch once")
        held = [self._get(s) for s in seqs]
        counts = [int(rows)] * len(held) if isinstance(rows, int) else [int(r) for r in rows]
        if len(counts) != len(held):
            raise ValueError(f"{len(counts)} row counts for {len(held)} sequences")
        for s, r in zip(held, counts):
            if not 0 <= r <= s.length:
                raise ValueError(f"rows must be in [0, {s.length}], got {r}")
        B, L = len(held), max(counts, default=0)
        longest = max((s.length for s in held), default=0)
        if max_len is None:
            max_len = longest
        elif max_len < longest:
            raise ValueError(f"max_len must be at least {longest}, got {max_len}")
        width = -(-max_len // self.page_size)
        starts = [s.length - r for s, r in zip(held, counts)]
        row = torch.arange(L)
        positions = torch.tensor(starts, dtype=torch.long).view(B, 1) + row
        slots = torch.where(row < torch.tensor(counts, dtype=torch.long).view(B, 1), positions, -1)
        table = [s.pages + [-1] * (width - len(s.pages)) for s in held]
        ints = torch.tensor([x for r in table for x in r] + [s.length for s in held] + starts,
                            dtype=torch.int32)
        host = torch.empty(16 * B * L + 4 * ints.numel(), dtype=torch.uint8,
                           pin_memory=self.k_pages.is_cuda)
        host[:8 * B * L].view(torch.long).copy_(slots.reshape(-1))
        host[8 * B * L:16 * B * L].view(torch.long).copy_(positions.reshape(-1))
        host[16 * B * L:].view(torch.int32).copy_(ints)
        dev = host.to(self.k_pages.device, non_blocking=True)
        ints = dev[16 * B * L:].view(torch.int32)
        return PagedBatch(
            seqs=seqs, lens=tuple(s.length for s in held), rows=tuple(counts),
            page_table=ints[:B * width].view(B, width),
            cache_lens=ints[B * width:B * width + B], query_starts=ints[B * width + B:],
            slots=dev[:8 * B * L].view(torch.long).view(B, L),
            positions=dev[8 * B * L:16 * B * L].view(torch.long).view(B, L),
            max_len=int(max_len), version=self.version)

    def _current(self, batch: PagedBatch) -> None:
        if batch.version != self.version:
            raise ValueError("the batch is out of date: pages have moved since it was made")

    def append(self, layer: int, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor, **rotary):
        """``paged_cache_append`` of the batch's newest rows into a layer's pages; keywords q,
        cos, sin, positions (default: the rows' places) and interleaved as there."""

        self._current(batch)
        P = self.page_size
        for i, seq in enumerate(batch.seqs):
            start, stop = batch.lens[i] - batch.rows[i], batch.lens[i]
            held = self._get(seq).pages[start // P:-(-stop // P)] if start < stop else ()
            if any(self._refs[p] > 1 for p in held):
                raise ValueError(f"rows of sequence {seq} lie in a shared page: make_writable "
                                 "first")
        if rotary.get("cos") is not None and rotary.get("positions") is None:
            rotary["positions"] = batch.positions
        return paged_cache_append(k, v, self.k_pages[layer], self.v_pages[layer],
                                  batch.page_table, batch.slots, **rotary)

    def attend(self, layer: int, batch: PagedBatch, q: torch.Tensor, *,
               max_len: Optional[int] = None, **options):
        """``paged_cached_attention`` of the batch's newest rows against a layer's pages;
        keywords causal, window, sm_scale and parts as there.  max_len: a larger bound of the
        lengths than the batch's (a captured call keeps its bound, parts and table width)."""

        self._current(batch)
        if max_len is None:
            max_len = batch.max_len
        elif max_len < batch.max_len:
            raise ValueError(f"max_len must be at least the batch's {batch.max_len}, got {max_len}")
        return paged_cached_attention(q, self.k_pages[layer], self.v_pages[layer],
                                      batch.page_table, batch.cache_lens,
                                      query_starts=batch.query_starts, max_len=max_len, **options)
