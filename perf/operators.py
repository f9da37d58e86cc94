"""Rotary positions and the paged K/V cache as a program calls them.

Head counts and sizes are those of the package's own configurations (28 query
heads over 4 KV heads, head size 128, 64-token chunks, 32-token decode blocks, a
1280-key sliding window) and of the shapes it is tested at.  Values are seeded
N(0, 1) projections.

Families ("kind"):
    rotary  query and key heads rotated by their positions, alone or with the
            gradient of a training step                 mrsa.rotary_qk
    append  rows of new tokens rotated and written into the pages of several
            sequences                                   mrsa.paged_cache_append
    attend  a block of rows of each sequence against its pages
                                                        mrsa.paged_cached_attention
    pages   pages copied inside a pool, K and V of every layer
                                                        mrsa.copy_cache_pages
"""

import glob
import math
import os
import sys

import torch

sys.path[:0] = glob.glob(os.path.join(os.getcwd(), "mask-routed-*_amd"))

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _rotary(**more):
    return {"kind": "rotary", "batch": 1, "len": 1024, "heads": 28, "kv_heads": 4, "dim": 128,
            "part": 128, "interleaved": False, "reach": 16384, "type": "bf16", "train": False,
            **more}


def _append(**more):
    return {"kind": "append", "batch": 1, "len": 1, "heads": 28, "kv_heads": 4, "dim": 128,
            "part": 128, "interleaved": False, "reach": 16384, "page": 64, "type": "bf16",
            "padded": False, **more}


def _attend(**more):
    return {"kind": "attend", "batch": 1, "rows": 1, "len": 1024, "heads": 28, "kv_heads": 4,
            "dim": 128, "page": 64, "window": -1, "causal": False, "type": "bf16",
            "ragged": False, "after": 0, **more}


def _pages(**more):
    return {"kind": "pages", "layers": 28, "count": 8, "kv_heads": 4, "dim": 128, "page": 64,
            "type": "bf16", **more}


def listed():
    return [
        # a decode block of one sequence: the launch counts
        _rotary(name="rotary_block", len=32),
        # a layer's training step at the length trained at
        _rotary(name="rotary_train_16k", len=16384, train=True),
        # half of each head in neighbouring pairs, odd lengths, positions far out
        _rotary(name="rotary_part_far", batch=3, len=1003, heads=8, kv_heads=8, part=64,
                interleaved=True, reach=131072, type="fp16", train=True),
        # one new token of sixteen sequences
        _append(name="append_step", batch=16),
        # two prompts of a batch, the shorter padded
        _append(name="append_prompt", batch=2, len=8001, padded=True),
        # one new token of one short sequence: latency
        _attend(name="attend_1k", len=1000),
        # one new token against one long cache: everything is in the split
        _attend(name="attend_128k", len=131072),
        # one new token of many sequences of different lengths: the cache's bytes
        _attend(name="attend_64x8k", batch=64, len=8192, ragged=True),
        # a decode block against a long cache: the matrix products
        _attend(name="attend_block_64k", rows=32, len=65503),
        # decode blocks of a sliding-window layer with a block cached behind them, small pages
        _attend(name="attend_window", batch=8, rows=32, len=16384, window=1280, page=16,
                ragged=True, after=32),
        # the last, shared pages of eight forked sequences
        _pages(name="pages_fork", count=8),
        # a pool of many sequences made dense again
        _pages(name="pages_compact", count=300),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    return rng.choice([(28, 4), (28, 4), (14, 2), (32, 8), (8, 8), (16, 1), (32, 4)])


def draw(rng):
    kind = rng.choice(["rotary", "append", "attend", "attend", "attend", "attend", "pages"])
    heads, kv_heads = _heads(rng)
    dim = rng.choice([128, 128, 64])
    type_ = rng.choice(["bf16", "bf16", "fp16"])
    page = rng.choice([16, 32, 64, 64, 128])
    if kind == "rotary":
        batch = rng.choice([1, 1, 2, 5])
        return _rotary(batch=batch, len=_log_int(rng, 1, 8192 / batch), heads=heads,
                       kv_heads=kv_heads, dim=dim, part=rng.choice([dim, dim, dim // 2]),
                       interleaved=rng.random() < 0.4, reach=rng.choice([8192, 131072]),
                       type=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                       train=rng.random() < 0.5)
    if kind == "append":
        batch = _log_int(rng, 1, 64)
        return _append(batch=batch, len=rng.choice([1, 32, _log_int(rng, 1, 8192 / batch)]),
                       heads=heads, kv_heads=kv_heads, dim=dim, part=rng.choice([dim, dim // 2]),
                       interleaved=rng.random() < 0.4, page=page, type=type_,
                       padded=rng.random() < 0.5)
    if kind == "attend":
        batch = _log_int(rng, 1, 64)
        rows = rng.choice([1, 1, 1, 4, 32, _log_int(rng, 1, 64)])
        # no more bytes than 64 sequences of 8192, no more products than a block at 64k
        most = min(131072, 64 * 8192 * 4 * 128 / (batch * kv_heads * dim),
                   32 * 65503 * 28 * 128 / (batch * rows * heads * dim))
        length = _log_int(rng, rows, most)
        # (the shortest of ragged sequences, an eighth as long, still holds its block)
        after = rng.choice([0, 0, 0, 100]) if length > 8 * (rows + 100) else 0
        return _attend(batch=batch, rows=rows, len=length, heads=heads, kv_heads=kv_heads, dim=dim,
                       page=page, window=rng.choice([-1, -1, -1, 319, 1280]),
                       causal=rng.random() < 0.3, type=type_, ragged=rng.random() < 0.6,
                       after=after)
    return _pages(layers=rng.choice([1, 7, 28]), count=_log_int(rng, 1, 300), kv_heads=kv_heads,
                  dim=dim, page=rng.choice([16, 32, 64]) if kv_heads < 8 else 16, type=type_)


def _lens(c):
    """Rows in use of each sequence: all alike, or spread between an eighth and the whole."""
    if not c["ragged"]:
        return [c["len"]] * c["batch"]
    n = c["batch"]
    return [max(1, c["len"] * (n + 7 * ((5 * b + 3) % n + 1)) // (8 * n)) for b in range(n)]


def _tokens(c):
    """Tokens that each sequence of an append brings."""
    return [c["len"] - (b * c["len"] // 3 if c["padded"] and b < 2 else 0)
            for b in range(c["batch"])]


def _tables(reach, part, device):
    """cos and sin of every position's angles, computed in 64 bits: rows [reach, part / 2]."""
    inv = 1.0e6 ** (-torch.arange(0, part, 2, dtype=torch.float64, device=device) / part)
    angles = torch.arange(reach, dtype=torch.float64, device=device)[:, None] * inv
    return angles.cos().float(), angles.sin().float()


def _paging(lens, page, gen, device, spare):
    """A pool's page count and the table of its sequences: pages in random order, -1 past the end."""
    need = [-(-n // page) for n in lens]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=gen, device=device).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=device)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return pool, table


def prepare(case, seed):
    c, device = case, torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    dtype = TYPES[c["type"]]

    def normal(*size):
        return torch.empty(*size, dtype=dtype, device=device).normal_(0.0, 1.0, generator=gen)

    s = {"case": c}
    if c["kind"] == "pages":
        # twice the pages moved, and an odd few that stay
        pool = 2 * c["count"] + 5
        size = (c["layers"], pool, c["page"], c["kv_heads"], c["dim"])
        s["k_pages"], s["v_pages"] = normal(*size), normal(*size)
        order = torch.randperm(pool, generator=gen, device=device).tolist()
        s["src"], s["dst"] = order[:c["count"]], order[c["count"]:2 * c["count"]]
        return s
    B, H, Hkv, D = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "rotary":
        L = c["len"]
        s["q"], s["k"] = normal(B, L, H, D), normal(B, L, Hkv, D)
        s["grad_q"], s["grad_k"] = normal(B, L, H, D), normal(B, L, Hkv, D)
        s["cos"], s["sin"] = _tables(c["reach"], c["part"], device)
        # each sequence starts somewhere and goes on from there
        start = torch.randint(0, max(1, c["reach"] - L), (B, 1), generator=gen, device=device)
        s["positions"] = start + torch.arange(L, device=device)
        return s
    if c["kind"] == "append":
        L, tokens = c["len"], _tokens(c)
        s["q"], s["k"], s["v"] = normal(B, L, H, D), normal(B, L, Hkv, D), normal(B, L, Hkv, D)
        s["cos"], s["sin"] = _tables(c["reach"], c["part"], device)
        # the rows come after a cached prefix of another length for each sequence
        prefix = [(37 * b + 61) % 500 for b in range(B)]
        pool, s["page_table"] = _paging([p + t for p, t in zip(prefix, tokens)], c["page"], gen,
                                        device, 3)
        s["k_pages"] = normal(pool, c["page"], Hkv, D)
        s["v_pages"] = normal(pool, c["page"], Hkv, D)
        rows = torch.arange(L, device=device)[None, :]
        slots = rows + torch.tensor(prefix, device=device)[:, None]
        s["slots"] = torch.where(rows < torch.tensor(tokens, device=device)[:, None], slots, -1)
        s["positions"] = slots
        return s
    lens = _lens(c)
    pool, s["page_table"] = _paging(lens, c["page"], gen, device, 3)
    s["q"] = normal(B, c["rows"], H, D)
    s["k_pages"] = normal(pool, c["page"], Hkv, D)
    s["v_pages"] = normal(pool, c["page"], Hkv, D)
    s["cache_lens"] = torch.tensor(lens, dtype=torch.int32, device=device)
    s["max_len"] = max(lens)
    # the block is the newest rows, or has some rows cached behind it
    s["query_starts"] = s["cache_lens"] - c["rows"] - c["after"] if c["after"] else None
    return s


def _turn(x, cos, sin, interleaved):
    """x [B, L, H, D] in 32 bits with its first pairs turned by the angles [B, L, part / 2]."""
    c, s = cos[:, :, None, :], sin[:, :, None, :]
    half = c.shape[-1]
    rest = x[..., 2 * half:]
    if interleaved:
        x1, x2 = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1).flatten(-2)
    else:
        x1, x2 = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _run_rotary(s):
    c = s["case"]
    if own:
        import mrsa

        if not c["train"]:
            return mrsa.rotary_qk(s["q"], s["k"], s["cos"], s["sin"], s["positions"],
                                  interleaved=c["interleaved"])
        q, k = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
        out = mrsa.rotary_qk(q, k, s["cos"], s["sin"], s["positions"],
                             interleaved=c["interleaved"])
        grads = torch.autograd.grad(out, (q, k), (s["grad_q"], s["grad_k"]))
        return [t.detach() for t in out] + list(grads)
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]

    def turn(x, sign):
        return _turn(x.float(), cos, sign * sin, c["interleaved"]).to(x.dtype)

    out = [turn(s["q"], 1.0), turn(s["k"], 1.0)]
    if c["train"]:  # the transpose of a rotation turns the other way
        out += [turn(s["grad_q"], -1.0), turn(s["grad_k"], -1.0)]
    return out


def _run_append(s):
    c = s["case"]
    if own:
        import mrsa

        q = mrsa.paged_cache_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"],
                                    s["slots"], q=s["q"], cos=s["cos"], sin=s["sin"],
                                    positions=s["positions"], interleaved=c["interleaved"])
        return q, s["k_pages"], s["v_pages"]
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    q = _turn(s["q"].float(), cos, sin, c["interleaved"]).to(s["q"].dtype)
    k = _turn(s["k"].float(), cos, sin, c["interleaved"]).to(s["k"].dtype)
    # a row that is not written repeats the first row of its sequence, which is
    slots = torch.where(s["slots"] >= 0, s["slots"], s["slots"][:, :1])
    skip = (s["slots"] < 0)[..., None, None]
    page = s["page_table"].long().gather(1, slots // c["page"])
    at = (page, slots % c["page"])
    s["k_pages"].index_put_(at, torch.where(skip, k[:, :1], k))
    s["v_pages"].index_put_(at, torch.where(skip, s["v"][:, :1], s["v"]))
    return q, s["k_pages"], s["v_pages"]


def _run_attend(s):
    c = s["case"]
    window = None if c["window"] < 0 else c["window"]
    if own:
        import mrsa

        return mrsa.paged_cached_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"],
                                           s["cache_lens"], causal=c["causal"], window=window,
                                           query_starts=s["query_starts"],
                                           max_len=s["max_len"])
    q, lens, page = s["q"], s["cache_lens"].long()[:, None], c["page"]
    B, R, H, D = q.shape
    Hkv, G = c["kv_heads"], H // c["kv_heads"]
    # the last rows of each sequence that any of its queries can see
    span = s["max_len"] if window is None else min(s["max_len"], R + c["after"] + window)
    j = lens - span + torch.arange(span, device=q.device)                       # [B, span]
    there = j >= 0
    at = j.clamp(min=0)
    pages = s["page_table"].long().gather(1, at // page)
    k = s["k_pages"][pages, at % page].permute(0, 2, 3, 1).contiguous().float()  # [B, Hkv, D, span]
    v = s["v_pages"][pages, at % page].permute(0, 2, 1, 3).contiguous().float()  # [B, Hkv, span, D]
    p = lens - R - c["after"] + torch.arange(R, device=q.device)                # [B, R]
    seen = there[:, None, :] & (p >= 0)[:, :, None]
    if c["causal"]:
        seen = seen & (j[:, None, :] <= p[:, :, None])
    if window is not None:
        seen = seen & ((j[:, None, :] - p[:, :, None]).abs() <= window)
    seen = seen[:, None, :, None, :]
    rows = q.float().reshape(B, R, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, R * G, D)
    score = torch.matmul(rows * D ** -0.5, k).reshape(B, Hkv, R, G, span)
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(dim=-1, keepdim=True).clamp(min=-1e30)
    e = (score - top).exp()
    total = e.sum(dim=-1, keepdim=True)
    out = torch.matmul(e.reshape(B, Hkv, R * G, span), v).reshape(B, Hkv, R, G, D)
    out = torch.where(total > 0, out / total, 0.0)
    lse = torch.where(total > 0, top + total.log(), float("-inf"))[..., 0]
    return (out.permute(0, 2, 1, 3, 4).reshape(B, R, H, D).to(q.dtype),
            lse.permute(0, 2, 1, 3).reshape(B, R, H))


def _run_pages(s):
    if own:
        import mrsa

        mrsa.copy_cache_pages(s["k_pages"], s["v_pages"], s["src"], s["dst"])
        return s["k_pages"], s["v_pages"]
    src = torch.tensor(s["src"], device=s["k_pages"].device)
    dst = torch.tensor(s["dst"], device=s["k_pages"].device)
    for pool in (s["k_pages"], s["v_pages"]):
        pool.index_copy_(1, dst, pool.index_select(1, src))
    return s["k_pages"], s["v_pages"]


def run(state):
    kind = state["case"]["kind"]
    if kind == "rotary":
        return _run_rotary(state)
    if kind == "append":
        return _run_append(state)
    return _run_attend(state) if kind == "attend" else _run_pages(state)


def _visible(c):
    """Keys that some query of each sequence sees, and pairs of a query and a key that it sees."""
    keys = pairs = 0
    for n in _lens(c):
        first, last = n, 0
        for i in range(c["rows"]):
            p = n - c["rows"] - c["after"] + i
            lo, hi = 0, n - 1 if p >= 0 else -1
            if c["causal"]:
                hi = min(hi, p)
            if c["window"] >= 0:
                lo, hi = max(lo, p - c["window"]), min(hi, p + c["window"])
            if hi >= lo:
                pairs += hi - lo + 1
                first, last = min(first, lo), max(last, hi + 1)
        keys += max(0, last - first)
    return keys, pairs


def work(case):
    c = case
    size = SIZES[c["type"]]
    if c["kind"] == "pages":
        page = c["page"] * c["kv_heads"] * c["dim"] * size
        return {"bytes": 2 * 2 * c["layers"] * c["count"] * page, "flops": 0}
    if c["kind"] == "rotary":
        tokens, steps = c["batch"] * c["len"], 2 if c["train"] else 1
        elements = tokens * (c["heads"] + c["kv_heads"]) * c["dim"]
        return {"bytes": steps * 2 * elements * size + tokens * (4 * c["part"] + 8),
                "flops": steps * 3 * tokens * (c["heads"] + c["kv_heads"]) * c["part"]}
    if c["kind"] == "append":
        tokens, rows = sum(_tokens(c)), c["batch"] * c["len"]
        elements = rows * c["heads"] + tokens * 2 * c["kv_heads"]
        return {"bytes": 2 * elements * c["dim"] * size + rows * (4 * c["part"] + 16),
                "flops": 3 * c["part"] * (rows * c["heads"] + tokens * c["kv_heads"])}
    keys, pairs = _visible(c)
    out = c["batch"] * c["rows"] * c["heads"]
    return {"bytes": keys * 2 * c["kv_heads"] * c["dim"] * size + out * (2 * c["dim"] * size + 4),
            "flops": 4 * pairs * c["heads"] * c["dim"]}


def _exact_turn(x, cos, sin, interleaved):
    """The pairs as complex numbers times cos + i sin."""
    half = cos.shape[-1]
    by = torch.complex(cos.double(), sin.double())[:, :, None, :]
    y = x.double().clone()
    if interleaved:
        pair = torch.view_as_complex(y[..., :2 * half].reshape(*y.shape[:-1], half, 2).contiguous())
        y[..., :2 * half] = torch.view_as_real(pair * by).reshape(*y.shape[:-1], 2 * half)
    else:
        pair = torch.complex(y[..., :half], y[..., half:2 * half]) * by
        y[..., :half], y[..., half:2 * half] = pair.real, pair.imag
    return y


def exact(case, seed):
    c = case
    if c["kind"] == "pages":  # nothing is computed
        return None
    s = prepare(case, seed)
    if c["kind"] == "rotary":
        cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
        out = [_exact_turn(s[n], cos, sin, c["interleaved"]) for n in ("q", "k")]
        if c["train"]:
            out += [_exact_turn(s[n], cos, -sin, c["interleaved"]) for n in ("grad_q", "grad_k")]
        return out
    if c["kind"] == "append":
        cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
        k = _exact_turn(s["k"], cos, sin, c["interleaved"])
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        for b in range(c["batch"]):
            got = (s["slots"][b] >= 0).nonzero()[:, 0]
            at = s["slots"][b, got]
            page = s["page_table"][b].long()[at // c["page"]]
            k_pages[page, at % c["page"]] = k[b, got]
            v_pages[page, at % c["page"]] = s["v"][b, got].double()
        return _exact_turn(s["q"], cos, sin, c["interleaved"]), k_pages, v_pages
    B, R, H, D = s["q"].shape
    G = H // c["kv_heads"]
    out = torch.zeros(B, R, H, D, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((B, R, H), float("-inf"), dtype=torch.float64, device=s["q"].device)
    for b, n in enumerate(_lens(c)):
        own_pages = s["page_table"][b, :-(-n // c["page"])].long()
        at = torch.arange(n, device=out.device)
        p0 = n - R - c["after"]
        far = at[None, :] - torch.arange(p0, p0 + R, device=out.device)[:, None]  # j - p
        seen = (at[None, :] - far) >= 0
        if c["causal"]:
            seen &= far <= 0
        if c["window"] >= 0:
            seen &= far.abs() <= c["window"]
        for h in range(H):
            k = s["k_pages"][own_pages, :, h // G].reshape(-1, D)[:n].double()
            v = s["v_pages"][own_pages, :, h // G].reshape(-1, D)[:n].double()
            t = (s["q"][b, :, h].double() @ k.T) / math.sqrt(D)
            t = t.masked_fill(~seen, float("-inf"))
            lse[b, :, h] = torch.logsumexp(t, dim=-1)
            p = (t - lse[b, :, h, None]).exp()
            out[b, :, h] = torch.nan_to_num(p, nan=0.0) @ v
    return out, lse
