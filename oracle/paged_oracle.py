"""Plain fp64 CPU forms of the rotary and paged-cache operators, from their
definitions: loops over sequences and heads, only visible keys ever touched."""

from __future__ import annotations

import torch


def rotary(x, cos, sin, positions=None, interleaved=False, inverse=False):
    """x [B, L, H, D] -> fp64: pairs of the first dims turned by row `position`."""

    B, L, _, D = x.shape
    half = cos.shape[1]
    if positions is None:
        positions = torch.arange(L)
    positions = positions.expand(B, L)
    out = x.double().clone()
    for b in range(B):
        for l in range(L):
            p = int(positions[b, l])
            if 0 <= p < cos.shape[0]:
                c, s = cos[p].double(), sin[p].double()
            else:
                c = s = torch.full((half,), float("nan"), dtype=torch.float64)
            if inverse:
                s = -s
            if interleaved:
                first, second = torch.arange(half) * 2, torch.arange(half) * 2 + 1
            else:
                first, second = torch.arange(half), torch.arange(half) + half
            x1, x2 = x[b, l, :, first].double(), x[b, l, :, second].double()
            out[b, l, :, first] = x1 * c - x2 * s
            out[b, l, :, second] = x2 * c + x1 * s
    return out


def rotary_magnitude(x, cos, sin, positions=None, interleaved=False):
    """|x1 c| + |x2 s| of each output (what its fp32 rounding scales with)."""

    return rotary(x.abs(), cos.abs(), -sin.abs(), positions, interleaved).abs().maximum(
        rotary(x.abs(), cos.abs(), sin.abs(), positions, interleaved).abs())


def place(page_table, b, slot, page_size, num_pages):
    """(page, row) of a slot of sequence b, or None."""

    if slot < 0 or slot // page_size >= page_table.shape[1]:
        return None
    page = int(page_table[b, slot // page_size])
    return (page, slot % page_size) if 0 <= page < num_pages else None


def append(rows, pages, page_table, slots):
    """A copy of pages [N, P, Hkv, D] with rows [B, L, Hkv, D] at their slots."""

    out = pages.clone()
    for b in range(rows.shape[0]):
        for l in range(rows.shape[1]):
            at = place(page_table, b, int(slots[b, l]), pages.shape[1], pages.shape[0])
            if at is not None:
                out[at[0], at[1]] = rows[b, l].to(pages.dtype)
    return out


def attention(q, k_pages, v_pages, page_table, cache_lens, query_starts=None, causal=False,
              window=None, sm_scale=None):
    """(out, lse, size, reach) in fp64: size = sum_j p_j |v_j| per output and
    reach = scale max_j sum_d |q_d k_jd| per row scale the rounding errors."""

    B, Lq, Hq, D = q.shape
    N, P, Hkv, _ = k_pages.shape
    scale = D ** -0.5 if sm_scale is None else sm_scale
    out = torch.zeros(B, Lq, Hq, D, dtype=torch.float64)
    size = torch.zeros_like(out)
    lse = torch.full((B, Lq, Hq), float("-inf"), dtype=torch.float64)
    reach = torch.zeros(B, Lq, Hq, dtype=torch.float64)
    for b in range(B):
        n = int(cache_lens[b])
        n = max(0, min(n, page_table.shape[1] * P))
        start = n - Lq if query_starts is None else int(query_starts[b])
        at = [place(page_table, b, j, P, N) for j in range(n)]
        for i in range(Lq):
            p = start + i
            if not 0 <= p < n:
                continue
            keys = [j for j in range(n) if at[j] is not None and (not causal or j <= p)
                    and (window is None or abs(j - p) <= window)]
            if not keys:
                continue
            page = torch.tensor([at[j][0] for j in keys])
            row = torch.tensor([at[j][1] for j in keys])
            for h in range(Hq):
                g = h // (Hq // Hkv)
                k, v = k_pages[page, row, g].double(), v_pages[page, row, g].double()
                qd = q[b, i, h].double()
                s = (k @ qd) * scale
                lse[b, i, h] = torch.logsumexp(s, 0)
                prob = (s - lse[b, i, h]).exp()
                out[b, i, h] = prob @ v
                size[b, i, h] = prob @ v.abs()
                reach[b, i, h] = (k.abs() @ qd.abs()).max() * scale
    return out, lse, size, reach
