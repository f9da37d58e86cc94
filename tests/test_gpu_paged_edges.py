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
