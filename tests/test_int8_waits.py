"""The 8-bit matrix product's operands, brought to LDS by DMA, are waited for before the
barrier that hands them to the other waves: read off the gfx950 assembly, since a missing wait
rarely shows in results.  (CPU: cross-compiled.)"""

import os
import re

import pytest

from test_dma_waits import HIPCC, device_assembly


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_int8_tiles_wait_for_their_operands_before_the_barrier(tmp_path):
    text = device_assembly("int8_linear", tmp_path / "int8.s")
    kernels = re.findall(r"^(_ZN\S*int8_tile_kernelI\S*?Li(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)EEELb1E"
                         r"\S*):(.*?)^\.Lfunc_end", text, re.S | re.M)
    assert len(kernels) >= 2  # tile sizes, rows by DMA
    for name, tm, tn, wm, wn, ws, xs, body in kernels:
        assert "global_load_lds_dwordx4" in body, name
        # a wave's DMA instructions of a step of W and of X: its KB
        of_w, of_x = (int(n) * 128 // 1024 // (int(wm) * int(wn)) for n in (tn, tm))
        # The barriers of the first step and of the steady state, each behind a wait for the
        # wave's own rows (those of the further steps that fit the slots may be on their way) and
        # for its reads of the slot that is filled next; and those of the last steps, behind all.
        waits = re.findall(r"s_waitcnt vmcnt\((\d+)\) lgkmcnt\(0\)\n\s*s_barrier", body)
        assert len(waits) == len(re.findall(r"\bs_barrier\b", body)) >= 4, name
        assert (int(ws), int(xs)) == (3, 2) or ws == xs
        ahead = of_w if ws != xs else (of_w + of_x) * (int(xs) - 2)
        assert sorted(set(map(int, waits))) == sorted({0, ahead}), (name, waits)
        assert ahead < 64, name   # (what the counter holds)
