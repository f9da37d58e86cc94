"""The paged block kernel's rows, brought to LDS by DMA, are waited for before the
barrier that hands them to the other waves: read off the gfx950 assembly, since a
missing wait rarely shows in results.  (CPU: cross-compiled.)"""

import os
import re

import pytest

from test_dma_waits import HIPCC, device_assembly


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_paged_block_tiles_wait_for_their_rows_before_the_barrier(tmp_path):
    text = device_assembly("paged_attention", tmp_path / "paged.s")
    kernels = re.findall(r"^(_ZN\S*paged_block_kernel\S*):(.*?)^\.Lfunc_end", text, re.S | re.M)
    assert len(kernels) == 8  # type x head dim x slots
    for name, body in kernels:
        assert "global_load_lds_dwordx4" in body, name
        waits = re.findall(r"s_waitcnt (vmcnt\(0\) )?lgkmcnt\(0\)\n\s*s_barrier", body)
        assert len(waits) == len(re.findall(r"\bs_barrier\b", body)) > 1, name
        # all but the one between a masked tile's patched values and their readers, which no
        # DMA crosses: the next tile's rows are not read before the next tile's barrier
        assert waits.count("") == 1, name
