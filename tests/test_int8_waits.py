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
    kernels = re.findall(r"^(_ZN\S*int8_tile_kernel\S*Lb1E\S*):(.*?)^\.Lfunc_end", text,
                         re.S | re.M)
    assert len(kernels) >= 2  # tile sizes, rows by DMA
    for name, body in kernels:
        assert "global_load_lds_dwordx4" in body, name
        # first step and steady state; a wave's own operands have been read, too, when their
        # slot is given to the next rows
        joint = re.findall(r"s_waitcnt vmcnt\(0\) lgkmcnt\(0\)\n\s*s_barrier\n\s*;;#ASMEND", body)
        assert len(joint) >= 2, name
        # no DMA behind the last joint wait but the loop's own
        others = len(re.findall(r"\bs_barrier\b", body)) - len(joint)
        assert others <= 1, name  # before the results
