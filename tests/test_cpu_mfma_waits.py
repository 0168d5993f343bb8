"""No built kernel reads a matrix product's result too early (tests/mfma_waits.py)."""
import os
import re

import pytest

import mfma_waits as waits
from frame_hip import abi

# attention over packed sequences and over a paged cache
KERNELS = re.compile(r"attention_(rows|keys|dq|dkv)_kernel")


@pytest.mark.skipif(not os.path.exists(waits.OBJDUMP), reason="no disassembler")
def test_results_of_products_are_read_when_written(tmp_path):
    looked, early = 0, {}
    for name, code in waits.functions(abi.KERNELS_LIB, str(tmp_path)):
        if KERNELS.search(name) is None:
            continue
        looked += 1
        if found := waits.early_reads(code):
            early[name] = found[:2]
    assert looked >= 32
    assert not early, early


def test_an_early_read_is_found():
    code = [(0, "v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], 0", None), (8, "s_cbranch_vccnz 2", 24),
            (12, "s_nop 6", None), (16, "v_max3_f32 v12, v12, v0, v1", None), (24, "s_nop 5", None),
            (28, "v_max3_f32 v12, v12, v2, v3", None), (36, "s_endpgm", None)]
    (found,) = waits.early_reads(code)
    assert found[1].startswith("v_max3_f32 v12, v12, v2") and found[2:] == (7, 8)
    code[4] = (24, "s_nop 6", None)
    assert waits.early_reads(code) == []
    code[4] = (24, "v_mov_b32_e32 v2, v20", None)  # written over: no longer the product's
    code[5] = (28, "v_max3_f32 v12, v12, v2, v13", None)
    assert waits.early_reads(code) == []
