"""No built kernel reads a matrix product's result too early (tests/mfma_waits.py)."""
import os

import pytest

import mfma_waits as waits
from frame_hip import abi


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(waits.OBJDUMP):
        pytest.skip("no disassembler")
    return dict(waits.functions(abi.KERNELS_LIB, str(tmp_path_factory.mktemp("code"))))


def test_results_of_products_are_read_when_written(kernels):
    early = {name: found[:2] for name, code in kernels.items() if (found := waits.early_reads(code))}
    assert len(kernels) >= 100
    assert not early, early


def test_no_result_is_read_early_through_an_index(kernels):
    early = {name: found[:2] for name, code in kernels.items() if (found := waits.early_reads(code, by_index_only=True))}
    assert len(kernels) >= 100
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


def test_an_early_read_through_an_index_is_found():
    code = [(0, "v_mfma_f32_32x32x16_bf16 v[16:31], v[32:35], v[36:39], 0", None), (8, "s_set_gpr_idx_on s15, gpr_idx(SRC0)", None),
            (12, "s_nop 9", None), (16, "v_mov_b32_e32 v90, v0", None), (20, "v_mov_b32_e32 v91, v1", None),
            (24, "s_set_gpr_idx_off", None), (28, "v_add_f32_e32 v0, v0, v1", None), (32, "s_endpgm", None)]
    (found,) = waits.early_reads(code, by_index_only=True)
    assert found[1] == "v_mov_b32_e32 v90, v0" and found[2:] == (11, 12)
    code[2] = (12, "s_nop 10", None)
    assert waits.early_reads(code) == []
