"""The scanner of the kernels' assembly (`make -C nanovllm-voxcpm_amd/csrc check`) for direct loads too soon behind a vector
instruction's write of their base, on hand-written snippets."""

import importlib.util
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def _scan(tmp_path, body):
    spec = importlib.util.spec_from_file_location("check_sgpr_reads", ROOT / "nanovllm-voxcpm_amd" / "csrc" / "check_sgpr_reads.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    path = tmp_path / "kernel.s"
    path.write_text("_Zkernel:\n" + "\n".join(f"\t{line}" if not line.endswith(":") else line for line in body) + "\n")
    return module.scan(path)


LOAD = "global_load_lds_dwordx4 v9, s[4:5]"


@pytest.mark.parametrize("between,found", [(["s_nop 0"], 1), (["s_nop 3"], 1), (["s_nop 4"], 0), (["v_add_u32_e32 v1, v2, v3"] * 4, 1),
                                           (["v_add_u32_e32 v1, v2, v3"] * 5, 0), ([".LBB0_1:", "s_nop 0"], 1), (["s_mov_b32 s5, s6"], 0)])
def test_distance_behind_a_vector_write_of_the_base(tmp_path, between, found):
    assert _scan(tmp_path, ["v_readfirstlane_b32 s5, v7", *between, LOAD]) == found


def test_other_registers_and_other_loads_do_not_count(tmp_path):
    assert _scan(tmp_path, ["v_readfirstlane_b32 s6, v7", LOAD]) == 0
    assert _scan(tmp_path, ["s_add_u32 s4, s6, s7", "s_addc_u32 s5, s8, s9", LOAD]) == 0
    assert _scan(tmp_path, ["v_readfirstlane_b32 s5, v7", "global_load_dwordx4 v[0:3], v9, s[4:5]"]) == 0  # the compiler's own


@pytest.mark.parametrize("reader", ["s_cmp_lg_u32 s5, 0", "s_cmpk_eq_i32 s5, 0x10", "s_cmp_eq_u64 s[4:5], 0", "s_bitcmp1_b32 s5, 3", "s_bitcmp0_b64 s[4:5], 3",
                                    "s_setreg_b32 hwreg(HW_REG_MODE, 0, 2), s5", "s_setprio 1", "s_cbranch_scc1 .LBB0_2"])
def test_scalar_instructions_that_only_read_do_not_hide_the_write(tmp_path, reader):
    assert _scan(tmp_path, ["v_readfirstlane_b32 s5, v7", reader, LOAD]) == 1
    assert _scan(tmp_path, ["v_readfirstlane_b32 s5, v7", reader, "s_nop 3", LOAD]) == 0  # five wait states with the reader's own


@pytest.mark.parametrize("writer,found", [("s_cselect_b32 s5, s6, s7", 0), ("s_add_u32 s5, s5, s6", 0), ("s_load_dwordx2 s[4:5], s[0:1], 0x10", 0),
                                          ("s_mov_b32 s6, s5", 1)])
def test_scalar_instructions_that_write_do(tmp_path, writer, found):
    assert _scan(tmp_path, ["v_readfirstlane_b32 s5, v7", writer, LOAD]) == found


def test_bases_in_vcc(tmp_path):
    assert _scan(tmp_path, ["v_readfirstlane_b32 vcc_hi, v7", "global_load_lds_dwordx4 v9, vcc"]) == 1
    assert _scan(tmp_path, ["v_cmp_gt_u32_e32 vcc, s6, v7", "global_load_lds_dwordx4 v9, vcc"]) == 1
    assert _scan(tmp_path, ["v_readfirstlane_b32 vcc_hi, v7", "s_mov_b32 vcc_hi, s6", "global_load_lds_dwordx4 v9, vcc"]) == 0
