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
