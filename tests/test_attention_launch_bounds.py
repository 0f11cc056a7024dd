"""The most rows times heads that a call takes, at the C entries (host side)."""

import ctypes as C

import pytest

from nanovllm_voxcpm_amd import _hip


@pytest.mark.parametrize("rows,heads", [((1 << 30) // 64 + 1, 64), ((1 << 30) + 1, 1), ((1 << 31) - 1, 1 << 15)])
def test_more_rows_and_heads_than_a_call_takes_are_refused(rows, heads):
    lib = _hip.load()
    args = _hip.MloraAttentionArgs(q=64, out=64, k=64, v=64, starts=64, block_tables=64, context_lens=64, table_width=1, num_blocks=1, page=16, num_rows=rows,
                                   sequences=rows, heads=heads, kv_heads=1, dim=8, dtype=2, causal=1, scale=1.0)
    for entry in (lib.mlora_decode_attention, lib.mlora_prompt_attention):
        assert entry(C.byref(args)) == -3 and "more than one launch holds" in lib.mlora_last_error().decode()
