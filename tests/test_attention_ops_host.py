"""Host side of the attention block: the C structs' layout, what is refused before any launch (all on host tensors), the
rotary table, and the oracle against torch's own softmax."""

import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch

from nanovllm_voxcpm_amd import _hip
from nanovllm_voxcpm_amd.attention_ops import decode_attention, prompt_attention, rotary_table, rotate_qk
from oracle import attention as oracle

ROOT = Path(__file__).resolve().parent.parent


def test_ctypes_structs_match_the_c_layout(tmp_path):
    structs = {"MloraRotateArgs": _hip.MloraRotateArgs, "MloraAttentionArgs": _hip.MloraAttentionArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "mlora.h"', "int main(void) {"]
    for name, st in structs.items():
        lines.append(f'  printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name}.{field} %zu\\n", offsetof({name}, {field}));' for field, _ in st._fields_]
    (tmp_path / "probe.c").write_text("\n".join([*lines, "  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", str(tmp_path / "probe.c"), "-o", str(tmp_path / "probe")], check=True)
    got = dict(line.split() for line in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, st in structs.items():
        assert int(got[name]) == C.sizeof(st)
        for field, _ in st._fields_:
            assert int(got[f"{name}.{field}"]) == getattr(st, field).offset, field


def _rotate_block(**change):
    a = _hip.MloraRotateArgs(q=64, k=64, q_out=64, k_out=64, positions=64, cos_sin=64, num_tokens=1, heads=2, kv_heads=1, dim=64, rotary=64,
                             num_positions=1, dtype=2)
    for name, value in change.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,code,text", [
    (dict(num_tokens=-1), -1, "negative"), (dict(heads=-2), -1, "negative"), (dict(dtype=7), -1, "dtype"), (dict(dim=60), -2, "dim"), (dict(dim=264), -2, "dim"),
    (dict(dim=0), -2, "dim"), (dict(rotary=24), -2, "rotary"), (dict(rotary=80), -2, "rotary"), (dict(rotary=-16), -2, "rotary"), (dict(positions=None), -1, "NULL"),
    (dict(cos_sin=None), -1, "NULL"), (dict(q_out=None), -1, "NULL"), (dict(k=None), -1, "NULL"), (dict(slots=64), -1, "cache"),
    (dict(k_cache=64, v_cache=64, slots=64, page=16), -1, "cache"), (dict(k_cache=64, v_cache=64, slots=64, v=64, page=0), -1, "cache"), (dict(v=64), -1, "cache"),
    (dict(num_tokens=1 << 30), -3, "launch"),
])
def test_rotation_refuses_at_the_c_entry(change, code, text):
    lib = _hip.load()
    assert lib.mlora_rotate_qk(C.byref(_rotate_block(**change))) == code
    assert text in lib.mlora_last_error().decode()


def test_null_and_empty_calls_at_the_c_entries():
    lib = _hip.load()
    for name in ("mlora_rotate_qk", "mlora_decode_attention", "mlora_prompt_attention"):
        assert getattr(lib, name)(None) == -1
    assert lib.mlora_rotate_qk(C.byref(_rotate_block(num_tokens=0))) == 0
    for change in (dict(num_rows=0), dict(sequences=0, num_rows=0)):
        assert lib.mlora_decode_attention(C.byref(_attention_block(**change))) == 0
        assert lib.mlora_prompt_attention(C.byref(_attention_block(**change))) == 0


def _attention_block(**change):
    a = _hip.MloraAttentionArgs(q=64, out=64, k=64, v=64, starts=64, block_tables=64, context_lens=64, table_width=4, num_blocks=9, page=16, num_rows=2,
                                sequences=2, heads=4, kv_heads=2, dim=64, dtype=2, causal=1, scale=1.0)
    for name, value in change.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,code,text", [
    (dict(num_rows=-1), -1, "negative"), (dict(window=-1), -1, "negative"), (dict(sinks=-1), -1, "negative"), (dict(dtype=9), -1, "dtype"), (dict(dim=4), -2, "dim"),
    (dict(dim=257), -2, "dim"), (dict(causal=0, window=3), -2, "causal"), (dict(causal=0, sinks=3), -2, "causal"), (dict(kv_heads=0), -1, "evenly"),
    (dict(heads=5), -1, "evenly"), (dict(q=None), -1, "NULL"), (dict(out=None), -1, "NULL"), (dict(k=None), -1, "NULL"), (dict(v=None), -1, "NULL"),
    (dict(context_lens=None), -1, "context_lens"), (dict(page=0), -1, "page"), (dict(table_width=1 << 28), -3, "positions"),
    (dict(num_rows=1 << 29, sequences=1 << 29), -3, "launch"),
])
def test_attention_refuses_at_the_c_entries(change, code, text):
    lib = _hip.load()
    for entry in (lib.mlora_decode_attention, lib.mlora_prompt_attention):
        assert entry(C.byref(_attention_block(**change))) == code
        assert text in lib.mlora_last_error().decode()


def test_attention_refuses_what_only_one_entry_knows():
    lib = _hip.load()
    for entry, change, text in ((lib.mlora_decode_attention, dict(block_tables=None), "pages"), (lib.mlora_decode_attention, dict(num_rows=3), "rows"),
                                (lib.mlora_decode_attention, dict(causal=0), "causal"), (lib.mlora_prompt_attention, dict(starts=None), "starts")):
        assert entry(C.byref(_attention_block(**change))) == -1
        assert text in lib.mlora_last_error().decode()


def _rotation(**change):
    t, h, hk, d = 5, 4, 2, 64
    call = dict(q=torch.zeros(t, h, d), k=torch.zeros(t, hk, d), positions=torch.zeros(t, dtype=torch.int32), cos_sin=torch.zeros(9, d))
    cache = dict(v=torch.zeros(t, hk, d), k_cache=torch.zeros(2, 16, hk, d), v_cache=torch.zeros(2, 16, hk, d), slot_mapping=torch.zeros(t, dtype=torch.int64))
    if change.pop("cached", False):
        call.update(cache)
    call.update(change)
    return call


@pytest.mark.parametrize("change,error,text", [
    (dict(q=torch.zeros(5, 256)), ValueError, "q must be"), (dict(k=torch.zeros(4, 2, 64)), ValueError, "differ"), (dict(k=torch.zeros(5, 2, 32)), ValueError, "differ"),
    (dict(k=torch.zeros(5, 2, 64, dtype=torch.float16)), ValueError, "element type"), (dict(q=torch.zeros(5, 64, 4).transpose(1, 2)), ValueError, "side by side"),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), ValueError, "positions has 4"), (dict(positions=torch.zeros(5)), ValueError, "positions must"),
    (dict(cos_sin=torch.zeros(9, 64, dtype=torch.float64)), ValueError, "cos_sin"), (dict(cos_sin=torch.zeros(64)), ValueError, "cos_sin"),
    (dict(q_weight=torch.ones(63)), ValueError, "q_weight"), (dict(k_weight=torch.ones(64, dtype=torch.float16)), ValueError, "k_weight"),
    (dict(v=torch.zeros(5, 2, 64)), ValueError, "together"), (dict(cached=True, slot_mapping=None), ValueError, "together"),
    (dict(cached=True, v=torch.zeros(5, 1, 64)), ValueError, "differ"), (dict(cached=True, k_cache=torch.zeros(2, 16, 1, 64)), ValueError, "differ"),
    (dict(cached=True, k_cache=torch.zeros(2, 16, 2, 32), v_cache=torch.zeros(2, 16, 2, 32)), ValueError, "size 64"),
    (dict(cached=True, slot_mapping=torch.zeros(3, dtype=torch.int32)), ValueError, "slot_mapping has 3"),
    (dict(cached=True, k_cache=torch.zeros(1, 16, 2, 64).expand(2, 16, 2, 64)), ValueError, "share memory"),
    (dict(q_out=torch.zeros(5, 4, 32)), ValueError, "shape"), (dict(k_out=torch.zeros(1, 2, 64).expand(5, 2, 64)), ValueError, "share memory"),
    (dict(q=torch.zeros(5, 4, 64, requires_grad=True)), RuntimeError, "no backward"), (dict(), RuntimeError, "GPU"),
])
def test_rotation_refuses_at_the_python_entry(change, error, text):
    with pytest.raises(error, match=text):
        rotate_qk(**_rotation(**dict(change)))


def _decode(**change):
    return {**dict(q=torch.zeros(3, 4, 64), k_cache=torch.zeros(5, 16, 2, 64), v_cache=torch.zeros(5, 16, 2, 64),
                   block_tables=torch.zeros(3, 2, dtype=torch.int32), context_lens=torch.zeros(3, dtype=torch.int32)), **change}


@pytest.mark.parametrize("change,error,text", [
    (dict(q=torch.zeros(3, 256)), ValueError, "q must be"), (dict(k_cache=torch.zeros(5, 16, 64)), ValueError, "k_cache must be"),
    (dict(v_cache=torch.zeros(4, 16, 2, 64)), ValueError, "differ"), (dict(q=torch.zeros(3, 4, 32)), ValueError, "size 32"),
    (dict(q=torch.zeros(3, 5, 64)), ValueError, "evenly"), (dict(window=-1), ValueError, "negative"), (dict(sinks=-1), ValueError, "negative"),
    (dict(block_tables=torch.zeros(2, 2, dtype=torch.int32)), ValueError, "2 rows for 3"), (dict(block_tables=torch.zeros(3, 2, dtype=torch.int64)), ValueError, "int32"),
    (dict(block_tables=torch.zeros(2, 3, dtype=torch.int32).T), ValueError, "side by side"), (dict(context_lens=torch.zeros(2, dtype=torch.int32)), ValueError, "2 entries"),
    (dict(context_lens=torch.zeros(3, dtype=torch.int64)), ValueError, "context_lens"), (dict(out=torch.zeros(3, 4, 32)), ValueError, "shape"),
    (dict(out=torch.zeros(3, 4, 64, dtype=torch.float16)), ValueError, "element type"), (dict(q=torch.zeros(3, 4, 64, requires_grad=True)), RuntimeError, "no backward"),
    (dict(), RuntimeError, "GPU"),
])
def test_decode_refuses_at_the_python_entry(change, error, text):
    with pytest.raises(error, match=text):
        decode_attention(**_decode(**change))


def test_outputs_may_not_overlap_their_inputs():
    memory = torch.zeros(4, 4, 64)
    with pytest.raises(ValueError, match="overlaps"):
        decode_attention(**_decode(q=memory[:3], out=memory[1:]))
    with pytest.raises(ValueError, match="overlaps"):
        decode_attention(**_decode(q=memory[:3], out=memory[:3]))


def _refused(call, arguments, text):
    """A call that passes its checks ends at the missing GPU."""
    with pytest.raises(ValueError if text else RuntimeError, match=text or "GPU"):
        call(**arguments)


def test_results_may_lie_between_their_inputs_but_not_on_them():
    qkv = torch.zeros(5, 8, 64)
    q, k, v = qkv.split([4, 2, 2], dim=1)
    rotation = _rotation(q=q, k=k)
    _refused(rotate_qk, {**rotation, "q_out": q, "k_out": k}, None)
    _refused(rotate_qk, {**rotation, "q_out": q, "k_out": v}, None)  # (v takes no part in a call without a cache)
    _refused(rotate_qk, {**rotation, "q_out": qkv[:, 1:5]}, "q_out overlaps")
    _refused(rotate_qk, {**rotation, "k_out": qkv[:, 5:7]}, "k_out overlaps")
    _refused(rotate_qk, {**rotation, "k_out": q[:, 2:]}, "k_out overlaps another")
    _refused(rotate_qk, {**rotation, "q_out": qkv[:, 4:]}, "q_out overlaps another")
    room = torch.zeros(5, 4, 64)
    _refused(rotate_qk, {**rotation, "q_out": room, "k_out": room[:, 1:3]}, "q_out overlaps another")
    _refused(rotate_qk, {**_rotation(cached=True, q=q, k=k, v=v), "k_out": v}, "k_out overlaps another")
    wide = torch.zeros(7, 10, 64)
    for out, text in ((wide[:, 6:], None), (wide[:, 5:9], "out overlaps v"), (wide[:, :4], "out overlaps k")):
        _refused(prompt_attention, _prompt(k=wide[:, 2:4], v=wide[:, 4:6], out=out), text)
    _refused(prompt_attention, _prompt(q=torch.zeros(7, 2, 64), k=wide[:, 2:4], v=wide[:, 4:6], out=wide[:, 4:6]), "out overlaps v")
    pages = torch.zeros(5, 16, 2, 64)
    _refused(decode_attention, _decode(k_cache=pages, out=pages.view(-1, 4, 64)[6:9]), "out overlaps k")


def _prompt(**change):
    return {**dict(q=torch.zeros(7, 4, 64), k=torch.zeros(7, 2, 64), v=torch.zeros(7, 2, 64), cu_seqlens=torch.tensor([0, 3, 7], dtype=torch.int32)), **change}


@pytest.mark.parametrize("change,error,text", [
    (dict(cu_seqlens=torch.tensor([0, 7])), ValueError, "cu_seqlens"), (dict(cu_seqlens=torch.zeros(0, dtype=torch.int32)), ValueError, "cu_seqlens has 0"),
    (dict(v=torch.zeros(6, 2, 64)), ValueError, "alike"), (dict(q=torch.zeros(7, 4, 32)), ValueError, "alike"), (dict(q=torch.zeros(7, 3, 64)), ValueError, "evenly"),
    (dict(causal=False, window=4), ValueError, "causal"), (dict(causal=False, sinks=4), ValueError, "causal"),
    (dict(block_tables=torch.zeros(2, 1, dtype=torch.int32)), ValueError, "together"), (dict(cu_seqlens_k=torch.zeros(2, dtype=torch.int32)), ValueError, "cu_seqlens_k has 2"),
    (dict(block_tables=torch.zeros(2, 1, dtype=torch.int32), context_lens=torch.zeros(2, dtype=torch.int32)), ValueError, "k must be"),
    (dict(k=torch.zeros(7, 2, 64, dtype=torch.bfloat16)), ValueError, "element type"), (dict(v=torch.zeros(7, 2, 64, requires_grad=True)), RuntimeError, "no backward"),
    (dict(), RuntimeError, "GPU"),
])
def test_prompts_refuse_at_the_python_entry(change, error, text):
    with pytest.raises(error, match=text):
        prompt_attention(**_prompt(**change))


def test_rotary_table():
    table = rotary_table(64, 100, base=500.0, scale=0.5, factors=[1.0 + i for i in range(32)])
    assert table.shape == (100, 64) and table.dtype == torch.float32
    angle = 99 * 500.0 ** (-7 / 32) / 8.0
    assert abs(table[99, 7].item() - 0.5 * torch.tensor(angle, dtype=torch.float64).cos().item()) < 1e-7
    assert abs(table[99, 39].item() - 0.5 * torch.tensor(angle, dtype=torch.float64).sin().item()) < 1e-7
    for args, kw in (((63, 4), {}), ((0, 4), {}), ((64, 0), {}), ((64, 4), dict(factors=[1.0]))):
        with pytest.raises(ValueError):
            rotary_table(*args, **kw)


def test_oracle_against_a_masked_softmax():
    g = torch.Generator().manual_seed(1)
    q, k, v = torch.randn(5, 4, 8, generator=g), torch.randn(9, 2, 8, generator=g), torch.randn(9, 2, 8, generator=g)
    got, bound = oracle.attend(q, k, v, True, 3, 1)
    place, key = torch.arange(4, 9)[:, None], torch.arange(9)[None]
    seen = (key <= place) & ((key > place - 3) | (key < 1))
    for h in range(4):
        scores = (q[:, h].double() @ k[:, h // 2].double().T * 8**-0.5).masked_fill(~seen, float("-inf"))
        assert torch.allclose(got[:, h], torch.softmax(scores, -1) @ v[:, h // 2].double(), atol=1e-12)
    assert (bound > 0).all()
    turned, _ = oracle.rotate(q, torch.arange(5), torch.cat([torch.zeros(5, 4), torch.ones(5, 4)], 1))  # by a quarter
    assert torch.equal(turned[..., :4], -q.double()[..., 4:]) and torch.equal(turned[..., 4:], q.double()[..., :4])
