"""What a batch says for the paged attention layer (host arithmetic)."""

import pytest
import torch

from nanovllm_voxcpm_amd.layers.attention import PagedAttention, build_attention_batch


def test_prompts_behind_cached_tokens():
    b = build_attention_batch([3, 0, 2], [0, 4, 5], [[7], [1, 2], [4, 0, 9]], 4, device="cpu")
    assert b.positions.tolist() == [0, 1, 2, 5, 6] and b.slot_mapping.tolist() == [28, 29, 30, 1, 2]
    assert b.context_lens.tolist() == [3, 4, 7] and b.cu_seqlens.tolist() == [0, 3, 3, 5]
    assert b.block_tables.tolist() == [[7, -1, -1], [1, 2, -1], [4, 0, 9]]
    assert all(t.dtype == torch.int32 and t.is_contiguous() for t in (b.positions, b.slot_mapping, b.context_lens, b.cu_seqlens, b.block_tables))


def test_decode_padded_to_a_graph():
    b = build_attention_batch([1, 1], [5, 0], [[3, 2], [8]], 4, device="cpu", rows=4, blocks=3)
    assert b.cu_seqlens is None and b.positions.tolist() == [5, 0, 0, 0] and b.slot_mapping.tolist() == [9, 32, -1, -1]
    assert b.context_lens.tolist() == [6, 1, 0, 0] and b.block_tables.tolist() == [[3, 2, -1], [8, -1, -1], [-1] * 3, [-1] * 3]


def test_empty_batches():
    b = build_attention_batch([], [], [], 16, device="cpu")
    assert b.positions.numel() == 0 and b.block_tables.shape == (0, 0)
    b = build_attention_batch([0], [0], [[]], 16, device="cpu")
    assert b.cu_seqlens.tolist() == [0, 0] and b.context_lens.tolist() == [0]


@pytest.mark.parametrize("args,kw,text", [
    (([1], [0, 0], [[0]], 4), {}, "cached lengths"), (([1], [0], [], 4), {}, "block tables"), (([5], [0], [[0]], 4), {}, "does not fit 1 blocks"),
    (([1], [4], [[0]], 4), {}, "does not fit"), (([-1], [0], [[0]], 4), {}, "-1 new"), (([1], [0], [[0]], 0), {}, "block_size"),
    (([2], [0], [[0]], 4), dict(rows=1), "does not fit 1 rows"), (([2], [0], [[0, 1]], 4), dict(blocks=1), "and 1 blocks"),
])
def test_batches_that_do_not_fit(args, kw, text):
    with pytest.raises(ValueError, match=text):
        build_attention_batch(*args, device="cpu", **kw)


def test_layer_refuses_uneven_heads_and_host_tensors():
    with pytest.raises(ValueError, match="evenly"):
        PagedAttention(6, 4, 64)
    layer = PagedAttention(4, 2, 64, qk_norm=True, max_position=32)
    assert {n for n, _ in layer.named_parameters()} == {"q_norm", "k_norm"} and not layer.state_dict().keys() - {"q_norm", "k_norm"}
    assert layer.to(torch.bfloat16).prepare("cpu").dtype == torch.float32
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        layer(torch.zeros(3, 8 * 64, dtype=torch.bfloat16), cache, cache, build_attention_batch([3], [0], [[0]], 16, device="cpu"))
