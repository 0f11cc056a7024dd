"""Head and rotary sizes of the paged attention layer (host side)."""

import pytest
import torch

from nanovllm_voxcpm_amd.layers.attention import PagedAttention


def test_a_layer_that_does_not_rotate():
    layer = PagedAttention(4, 2, 64, rotary_dim=0, max_position=32)
    assert layer.rotary_dim == 0 and layer.prepare("cpu").shape == (32, 0)
    assert PagedAttention(4, 2, 64, max_position=32).prepare("cpu").shape == (32, 64)


@pytest.mark.parametrize("head_size,rotary_dim,text", [(24, None, "rotary_dim = 24 is not a multiple of 16"), (40, None, "rotary_dim = 40"), (64, 8, "rotary_dim = 8"), (64, 80, "up to the head size 64"),
                                                       (64, -16, "rotary_dim = -16"), (60, 16, "head_size = 60 is not a multiple of 8"), (264, 64, "head_size = 264"), (0, 0, "head_size = 0")])
def test_sizes_that_no_call_serves_are_refused_when_the_layer_is_made(head_size, rotary_dim, text):
    with pytest.raises(ValueError, match=text):
        PagedAttention(4, 2, head_size, rotary_dim=rotary_dim)


def test_sizes_that_are_served():
    for head_size, rotary_dim in ((8, 0), (24, 16), (40, 32), (96, None), (256, None), (80, None)):
        PagedAttention(4, 2, head_size, rotary_dim=rotary_dim, max_position=4)


def test_a_decoder_of_other_head_sizes_keeps_its_dense_form():
    from nanovllm_voxcpm_amd.backbone import MiniDecoder

    model = MiniDecoder(layers=1, hidden=64, heads=2, kv_heads=1, head_dim=24, inter=64, max_loras=2, rank=8)
    for p in model.parameters():
        torch.nn.init.normal_(p, generator=torch.Generator().manual_seed(1))
    caches = [(torch.zeros(3, 1, 8, 24), torch.zeros(3, 1, 8, 24))]
    with torch.no_grad():
        assert torch.isfinite(model(torch.randn(3, 64), caches, torch.zeros(3, dtype=torch.int64))).all()
    with pytest.raises(ValueError, match="rotary_dim = 24"):
        model.make_paged_cache(4, 16, torch.float32, "cpu")


@pytest.mark.parametrize("new,cached,rotary_dim,refused", [([33], [0], None, True), ([32], [0], None, False), ([1, 1], [3, 32], None, True), ([1, 1], [3, 31], None, False),
                                                           ([0, 2], [40, 0], None, False), ([33], [0], 0, False), ([], [], None, False)])
def test_positions_behind_the_layers_table_are_refused(new, cached, rotary_dim, refused):
    from nanovllm_voxcpm_amd.layers.attention import AttentionBatch, build_attention_batch

    layer, cache = PagedAttention(2, 1, 64, max_position=32, rotary_dim=rotary_dim), torch.zeros(9, 16, 1, 64)
    batch = build_attention_batch(new, cached, [[3 * s, 3 * s + 1, 3 * s + 2] for s in range(len(new))], 16, device="cpu", rows=sum(new) + 2)
    with torch.no_grad(), pytest.raises(ValueError if refused else RuntimeError, match="position 32 .* 32 positions" if refused else "GPU"):
        layer(torch.zeros(sum(new) + 2, 4 * 64), cache, cache, batch)
    unknown = AttentionBatch(batch.positions, batch.slot_mapping, batch.block_tables, batch.context_lens, batch.cu_seqlens)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):  # (what the host does not know is the kernel's: NaN)
        layer(torch.zeros(sum(new) + 2, 4 * 64), cache, cache, unknown)
