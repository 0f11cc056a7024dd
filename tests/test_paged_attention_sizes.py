"""Head and rotary sizes of the paged attention layer (host side)."""

import pytest
import torch

from nanovllm_voxcpm_amd.layers.attention import PagedAttention


def test_a_layer_that_does_not_rotate():
    layer = PagedAttention(4, 2, 64, rotary_dim=0, max_position=32)
    assert layer.rotary_dim == 0 and layer.prepare("cpu").shape == (32, 0)
    assert PagedAttention(4, 2, 64, max_position=32).prepare("cpu").shape == (32, 64)
