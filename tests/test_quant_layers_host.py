"""What a layer refuses before its base weight is put in 8 bits, so that no layer is left that its forward cannot serve; no GPU."""

import pytest
import torch

from nanovllm_voxcpm_amd.layers.lora import LoRALinear, LoRAMergedColumnParallelLinear


def _kept(layer):
    return not layer.base_in_8_bits and layer.weight is not None and "weight_values" not in layer.state_dict()


@pytest.mark.parametrize("make,match", [
    (lambda: LoRAMergedColumnParallelLinear(32, [16] * 9, max_loras=2, max_lora_rank=8), "targets"),  # (the 16-bit forward takes nine in two launches)
    (lambda: LoRALinear(32, 16, max_loras=2, max_lora_rank=257), "rank"),
    (lambda: LoRALinear(32, 16, max_loras=1025, max_lora_rank=1), "slots"),
    (lambda: LoRALinear(16, 2**22 + 16), "features"),
    (lambda: LoRALinear(2**22 + 16, 2), "features"),
])
def test_layers_that_no_call_would_serve_stay_as_they_are(make, match):
    with torch.device("meta"):
        layer = make()
    layer = layer.to(torch.bfloat16)
    with pytest.raises(ValueError, match=match):
        layer.quantize_base_()
    assert _kept(layer)


def test_adapters_of_another_type_are_refused_beforehand():
    layer = LoRALinear(32, 16, max_loras=2, max_lora_rank=8).to(torch.bfloat16)
    layer.lora_B.data = layer.lora_B.data.half()
    with pytest.raises(ValueError, match="own type"):
        layer.quantize_base_()
    assert _kept(layer)


def test_eight_targets_pass():
    layer = LoRAMergedColumnParallelLinear(32, [16] * 8, max_loras=2, max_lora_rank=8).to(torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):  # (the last that is looked at)
        layer.quantize_base_()
