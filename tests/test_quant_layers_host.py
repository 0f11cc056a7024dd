"""LoRA linears with base weights in 8 bits: what a layer refuses beforehand, so that none is left that its forward cannot serve, and what it does on the host around its two calls; no GPU."""

import copy
import gc
import weakref

import pytest
import torch

from nanovllm_voxcpm_amd.layers import lora as layers
from nanovllm_voxcpm_amd.layers.lora import LoRALinear, LoRAMergedColumnParallelLinear
from nanovllm_voxcpm_amd.quant_ops import QuantizedRows
from oracle import quant as oracle


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


@pytest.fixture
def on_the_host(monkeypatch):
    """The ops by their definitions."""

    def quantize(x):
        assert x.dim() == 2 and (x.stride(1) == 1 or x.size(1) == 1)  # (as the op does)
        scales, _, values, _ = oracle.eight_bits(x.double(), 0.0)
        return QuantizedRows(values.to(torch.float8_e4m3fn), scales.float())

    def linear(rows, weight, *, bias=None, dtype=None, **adapters):
        assert not adapters and (bias is None or bias.dtype == dtype)
        return oracle.linear(rows.values.float(), rows.scales, weight.values.float(), weight.scales, bias, dtype=dtype)[0].to(dtype)

    monkeypatch.setattr(layers, "quantize_rows", quantize)
    monkeypatch.setattr(layers, "quantized_linear", linear)
    monkeypatch.setattr(layers._LoRALayerBase, "check_base_for_8_bits", lambda self: None)
    return quantize


@torch.no_grad()
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("loras", [0, 2])
def test_the_output_has_the_layers_type_after_a_change_of_it(on_the_host, bias, loras):
    layer = LoRALinear(32, 8, bias=bias, max_loras=loras, max_lora_rank=4 if loras else 0).to(torch.bfloat16)
    layer.weight.copy_(torch.randn(8, 32, generator=torch.Generator().manual_seed(1)))
    layer.quantize_base_()
    names = set(layer.state_dict())
    x = torch.randn(3, 32)
    for dtype in (torch.bfloat16, torch.float16, torch.bfloat16):
        layer.to(dtype)
        want = layer(x.to(dtype))
        got = layer(on_the_host(x.to(dtype)))
        assert want.dtype == got.dtype == dtype and torch.equal(got, want)
        with pytest.raises(ValueError, match="the layer"):
            layer(x.to(torch.bfloat16 if dtype == torch.float16 else torch.float16))
    assert set(layer.state_dict()) == names == {"weight_values", "weight_scales"} | ({"bias"} if bias else set()) | ({"lora_A", "lora_B"} if loras else set())


@torch.no_grad()
def test_the_8_bit_weight_is_what_its_buffers_hold(on_the_host):
    """Whichever way other numbers come into them; and a layer whose weight lies elsewhere now keeps nothing of where it was."""
    g = torch.Generator().manual_seed(2)
    one, other = (LoRALinear(32, 8, bias=False).half() for _ in range(2))
    for layer in (one, other):
        layer.weight.copy_(torch.randn(8, 32, generator=g))
        layer.quantize_base_()
    x = torch.randn(3, 32, generator=g).half()
    first, want = one(x), other(x)
    assert not torch.equal(first, want)
    held = {name: t.clone() for name, t in one.state_dict().items()}
    for take in (lambda: one.load_state_dict(other.state_dict()), lambda: one.load_state_dict(copy.deepcopy(other.state_dict()), assign=True),
                 lambda: [setattr(one._buffers[n], "data", t.clone()) for n, t in other.state_dict().items()], lambda: [one._buffers[n].set_(t.clone()) for n, t in other.state_dict().items()],
                 lambda: [one.register_buffer(n, t.clone()) for n, t in other.state_dict().items()]):
        one.load_state_dict(held)
        assert torch.equal(one(x), first)
        take()
        assert torch.equal(one(x), want)
    twin = copy.deepcopy(one)
    one.load_state_dict(held)
    assert torch.equal(twin(x), want) and torch.equal(one(x), first)
    gone = weakref.ref(one._buffers["weight_values"])
    one.register_buffer("weight_values", held["weight_values"].clone())
    gc.collect()
    assert gone() is None


@torch.no_grad()
def test_inputs_lie_as_a_linear_takes_them(on_the_host):
    g = torch.Generator().manual_seed(3)
    layer = LoRALinear(32, 8, bias=False).half()
    layer.weight.copy_(torch.randn(8, 32, generator=g))
    layer.quantize_base_()
    x = torch.randn(6, 32, generator=g).half()
    want = layer(x)
    apart = torch.zeros(6, 64).half()
    apart[:, ::2] = x
    for same in (x.t().contiguous().t(), apart[:, ::2], x.view(2, 3, 32), x.view(2, 3, 32).permute(2, 0, 1).contiguous().permute(1, 2, 0), x.view(3, 2, 32).transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(layer(same).reshape(6, 8), want) and layer(same).shape == (*same.shape[:-1], 8)
    assert torch.equal(layer(x[2]), want[2])
    assert torch.equal(layer(x[:1, 0:1].expand(4, 32)), layer(x[:1, 0:1].expand(4, 32).contiguous()))
    assert layer(x[:0]).shape == (0, 8) and layer(x[:0].view(0, 3, 32)).shape == (0, 3, 8)
