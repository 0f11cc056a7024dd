"""The LoRA linears with base weights in 8 bits against the linear's definition in 64 bits, and the synthetic decoder over them: its paged forward against the calls that it is
made of, in graphs too."""

import copy

import pytest
import torch

from oracle import quant as oracle

pytestmark = pytest.mark.gpu

HALVES = [torch.bfloat16, torch.float16]


def _layers(dtype, bias, rank=16):
    from nanovllm_voxcpm_amd.layers.lora import LoRALinear, LoRAMergedColumnParallelLinear, LoRAQKVParallelLinear, LoRARowParallelLinear

    kw = dict(max_loras=3, max_lora_rank=rank, bias=bias)
    return [
        (LoRAQKVParallelLinear(96, 16, 6, 2, **kw), [0, 96, 128], [96, 32, 32]),
        (LoRAQKVParallelLinear(96, 16, 6, 2, lora_targets=["v", "q"], **kw), [128, 0], [32, 96]),
        (LoRAMergedColumnParallelLinear(96, [80, 48], **kw), [0, 80], [80, 48]),
        (LoRAMergedColumnParallelLinear(96, [80, 48], lora_targets=[1], **kw), [80], [48]),
        (LoRARowParallelLinear(96, 72, **kw), [0], [72]),
        (LoRALinear(96, 40, **kw), [0], [40]),
    ]


def _fill(layer, g, dtype, slots=(0, 2)):
    layer.to(device="cuda", dtype=dtype)
    layer.weight.data.copy_(torch.randn(layer.weight.shape, generator=g) * 0.1)
    if layer.bias is not None:
        layer.bias.data.copy_(torch.randn(layer.bias.shape, generator=g))
    for slot in slots:
        rank, targets = 16 - 5 * slot, layer._num_targets()
        a = torch.randn(targets, rank, 96, generator=g).cuda() * 0.1
        b = [torch.randn(layer._b_of(p).size(1), rank, generator=g).cuda() * 0.1 for p in range(targets)]
        if layer._target_keys():
            layer.set_slot_lora(slot, a, b, rank, 0.5)
        else:
            layer.set_slot_lora(slot, a[0], b[0], rank, 0.5)


def _with_slots(slots, **kw):
    from nanovllm_voxcpm_amd.utils.context import LoRAContext, set_lora_context

    slots = slots if torch.is_tensor(slots) else torch.tensor(slots, dtype=torch.int32, device="cuda")
    set_lora_context(LoRAContext(token_to_slot=slots, no_lora_flag=False, **kw))


@pytest.fixture(autouse=True)
def _no_context():
    from nanovllm_voxcpm_amd.utils.context import reset_lora_context

    reset_lora_context()
    yield
    reset_lora_context()


@torch.no_grad()
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("which", range(6))
def test_linears_match_the_definition(dtype, bias, which):
    from nanovllm_voxcpm_amd.quant_ops import quantize_rows

    g = torch.Generator().manual_seed(which + 10 * bias)
    layer, first, widths = _layers(dtype, bias)[which]
    _fill(layer, g, dtype)
    weight = quantize_rows(layer.weight.detach())
    layer.quantize_base_()
    assert layer.weight is None and torch.equal(layer.base_weight_rows().values.float(), weight.values.float()) and torch.equal(layer.base_weight_rows().scales, weight.scales)
    slots = torch.tensor([0, 2, 2, -1, 1, 0, 2], dtype=torch.int32)  # (nothing lies in slot 1)
    x = torch.randn(7, 96, generator=g).to(dtype).cuda()
    rows = quantize_rows(x)
    order = sorted(range(len(first)), key=first.__getitem__)
    a, b = [layer._a_of(p).detach().cpu() for p in order], [layer._b_of(p).detach().cpu() for p in order]
    held = [t.cpu() for t in (rows.values.float(), rows.scales, weight.values.float(), weight.scales)]
    own_bias = None if layer.bias is None else layer.bias.detach().cpu()
    want, bound = oracle.linear(*held, own_bias, a, b, [first[p] for p in order], slots, dtype)
    base, base_bound = oracle.linear(*held, own_bias, dtype=dtype)

    def check(got, want, bound):
        assert got.dtype == dtype and ((got.cpu().double().view(want.shape) - want).abs() <= bound).all()

    check(layer(x), base, base_bound)  # no context
    _with_slots(slots.cuda())
    got = layer(x)
    check(got, want, bound)
    assert torch.equal(layer(rows), got)
    _with_slots(slots[:6].cuda())
    cube = layer(x[:6].view(2, 3, 96))
    assert cube.shape[:2] == (2, 3) and torch.equal(cube.view(6, -1), layer(x[:6]))
    _with_slots(slots[:6].long().cuda())
    assert torch.equal(layer(x[:6]), cube.view(6, -1))
    _with_slots([-1] * 7)
    check(layer(x), base, base_bound)
    for slot in (0, 2):
        layer.clear_slot_lora(slot)
    _with_slots(slots.cuda())
    check(layer(x), base, base_bound)
    _with_slots([0] * 6)
    with pytest.raises(RuntimeError, match="does not match"):
        layer(x)


@torch.no_grad()
def test_a_layer_without_adapters_and_what_it_refuses():
    from nanovllm_voxcpm_amd.layers.lora import LoRALinear
    from nanovllm_voxcpm_amd.quant_ops import quantize_rows

    g = torch.Generator().manual_seed(1)
    layer = LoRALinear(96, 40, bias=False).to(device="cuda", dtype=torch.bfloat16)
    layer.weight.data.copy_(torch.randn(40, 96, generator=g))
    x = torch.randn(5, 96, generator=g).to(torch.bfloat16).cuda()
    layer.quantize_base_()
    assert layer(x).dtype == layer(quantize_rows(x)).dtype == torch.bfloat16 and torch.equal(layer(x), layer(quantize_rows(x)))
    with pytest.raises(RuntimeError, match="already"):
        layer.quantize_base_()
    layer = LoRALinear(96, 40, bias=True, max_loras=2, max_lora_rank=8).to(device="cuda", dtype=torch.bfloat16)
    layer.quantize_base_()
    with pytest.raises(ValueError, match="float16"):
        layer(x.half())
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no backward"):
        layer(x)


@torch.no_grad()
def test_the_weight_outlives_moves_copies_and_the_state_dict():
    from nanovllm_voxcpm_amd.layers.lora import LoRALinear
    from nanovllm_voxcpm_amd.quant_ops import quantize_rows

    g = torch.Generator().manual_seed(2)
    layer = LoRALinear(96, 40, max_loras=3, max_lora_rank=16)
    _fill(layer, g, torch.bfloat16)
    layer.quantize_base_()
    x = torch.randn(5, 96, generator=g).to(torch.bfloat16).cuda()
    _with_slots([0, 2, -1, 0, 2])
    want = layer(x)
    twin = copy.deepcopy(layer)
    assert torch.equal(twin(x), want)
    assert torch.equal(layer.cpu().cuda()(x), want)
    other = LoRALinear(96, 40, max_loras=3, max_lora_rank=16)
    _fill(other, g, torch.bfloat16)
    other.quantize_base_()
    assert not torch.equal(other(x), want)
    assert "weight" not in layer.state_dict()
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), want)
    # another type: the same weight
    layer.half()
    rows = quantize_rows(x)
    assert layer(rows).dtype == torch.float16 and torch.equal(layer.base_weight_rows().values.float(), twin.base_weight_rows().values.float())
    assert torch.equal(layer.base_weight_rows().scales, twin.base_weight_rows().scales)


def _model(dtype, layers=2, rank=16, **attention):
    from nanovllm_voxcpm_amd.backbone import MiniDecoder

    model = MiniDecoder(layers=layers, hidden=256, heads=4, kv_heads=2, head_dim=64, inter=512, max_loras=4, rank=rank, max_position=512, **attention)
    model = model.to(device="cuda", dtype=dtype)
    model.init_random(seed=11, adapters=3, rank=rank)
    for layer in model.layers:
        for norm in (layer.input_norm, layer.post_norm):
            norm.weight.copy_(1 + 0.2 * torch.randn(256, generator=torch.Generator().manual_seed(3)))
    return model


def _by_hand(model, x, caches, batch, slots):
    """The layers as calls of the ops."""
    from nanovllm_voxcpm_amd.quant_ops import add_rms_norm, quantize_rows, quantized_linear, silu_mul

    def linear(layer, rows):
        n = layer._num_targets()
        return quantized_linear(rows, layer.base_weight_rows(), dtype=x.dtype, lora_a=[layer._a_of(p).detach() for p in range(n)], lora_b=[layer._b_of(p).detach() for p in range(n)], token_to_slot=slots)

    total, update = x, None
    for layer, pair in zip(model.layers, caches):
        if update is None:
            rows, _ = add_rms_norm(total, layer.input_norm.weight, quantize=True)
        else:
            rows, total = add_rms_norm(update, layer.input_norm.weight, residual=total, quantize=True)
        attended = layer.attention(linear(layer.qkv, rows), *pair, batch)
        rows, total = add_rms_norm(linear(layer.o, quantize_rows(attended)), layer.post_norm.weight, residual=total, quantize=True)
        update = linear(layer.down, silu_mul(linear(layer.gate_up, rows), quantize=True))
    return add_rms_norm(update, model.norm.weight, residual=total)[0]


@torch.no_grad()
@pytest.mark.parametrize("dtype", HALVES)
def test_prompts_and_decode_steps_are_the_ops_one_behind_the_other(dtype):
    from nanovllm_voxcpm_amd.layers.attention import build_attention_batch

    model, g = _model(dtype), torch.Generator().manual_seed(4)
    wide = copy.deepcopy(model)
    model.quantize_base_()
    tables = [[7, 3, 11, 0, 19], [5, 1, 2, 13, 6], [4, 9, 8, 10, 12]]
    caches, twin, others = (m.make_paged_cache(20, 16, dtype, "cuda") for m in (model, model, wide))
    lens, adapters = [37, 20, 66], [2, -1, 0]
    for new, cached in ((lens, [0, 0, 0]), ([1, 1, 1], lens), ([3, 0, 2], [38, 21, 67])):
        batch = build_attention_batch(new, cached, tables, 16, device="cuda")
        slots = torch.tensor([a for a, n in zip(adapters, new) for _ in range(n)], dtype=torch.int32, device="cuda")
        x = torch.randn(sum(new), 256, generator=g).to(dtype).cuda()
        given = x.clone()
        _with_slots(slots)
        got = model.forward_paged(x, caches, batch)
        assert torch.equal(x, given)
        assert torch.equal(got, _by_hand(model, x, twin, batch, slots))
        for a, b in zip(caches, twin):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        # beside the 16-bit weights: an element's rounding to 8 bits is at most 2^-4 of it, 2^-4 / sqrt(3) in the mean over a binade, in rows and weights independently, so that a linear's
        # output is off by sqrt(2 / 3) 2^-4 = 5% of its norm; eight linears whose updates add up: 15%, and the norms and softmaxes between them do not more than double it.
        # (A wrong slot, scale or row is off by its own size.)
        want = wide.forward_paged(x, others, batch).float()
        assert (got.float() - want).norm() < 0.35 * want.norm()
    # the dense forward has the same linears
    dense = [(torch.zeros(3, 2, 8, 64, dtype=dtype, device="cuda"), torch.zeros(3, 2, 8, 64, dtype=dtype, device="cuda")) for _ in model.layers]
    _with_slots(adapters)
    x = torch.randn(3, 256, generator=g).to(dtype).cuda()
    got = model(x, dense, torch.zeros(3, dtype=torch.int64, device="cuda"))
    want = wide(x, [(a.clone(), b.clone()) for a, b in dense], torch.zeros(3, dtype=torch.int64, device="cuda")).float()
    assert (got.float() - want).norm() < 0.35 * want.norm()


@torch.no_grad()
def test_a_decode_step_in_a_graph_with_padding_and_adapters_that_come_later():
    from nanovllm_voxcpm_amd.layers.attention import build_attention_batch

    model, g = _model(torch.bfloat16, qk_norm=True, window=40, sinks=4), torch.Generator().manual_seed(5)
    model.quantize_base_()
    caches = model.make_paged_cache(32, 16, torch.bfloat16, "cuda")
    for pair in caches:
        for c in pair:
            c.copy_(torch.randn(c.shape, generator=g))
    held = build_attention_batch([1] * 5, [0] * 5, [[0, 1, 2, 3, 4, 5]] * 5, 16, device="cuda", rows=8, blocks=6)
    x, slots = torch.zeros(8, 256, dtype=torch.bfloat16, device="cuda"), torch.full((8,), -1, dtype=torch.int32, device="cuda")
    _with_slots(slots)
    model.forward_paged(x, caches, held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.forward_paged(x, caches, held)
    last = None
    for step in range(5):
        n = 5 - step % 2
        tables = torch.randperm(30, generator=g)[: 6 * n].view(n, 6).tolist()
        batch = build_attention_batch([1] * n, [30 + 11 * s + step for s in range(n)], tables, 16, device="cuda", rows=8, blocks=6)
        x.copy_(torch.randn(8, 256, generator=g).to(torch.bfloat16))
        slots.copy_(torch.cat([torch.randint(-1, 4, (n,), generator=g), torch.full((8 - n,), -1)]))
        if step == 3:  # slot 3 was empty when the graph was captured
            for layer in model.layers:
                q, kv = layer.qkv.q_size, layer.qkv.kv_size
                layer.qkv.set_slot_lora(3, torch.randn(3, 16, 256, generator=g).cuda(), [torch.randn(w, 16, generator=g).cuda() for w in (q, kv, kv)], 16, 0.1)
            slots[0] = 3
        for name in ("positions", "slot_mapping", "block_tables", "context_lens"):
            getattr(held, name).copy_(getattr(batch, name))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, model.forward_paged(x, caches, batch)), step
        assert last is None or not torch.equal(got, last)
        last = got


@torch.no_grad()
def test_models_with_some_linears_in_8_bits_and_models_that_stay_as_they_are():
    from nanovllm_voxcpm_amd.backbone import MiniDecoder
    from nanovllm_voxcpm_amd.layers.attention import build_attention_batch

    dtype, g = torch.bfloat16, torch.Generator().manual_seed(6)
    wide, some = _model(dtype), _model(dtype)
    some.layers[0].qkv.quantize_base_()
    some.layers[1].down.quantize_base_()
    batch = build_attention_batch([5, 9], [0, 0], [[0], [1]], 16, device="cuda")
    x = torch.randn(14, 256, generator=g).to(dtype).cuda()
    _with_slots([1] * 5 + [-1] * 9)
    want, got = (m.forward_paged(x, m.make_paged_cache(2, 16, dtype, "cuda"), batch).float() for m in (wide, some))
    assert not torch.equal(got, want) and (got - want).norm() < 0.35 * want.norm()
    with pytest.raises(RuntimeError, match="already"):
        some.quantize_base_()
    assert not some.layers[0].o.base_in_8_bits  # all or none
    odd = MiniDecoder(layers=1, hidden=32, heads=3, kv_heads=1, head_dim=8, inter=64, max_loras=1, rank=8).to(device="cuda", dtype=dtype)  # (o has 24 input features)
    with pytest.raises(ValueError, match="multiple of 16"):
        odd.quantize_base_()
    assert not odd.layers[0].qkv.base_in_8_bits and not odd.base_in_8_bits
