"""The synthetic decoder over a paged cache (prompts, chunks, decode steps, LoRA on every linear) against its own forward over a
dense cache, token by token, and the attention layer against the definitions in 64 bits."""

import pytest
import torch

from oracle import attention as oracle

pytestmark = pytest.mark.gpu


def _model(dtype, layers=2, **attention):
    from nanovllm_voxcpm_amd.backbone import MiniDecoder

    model = MiniDecoder(layers=layers, hidden=256, heads=4, kv_heads=2, head_dim=64, inter=512, max_loras=4, rank=16, max_position=512, **attention)
    model = model.to(device="cuda", dtype=dtype)
    model.init_random(seed=11, adapters=4, rank=16)
    return model


def _with_slots(slots):
    from nanovllm_voxcpm_amd.utils.context import LoRAContext, set_lora_context

    set_lora_context(LoRAContext(token_to_slot=torch.tensor(slots, dtype=torch.int32, device="cuda"), no_lora_flag=False))


@torch.no_grad()
def test_prompts_chunks_and_decode_match_the_dense_decoder_token_by_token():
    from nanovllm_voxcpm_amd.layers.attention import build_attention_batch

    model, g = _model(torch.float32), torch.Generator().manual_seed(3)
    lens, page, adapters = [37, 20, 66], 16, [2, -1, 0]
    x = torch.randn(3, 70, 256, generator=g).cuda()
    # token by token over the dense cache
    dense = [(torch.zeros(3, 2, 80, 64, device="cuda"), torch.zeros(3, 2, 80, 64, device="cuda")) for _ in model.layers]
    want = []
    for p in range(70):
        _with_slots(adapters)
        want.append(model(x[:, p], dense, torch.full((3,), p, device="cuda")))
    want = torch.stack(want, dim=1)
    # whole prompts, the last one in two chunks, then decode steps, in pages in some order
    caches = model.make_paged_cache(20, page, torch.float32, "cuda")
    tables = [[7, 3, 11, 0, 19], [5, 1, 2, 13, 6], [4, 9, 8, 10, 12]]
    bound = dict(rtol=1e-4, atol=1e-5)  # (as the dense decoder's own fp32 test)

    def prompts(new, cached):
        batch = build_attention_batch(new, cached, tables, page, device="cuda")
        _with_slots([a for a, n in zip(adapters, new) for _ in range(n)])
        rows = torch.cat([x[s, c : c + n] for s, (n, c) in enumerate(zip(new, cached))])
        got = model.forward_paged(rows, caches, batch)
        assert torch.allclose(got, torch.cat([want[s, c : c + n] for s, (n, c) in enumerate(zip(new, cached))]), **bound)

    prompts([37, 20, 30], [0, 0, 0])
    prompts([0, 0, 36], [37, 20, 30])
    for step in range(4):
        at = [n + step for n in lens]
        _with_slots(adapters)
        batch = build_attention_batch([1, 1, 1], at, tables, page, device="cuda")
        got = model.forward_paged(torch.stack([x[s, p] for s, p in enumerate(at)]), caches, batch)
        assert torch.allclose(got, torch.stack([want[s, p] for s, p in enumerate(at)]), **bound)


@torch.no_grad()
def test_decode_step_in_a_graph_with_padding():
    from nanovllm_voxcpm_amd.layers.attention import build_attention_batch

    model, g = _model(torch.bfloat16, qk_norm=True, window=40, sinks=4), torch.Generator().manual_seed(4)
    caches = model.make_paged_cache(32, 16, torch.bfloat16, "cuda")
    for pair in caches:
        for c in pair:
            c.copy_(torch.randn(c.shape, generator=g))
    held = build_attention_batch([1] * 5, [0] * 5, [[0, 1, 2, 3, 4, 5]] * 5, 16, device="cuda", rows=8, blocks=6)
    x = torch.zeros(8, 256, dtype=torch.bfloat16, device="cuda")
    model.forward_paged(x, caches, held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.forward_paged(x, caches, held)
    for step in range(4):
        n = 5 - step % 2
        tables = torch.randperm(30, generator=g)[: 6 * n].view(n, 6).tolist()
        batch = build_attention_batch([1] * n, [30 + 11 * s + step for s in range(n)], tables, 16, device="cuda", rows=8, blocks=6)
        x.copy_(torch.randn(8, 256, generator=g).to(torch.bfloat16))
        for name in ("positions", "slot_mapping", "block_tables", "context_lens"):
            getattr(held, name).copy_(getattr(batch, name))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, model.forward_paged(x, caches, batch)), step


@torch.no_grad()
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_layer_against_the_definition(dtype):
    from nanovllm_voxcpm_amd.layers.attention import PagedAttention, build_attention_batch

    g = torch.Generator().manual_seed(5)
    heads, kv_heads, dim, page = 6, 2, 64, 16
    layer = PagedAttention(heads, kv_heads, dim, qk_norm=True, window=30, sinks=3, rotary_dim=32, max_position=256).to(device="cuda", dtype=dtype)
    layer.q_norm.copy_(1 + 0.1 * torch.randn(dim, generator=g))
    layer.k_norm.copy_(1 + 0.1 * torch.randn(dim, generator=g))
    caches = [torch.zeros(9, page, kv_heads, dim, dtype=dtype, device="cuda") for _ in range(2)]
    qkv = torch.randn(90, (heads + 2 * kv_heads) * dim, generator=g).to(dtype).cuda()
    batch = build_attention_batch([90], [0], [[8, 0, 2, 5, 1, 7]], page, device="cuda")
    got = layer(qkv, *caches, batch).view(90, heads, dim).cpu().double()
    table = layer.prepare("cuda").cpu()
    q, k, v = (p.view(90, -1, dim).cpu() for p in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1))
    # the operands as they are rounded in between, then the attention of those
    q, _ = oracle.rotate(q, torch.arange(90), table, layer.q_norm.cpu())
    k, _ = oracle.rotate(k, torch.arange(90), table, layer.k_norm.cpu())
    want, bound = oracle.attend(q, k, v, True, 30, 3, dtype=dtype)
    # q and k are off by half a step each before they meet (and by their own fp32 error, below a step of fp32 times 40): a score by as much of
    # its terms, a weight by as much relative to itself, and so the result, numerator and sum
    step = oracle.HALF_STEP[dtype] + 40 * 2.0**-24
    terms = torch.einsum("ihd,jhd->ijh", q.abs(), k.abs().repeat_interleave(heads // kv_heads, dim=1)).amax() * dim**-0.5
    spread = 2 * torch.expm1(2 * step * (1 + step) * terms) * v.double().abs().amax()
    assert ((got - want).abs() <= bound + spread).all()
    # one more token
    more = torch.randn(1, (heads + 2 * kv_heads) * dim, generator=g).to(dtype).cuda()
    step_batch = build_attention_batch([1], [90], [[8, 0, 2, 5, 1, 7]], page, device="cuda")
    whole = build_attention_batch([91], [0], [[8, 0, 2, 5, 1, 7]], page, device="cuda")
    alone = layer(more, *caches, step_batch)
    together = layer(torch.cat([qkv, more]), *caches, whole)[-1:]
    # two ways to the same row: each within its bound of the definition
    q1, _ = oracle.rotate(more[:, : heads * dim].view(1, heads, dim).cpu(), torch.tensor([90]), table, layer.q_norm.cpu())
    kk, vv = (c.view(-1, kv_heads, dim)[torch.tensor([b * page + i for b in [8, 0, 2, 5, 1, 7] for i in range(page)])[:91].cuda()].cpu() for c in caches)
    _, between = oracle.attend(q1.to(dtype), kk, vv, True, 30, 3, dtype=dtype)
    assert ((alone - together).cpu().double().view(1, heads, dim).abs() <= 2 * between).all()
