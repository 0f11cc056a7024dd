"""Head and rotary sizes of the paged attention layer."""

import pytest
import torch

from oracle import attention as oracle

pytestmark = pytest.mark.gpu


@torch.no_grad()
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_layer_that_does_not_rotate_stores_and_reads_heads_as_they_are(dtype):
    from nanovllm_voxcpm_amd.layers.attention import PagedAttention, build_attention_batch

    g = torch.Generator().manual_seed(1)
    rows, heads, kv_heads, dim, page = 37, 4, 2, 64, 16
    layer = PagedAttention(heads, kv_heads, dim, rotary_dim=0, max_position=8).cuda()  # (positions beyond 8 turn nothing)
    qkv = torch.randn(rows, (heads + 2 * kv_heads) * dim, generator=g).to(dtype)
    caches = [torch.zeros(3, page, kv_heads, dim, dtype=dtype, device="cuda") for _ in range(2)]
    got = layer(qkv.cuda(), *caches, build_attention_batch([rows], [0], [[2, 0, 1]], page, device="cuda")).view(rows, heads, dim)
    q, k, v = (p.view(rows, -1, dim) for p in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1))
    place = torch.tensor([[2, 0, 1][p // page] * page + p % page for p in range(rows)])
    assert torch.equal(caches[0].cpu().view(-1, kv_heads, dim)[place], k) and torch.equal(caches[1].cpu().view(-1, kv_heads, dim)[place], v)
    want, bound = oracle.attend(q, k, v, dtype=dtype)
    assert ((got.cpu().double() - want).abs() <= bound).all()
