"""Calls with more rows and heads than a launch has room for along one dimension (2^32 threads): a single key's value comes back for every one."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_more_rows_and_heads_than_one_dimension_of_a_launch():
    """2^26 and some (row, head) units, of 64 threads each."""
    from nanovllm_voxcpm_amd.attention_ops import decode_attention, prompt_attention

    n, heads, dim = (1 << 20) + 3, 64, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    v = torch.randn(n, 1, dim, generator=g, device="cuda", dtype=torch.float16)
    q = torch.ones(n, heads, dim, device="cuda", dtype=torch.float16)
    assert torch.equal(prompt_attention(q, v, v, torch.arange(n + 1, dtype=torch.int32, device="cuda")), v.expand(n, heads, dim))
    lens, tables = torch.ones(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")[:, None]
    cache = v.view(n, 1, 1, dim)
    assert torch.equal(decode_attention(q, cache, cache, tables, lens), v.expand(n, heads, dim))


def test_more_sequences_than_one_dimension_of_a_launch():
    """2^24 and some sequences, of a workgroup of 256 threads each in the kernel of head size 64."""
    from nanovllm_voxcpm_amd.attention_ops import decode_attention

    n, dim = (1 << 24) + 5, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    cache = torch.randn(3, 16, 1, dim, generator=g, device="cuda", dtype=torch.bfloat16)
    q = torch.ones(1, 1, dim, device="cuda", dtype=torch.bfloat16).expand(n, 1, dim)
    tables = torch.full((n, 1), 2, dtype=torch.int32, device="cuda")
    tables[-1] = 1
    got = decode_attention(q, cache, cache, tables, torch.ones(n, dtype=torch.int32, device="cuda"))
    assert torch.equal(got[:-1], cache[2, 0].expand(n - 1, 1, dim)) and torch.equal(got[-1], cache[1, 0])
