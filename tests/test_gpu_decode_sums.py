"""The two sums of decode attention, of the weights and of the weighted values, are of the same weights: the rounded ones."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# (sequences, longest): a workgroup of four wavefronts a sequence, a wide one, parts that are joined
WAYS = [(208, 1000), (3, 1000), (2, 20011)]


def _batch(sequences, longest, kv_heads, dim, dtype, page=64):
    pages = -(-longest // page)
    lens = [longest - (7 * s) % 400 for s in range(sequences)]
    shape = (sequences * pages, page, kv_heads, dim)
    tables = torch.arange(sequences * pages, dtype=torch.int32).view(sequences, pages)
    return shape, tables.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sequences,longest", WAYS)
@pytest.mark.parametrize("scores", ["random", "alike"])
def test_equal_values_come_back(scores, dtype, dim, sequences, longest):
    """With v_j = c for every key sum p c / sum p is c.  A weight times an element is exact in fp32 (8 + 8 or 11 + 11 bits), so the two sums
    differ by their additions alone, fewer than 1000 one behind the other in each: by 2000 * 2^-24, below the 2^-12 that is half the
    least distance of two fp16 values (2^-9 in bf16).  Scores alike: every 32nd key at 0 and the others at -1.1, whose weights of 0.33287 are all
    rounded the same way (bf16: by 0.0025 of themselves, fp16 0.0003)."""
    from nanovllm_voxcpm_amd.attention_ops import decode_attention

    print(scores, dtype, dim, sequences, longest, flush=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    heads, kv_heads = 4, 2
    shape, tables, lens = _batch(sequences, longest, kv_heads, dim, dtype)
    k = torch.randn(shape, generator=g, device="cuda").to(dtype)
    c = torch.randn(kv_heads, dim, generator=g, device="cuda").to(dtype)
    q = (1.5 * torch.randn(sequences, heads, dim, generator=g, device="cuda")).to(dtype)
    if scores == "alike":
        k[..., 0] = -1.0
        k[:, ::32, :, 0] = 0.0
        q = torch.zeros_like(q)
        q[..., 0] = 1.0
    got = decode_attention(q, k, c.expand(shape).contiguous(), tables, lens, scale=1.1 if scores == "alike" else None)
    assert torch.equal(got, c.repeat_interleave(heads // kv_heads, dim=0).expand_as(got))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sequences,longest", WAYS)
def test_small_weights_of_many_keys_count(dim, sequences, longest):
    """fp16: one key of weight 1 with a value of 0, n others of weight 2^-25.5 with values of 1, below fp16's numbers unless they are held larger.
    Their weights are off by half a step (2^-11) each, numerator and sum, the result by another: 3 * 2^-11 of it, and 2^-12 of it
    for fp32's products, exponentials and additions (2^-24 * 25.5 * 2 in the exponent, fewer than 1000 additions in each sum)."""
    from nanovllm_voxcpm_amd.attention_ops import decode_attention

    print(dim, sequences, longest, flush=True)
    shape, tables, lens = _batch(sequences, longest, 1, dim, torch.float16)
    k, v = torch.zeros(shape, device="cuda", dtype=torch.float16), torch.ones(shape, device="cuda", dtype=torch.float16)
    k[..., 0] = -51.0
    first = tables[:, 0].long()
    k[first, 5], v[first, 5] = 0.0, 0.0
    q = torch.zeros(sequences, 2, dim, device="cuda", dtype=torch.float16)
    q[..., 0] = 1.0
    got = decode_attention(q, k, v, tables, lens, scale=0.5 * math.log(2.0)).double()
    others = (lens.double() - 1) * 2.0**-25.5
    want = (others / (1 + others))[:, None, None].expand_as(got)
    # (the results are below fp16's least normal number, 2^-14, for the short sequences: steps of 2^-24 there)
    assert ((got - want).abs() <= 3.5 * 2.0**-11 * want + 2.0**-25).all(), ((got - want).abs() / want).max().item()
