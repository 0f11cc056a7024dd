"""How many bits of the adapters' intermediate reach the result: ranks that cancel, so that what is left is far smaller than what they add, in every form."""

import math

import pytest
import torch

from oracle import quant as oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank", [16, 20, 32, 72])
@pytest.mark.parametrize("t,k,n", [(1, 64, 40), (2, 144, 40), (9, 272, 70), (30, 144, 50), (60, 272, 4200), (200, 144, 70), (300, 272, 90), (700, 400, 4200), (1100, 144, 4104)])
def test_ranks_that_cancel(dtype, rank, t, k, n):
    from nanovllm_voxcpm_amd.quant_ops import QuantizedRows, quantized_linear

    print(dtype, rank, t, k, n, flush=True)
    g = torch.Generator().manual_seed(t + rank)
    x = torch.randn(t, k, generator=g)
    scales = x.abs().amax(-1) / 448
    x = (x / scales[:, None]).to(torch.float8_e4m3fn)
    w, w_scales = torch.zeros(n, k, dtype=torch.float8_e4m3fn), torch.full((n,), 2.0**-100)  # (no base product, whose instruction keeps fewer bits)
    slots = 5
    # of every two ranks B is the same with opposite signs, and A nearly the same: h differs by 2^-6 of itself
    a = torch.randn(slots, rank // 2, 1, k, generator=g).expand(-1, -1, 2, -1).reshape(slots, rank, k) / math.sqrt(k)
    a = (a * (1 + 2.0**-6 * torch.randn(slots, rank, k, generator=g))).to(dtype)
    b = torch.randn(slots, n, rank // 2, 1, generator=g)
    b = torch.cat([b, -b], dim=-1).reshape(slots, n, rank).to(dtype)
    of = torch.randint(-1, slots, (t,), generator=g, dtype=torch.int32)
    of[0] = 2
    rows = torch.arange(t) if t <= 300 else torch.arange(0, t, t // 100)
    want, bound = oracle.linear(x[rows], scales[rows], w, w_scales, a=[a], b=[b], slots=of[rows], dtype=dtype)
    got = quantized_linear(QuantizedRows(x.cuda(), scales.cuda()), QuantizedRows(w.cuda(), w_scales.cuda()), dtype=dtype, lora_a=[a.cuda()], lora_b=[b.cuda()], token_to_slot=of.cuda())
    off = (got.cpu()[rows].double() - want).abs() - bound
    assert off.max().item() <= 0, off.max().item()
