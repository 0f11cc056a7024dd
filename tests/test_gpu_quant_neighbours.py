"""A row's result is its own: among as many rows it is the same, bit for bit, whichever adapters and whatever numbers the other rows have, in every form."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALVES = [torch.bfloat16, torch.float16]


def _rows8(g, n, k, scale=1.0):
    x = torch.randn(n, k, generator=g) * scale
    scales = (x.abs().amax(-1) / 448).clamp(min=2.0**-100)
    return (x / scales[:, None]).to(torch.float8_e4m3fn), scales


# one launch for one or two rows, rows by themselves (two, four and eight wavefronts to a block of sixteen; in their own order and sorted), tiles of three sizes
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rank", [8, 13, 16, 24, 32, 40, 64, 72, 136])
@pytest.mark.parametrize("t,k,n,slots", [(2, 144, 40, 7), (9, 1040, 70, 12), (16, 256, 4200, 12), (30, 400, 100, 30), (64, 272, 100, 6), (64, 272, 4100, 40), (200, 1040, 90, 20), (300, 144, 90, 9),
                                         (700, 272, 4200, 20), (1100, 144, 4104, 5)])
def test_other_rows_change_nothing(dtype, rank, t, k, n, slots):
    from nanovllm_voxcpm_amd.quant_ops import QuantizedRows, quantized_linear

    print(dtype, rank, t, k, n, slots, flush=True)
    g = torch.Generator().manual_seed(t + rank)
    w = QuantizedRows(*(v.cuda() for v in _rows8(g, n, k, k**-0.5)))
    widths = [n // 3, n // 2]
    a = [(torch.randn(slots, rank, k, generator=g) / math.sqrt(k)).to(dtype).cuda() for _ in widths]
    b = [(torch.randn(slots, wide, rank, generator=g) / math.sqrt(rank)).to(dtype).cuda() for wide in widths]
    values, scales = _rows8(g, t, k)
    of = torch.randint(-1, slots, (t,), generator=g, dtype=torch.int32)
    kept = torch.rand(t, generator=g) < 0.3
    kept[t // 2] = True
    of[t // 2] = slots - 1

    def call():
        return quantized_linear(QuantizedRows(values.cuda(), scales.cuda()), w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of.cuda()).cpu()[kept]

    want = call()
    assert want.isfinite().all()
    for change in range(5):
        other = _rows8(g, t, k, 3.0)
        values = torch.where(kept[:, None], values.view(torch.uint8), other[0].view(torch.uint8)).view(torch.float8_e4m3fn)
        scales = torch.where(kept, scales, other[1])
        new = [torch.full((t,), -1), torch.full((t,), slots - 1), torch.arange(t) % slots, torch.randint(-1, slots, (t,), generator=g), torch.randint(0, min(slots, 3), (t,), generator=g)][change]
        of = torch.where(kept, of, new.int())
        assert torch.equal(call(), want), (change, (call() != want).sum().item())
