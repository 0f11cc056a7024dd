"""Rows in 8 bits are what their formula says, bit for bit: scale = max(max|x| / 448, 2^-100) and values = e4m3(x / scale), each step rounded in fp32; and what the norm and the gate put in 8
bits are the rows that they give in fp32."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _definition(x):
    scales = (x.float().abs().amax(-1) / 448).clamp(min=2.0**-100)
    return (x.float() / scales[:, None]).to(torch.float8_e4m3fn), scales


def _same(rows, want):
    assert torch.equal(rows.scales.cpu(), want[1].cpu())
    assert torch.equal(rows.values.cpu().view(torch.uint8), want[0].cpu().view(torch.uint8)), int((rows.values.cpu().float() != want[0].cpu().float()).sum())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,width", [(4000, 64), (700, 513), (500, 1024), (300, 2048), (200, 5000), (60, 9000), (20, 40001)])
def test_values_and_scales_are_the_formula(dtype, rows, width):
    from nanovllm_voxcpm_amd.quant_ops import quantize_rows

    g = torch.Generator().manual_seed(rows + width)
    x = (torch.randn(rows, width, generator=g) * torch.exp(4 * torch.randn(rows, 1, generator=g))).to(dtype)
    x[0] = 0
    _same(quantize_rows(x.cuda()), _definition(x))
    # ties: numbers half way between two of e4m3, times a power of two that the scale takes away again
    if width >= 513:
        x = torch.zeros(3, width)
        grid = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
        x[:, :126] = (grid[1:] + grid[:-1]) / 2
        x[:, 126], x[1], x[2] = 448, x[1] * 4, x[2] * -0.125
        x[:, 126] = torch.tensor([448, 1792, 56])
        _same(quantize_rows(x.to(dtype).cuda()), _definition(x.to(dtype)))


@pytest.mark.parametrize("rows,width", [(2000, 64), (300, 513), (200, 2048), (100, 5000), (20, 20001)])
def test_the_norm_and_the_gate_put_their_fp32_rows_in_8_bits(rows, width):
    from nanovllm_voxcpm_amd.quant_ops import add_rms_norm, quantize_rows, silu_mul

    g = torch.Generator().manual_seed(rows + width)
    x, residual = ((torch.randn(rows, width, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).cuda() for _ in range(2))
    weight = torch.randn(width, generator=g).cuda()
    for other in (None, residual):
        _same(add_rms_norm(x, weight, residual=other, quantize=True)[0], quantize_rows(add_rms_norm(x, weight, residual=other)[0]))
    both = torch.cat([x, residual], dim=1)
    _same(silu_mul(both, quantize=True), quantize_rows(silu_mul(both)))
