"""Infinities and NaN in the adapters beside an 8-bit linear: what the definition makes of them, in every form, and nowhere but in the rows of their slot and the columns of their target."""

import math

import pytest
import torch

from oracle import quant as oracle

pytestmark = pytest.mark.gpu

HALVES = [torch.bfloat16, torch.float16]
NAN, INF = float("nan"), float("inf")


def _rows8(g, n, k, scale=1.0):
    x = torch.randn(n, k, generator=g) * scale
    scales = (x.abs().amax(-1) / 448).clamp(min=2.0**-100)
    return (x / scales[:, None]).to(torch.float8_e4m3fn), scales


def _call(x, w, a, b, of, dtype, columns):
    from nanovllm_voxcpm_amd.quant_ops import QuantizedRows, quantized_linear

    return quantized_linear(QuantizedRows(*(t.cuda() for t in x)), QuantizedRows(*(t.cuda() for t in w)), dtype=dtype, lora_a=[t.cuda() for t in a], lora_b=[t.cuda() for t in b],
                            token_to_slot=of.cuda(), lora_columns=columns).cpu()


# forms: one launch for one or two rows, rows by themselves (unsorted, sorted), tiles of 64 x 64, of 64 x 128 and of 128 x 128
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rank", [16, 20, 72])
@pytest.mark.parametrize("t,k,widths,columns", [(1, 64, [33, 60], [0, 33]), (2, 144, [33, 60], [5, 41]), (24, 144, [33, 100], [0, 33]), (60, 272, [33, 60], [5, 41]), (200, 144, [33, 100], [3, 36]),
                                                (400, 112, [33, 100], [0, 40]), (700, 400, [1000, 1500], [90, 1111]), (1100, 144, [2011, 2000], [3, 2020])])
def test_what_the_definition_makes_of_them(dtype, rank, t, k, widths, columns):
    print(dtype, rank, t, k, widths, columns, flush=True)
    g = torch.Generator().manual_seed(t + rank)
    slots, n = 9, columns[-1] + widths[-1] + 7
    x, w = _rows8(g, t, k), _rows8(g, n, k, k**-0.5)
    a = [(torch.randn(slots, rank, k, generator=g) / math.sqrt(k)).to(dtype) for _ in widths]
    b = [(torch.randn(slots, wide, rank, generator=g) / math.sqrt(rank)).to(dtype) for wide in widths]
    of = (torch.arange(t, dtype=torch.int32) * 7 + 1) % (slots + 1) - 1  # (slot 0 first, then slot 7)
    a[0][0, rank - 3, 17], a[1][7, 2, 5] = NAN, INF
    a[0][3, 4, 9], a[0][3, 5, 9] = -INF, INF
    b[0][4, 30, 3], b[0][4, 31, 4], b[1][4, 7, rank - 1], b[1][5, 8, 0] = NAN, INF, -INF, INF
    rows = torch.arange(t) if t <= 400 else torch.cat([torch.arange(0, t, t // 100), torch.arange(t - 40, t)]).unique()
    want, bound = oracle.linear(x[0][rows], x[1][rows], *w, a=a, b=b, columns=columns, slots=of[rows], dtype=dtype)
    got = _call(x, w, a, b, of, dtype, columns)[rows].double()
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(kind(got), kind(want)), (kind.__name__, int(kind(got).sum()), int(kind(want).sum()))
    finite = want.isfinite()
    assert bound[finite].isfinite().all() and ((got - want).abs() <= bound)[finite].all()
