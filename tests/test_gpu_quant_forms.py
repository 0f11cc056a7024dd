"""The linear over 8-bit rows at the sizes where another kernel, tile or order of rows serves it, and what the forms have to share: results, rows without an adapter, numbers that are none."""

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


def _adapters(g, slots, rank, k, columns, dtype):
    a = [(torch.randn(slots, rank, k, generator=g) / math.sqrt(k)).to(dtype) for _ in columns]
    b = [(torch.randn(slots, n, rank, generator=g) / math.sqrt(rank)).to(dtype) for n in columns]
    return a, b


def _call(x, w, **kw):
    from nanovllm_voxcpm_amd.quant_ops import QuantizedRows, quantized_linear

    move = lambda v: [t.cuda() for t in v] if isinstance(v, (list, tuple)) and v and torch.is_tensor(v[0]) else v.cuda() if torch.is_tensor(v) else v  # noqa: E731
    return quantized_linear(QuantizedRows(*(t.cuda() for t in x)), QuantizedRows(*(t.cuda() for t in w)), **{n: move(v) for n, v in kw.items()})


def _check(x, w, a, b, of, dtype, columns=None, bias=None):
    want, bound = oracle.linear(*x, *w, bias=bias, a=a, b=b, columns=columns, slots=of, dtype=dtype)
    got = _call(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of, lora_columns=columns, bias=bias)
    off = (got.cpu().double() - want).abs() - bound
    assert not got.isnan().any() and off.max().item() <= 0, off.max().item()
    base = _call(x, w, dtype=dtype, bias=bias)
    want, bound = oracle.linear(*x, *w, bias=bias, dtype=dtype)
    assert ((base.cpu().double() - want).abs() <= bound).all()
    without = (of < 0) | (of >= a[0].size(0))
    assert torch.equal(got.cpu()[without], base.cpu()[without])
    assert torch.equal(_call(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of, lora_columns=columns, bias=bias), got)  # the same every time


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40])
@pytest.mark.parametrize("t,k", [(1, 16), (1, 1040), (1, 2048), (1, 2064), (2, 144), (2, 2048), (3, 128)])
def test_one_or_two_rows(dtype, rank, t, k):
    """Around what one launch serves: ranks, K and rows; targets that meet inside sixteen columns, and columns of none."""
    print(dtype, rank, t, k, flush=True)
    g = torch.Generator().manual_seed(rank * 10 + t + k)
    n = 77
    x, w = _rows8(g, t, k), _rows8(g, n, k, k**-0.5)
    a, b = _adapters(g, 4, rank, k, [20, 3, 30], dtype)
    bias = torch.randn(n, generator=g).to(dtype)
    for of in ([3, 0, 3], [2, 2, 2], [-1, 1, 4], [-1, -1, -1]):
        _check(x, w, a, b, torch.tensor(of[:t], dtype=torch.int32), dtype, [5, 25, 40], bias)


@pytest.mark.parametrize("t", [1, 2, 40, 200])
@pytest.mark.parametrize("dtype", HALVES)
def test_numbers_that_are_none_in_few_rows(dtype, t):
    g = torch.Generator().manual_seed(t)
    k, n, rank = 144, 50, 16
    x, w = _rows8(g, t, k), _rows8(g, n, k, k**-0.5)
    a, b = _adapters(g, 9, rank, k, [n], dtype)
    of = (torch.arange(t, dtype=torch.int32) * 7 + 1) % 10 - 1  # (1 is slot 0's, and of two rows the other is slot 7's)
    want, bound = oracle.linear(*x, *w, a=a, b=b, slots=of, dtype=dtype)
    b[0][7, 30, 3], b[0][7, 31, 4] = NAN, INF
    a[0][0, 5, 17] = NAN
    got = _call(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of).cpu()
    bad = torch.zeros(t, n, dtype=torch.bool)
    bad[of == 0] = True
    bad[of == 7, 30] = bad[of == 7, 31] = True
    assert torch.equal(~got.isfinite(), bad)
    assert ((got.double() - want).abs() <= bound)[~bad].all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t", [33, 64, 65, 255, 256, 257])
def test_rows_in_the_order_of_their_slots(dtype, t):
    """Few slots and many, some rows without one, ranks of one piece and of several, that fill a group of 32 or do not."""
    print(dtype, t, flush=True)
    g = torch.Generator().manual_seed(t)
    for slots, rank in ((7, 16), (8, 32), (50, 24), (300, 8), (20, 13)):
        k, columns = 208, [33, 15]
        x, w = _rows8(g, t, k), _rows8(g, 48, k, k**-0.5)
        a, b = _adapters(g, slots, rank, k, columns, dtype)
        for of in (torch.randint(-1, slots, (t,), generator=g, dtype=torch.int32), torch.full((t,), slots - 1, dtype=torch.int32), torch.arange(t, dtype=torch.int32) // 5 % (slots + 1) - 1):
            _check(x, w, a, b, of, dtype)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rank", [16, 20, 72])
@pytest.mark.parametrize("t,k,n", [(300, 128, 70), (700, 144, 4200), (900, 16, 4096), (1000, 272, 4000), (1100, 400, 4104), (2100, 112, 4096), (9000, 16, 1030), (4500, 48, 2048)])
def test_tiles_of_every_size(dtype, rank, t, k, n):
    """Tiles of 64 x 64, 64 x 128 and 128 x 128, several to a workgroup, of one step along K, two, three and four, that end inside rows, columns and K."""
    print(dtype, rank, t, k, n, flush=True)
    g = torch.Generator().manual_seed(t + k + n + rank)
    x, w = _rows8(g, t, k), _rows8(g, n, k, k**-0.5)
    slots, columns = 11, [n // 3, n // 2]
    a, b = _adapters(g, slots, rank, k, columns, dtype)
    some = torch.randint(-1, slots, (t,), generator=g, dtype=torch.int32)
    runs = (torch.arange(t, dtype=torch.int32) // 90) % (slots + 1) - 1
    # (the definition row by row where rows are, but not all of ten thousand)
    rows = torch.cat([torch.arange(0, t, max(1, t // 150)), torch.arange(max(0, t - 70), t)]).unique()
    for of in (some, runs):
        got = _call(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of).cpu()
        want, bound = oracle.linear(x[0][rows], x[1][rows], *w, a=a, b=b, slots=of[rows], dtype=dtype)
        assert not got.isnan().any() and ((got[rows].double() - want).abs() <= bound).all()
        base = _call(x, w, dtype=dtype).cpu()
        assert torch.equal(got[of < 0], base[of < 0])
        want, bound = oracle.linear(x[0][rows], x[1][rows], *w, dtype=dtype)
        assert ((base[rows].double() - want).abs() <= bound).all()
        # a row's result is its own: the same among fewer rows of the same tiles' kernel
        again = _call(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of)
        assert torch.equal(again.cpu(), got)


def test_more_rows_than_one_trip_of_the_order_takes():
    g = torch.Generator().manual_seed(8)
    t, k, n, slots, dtype = 33000, 32, 40, 300, torch.bfloat16
    x, w = _rows8(g, t, k), _rows8(g, n, k, k**-0.5)
    a, b = _adapters(g, slots, 8, k, [n], dtype)
    of = torch.randint(-1, slots, (t,), generator=g, dtype=torch.int32)
    got = _call(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of).cpu()
    rows = torch.randperm(t, generator=g)[:500]
    want, bound = oracle.linear(x[0][rows], x[1][rows], *w, a=a, b=b, slots=of[rows], dtype=dtype)
    assert ((got[rows].double() - want).abs() <= bound).all()
    # all of them, against the same rows in calls of 200
    for first in range(0, t, 6600):
        part = slice(first, first + 200)
        want, bound = oracle.linear(x[0][part], x[1][part], *w, a=a, b=b, slots=of[part], dtype=dtype)
        assert ((got[part].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", HALVES)
def test_rows_too_far_apart_for_tiles(dtype):
    """A weight whose rows are more than 4 MB apart, and many rows: the kernel for few of them serves the call."""
    g = torch.Generator().manual_seed(9)
    t, k, n = 330, 144, 20
    x, w = _rows8(g, t, k), _rows8(g, n, k, k**-0.5)
    home = torch.zeros(n, (1 << 22) + 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    home[:, :k].copy_(w[0])
    a, b = _adapters(g, 9, 16, k, [n], dtype)
    of = torch.randint(-1, 9, (t,), generator=g, dtype=torch.int32)
    from nanovllm_voxcpm_amd.quant_ops import QuantizedRows, quantized_linear

    got = quantized_linear(QuantizedRows(x[0].cuda(), x[1].cuda()), QuantizedRows(home[:, :k], w[1].cuda()), dtype=dtype, lora_a=[v.cuda() for v in a], lora_b=[v.cuda() for v in b], token_to_slot=of.cuda())
    want, bound = oracle.linear(*x, *w, a=a, b=b, slots=of, dtype=dtype)
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("t", [1, 2, 70, 600])
def test_the_python_path_makes_the_same_call(t, monkeypatch):
    from nanovllm_voxcpm_amd import _hip
    from nanovllm_voxcpm_amd.quant_ops import add_rms_norm, quantize_rows, silu_mul

    g = torch.Generator().manual_seed(t)
    x, w = _rows8(g, t, 144), _rows8(g, 90, 144)
    a, b = _adapters(g, 5, 16, 144, [30, 60], torch.float16)
    of = torch.randint(-1, 5, (t,), generator=g, dtype=torch.int32)
    y, r, weight = (torch.randn(t, 288, generator=g).half().cuda(), torch.randn(t, 288, generator=g).half().cuda(), torch.randn(288, generator=g).cuda())

    def calls():
        norm, total = add_rms_norm(y, weight, residual=r, quantize=True)
        return [_call(x, w, dtype=torch.float16, lora_a=a, lora_b=b, token_to_slot=of, bias=torch.ones(90).half()), *norm, total, add_rms_norm(y, weight)[0], *quantize_rows(y), silu_mul(y), *silu_mul(y, quantize=True)]

    assert _hip.load_fastcall() is not None
    want = calls()
    monkeypatch.setattr(_hip, "load_fastcall", lambda: None)
    for got, one in zip(calls(), want):
        assert got.dtype == one.dtype and torch.equal(got.float(), one.float())


def test_two_graphs_in_turn():
    """Two captured graphs of one memory pool, with few rows and with many, replayed in turn between eager calls, while rows and slots change."""
    from nanovllm_voxcpm_amd.quant_ops import QuantizedRows, quantized_linear

    g = torch.Generator().manual_seed(10)
    k, n, dtype = 144, 96, torch.bfloat16
    w = QuantizedRows(*(v.cuda() for v in _rows8(g, n, k, k**-0.5)))
    a, b = _adapters(g, 9, 16, k, [n], dtype)
    a, b = [v.cuda() for v in a], [v.cuda() for v in b]
    held, graphs, pool = [], [], None
    for t in (1, 50, 400):
        x = QuantizedRows(*(v.cuda() for v in _rows8(g, t, k)))
        of = torch.full((t,), -1, dtype=torch.int32, device="cuda")
        call = lambda x=x, of=of: quantized_linear(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of)  # noqa: E731
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = call()
        pool = graph.pool()
        held.append((x, of, call, out))
        graphs.append(graph)
    for step in range(6):
        for i in torch.randperm(3, generator=g).tolist():
            x, of, call, out = held[i]
            fresh = _rows8(g, of.numel(), k)
            x.values.copy_(fresh[0])
            x.scales.copy_(fresh[1])
            of.copy_(torch.randint(-1, 9, (of.numel(),), generator=g, dtype=torch.int32))
            graphs[i].replay()
            got = out.clone()
            assert torch.equal(got, call()), (step, i)


@pytest.mark.parametrize("rank", [8, 20])
@pytest.mark.parametrize("k", [16, 128, 144])
def test_many_tiles_of_one_step_and_two(rank, k):
    """Workgroups with many tiles of a step or two, whose wavefronts take different times at a tile's end (ranks that are no multiple of eight most of all): the same every time, and the definition's."""
    g = torch.Generator().manual_seed(rank + k)
    t, n, slots, dtype = 9000, 2048, 11, torch.float16
    x, w = _rows8(g, t, k), _rows8(g, n, k, k**-0.5)
    a, b = _adapters(g, slots, rank, k, [n // 3, n // 2], dtype)
    x, w, a, b = ([v.cuda() for v in group] for group in (x, w, a, b))
    of = torch.randint(-1, slots, (t,), generator=g, dtype=torch.int32)
    first = _call(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of)
    rows = torch.randperm(t, generator=g)[:300]
    held = [v.cpu() for v in (x[0].float().cpu()[rows], x[1].cpu()[rows], w[0].float(), w[1])]
    want, bound = oracle.linear(*held, a=[v.cpu() for v in a], b=[v.cpu() for v in b], slots=of[rows], dtype=dtype)
    assert ((first.cpu()[rows].double() - want).abs() <= bound).all()
    for _ in range(30):
        assert torch.equal(_call(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of), first)
