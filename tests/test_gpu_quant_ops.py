"""Rows in 8 bits, norm with residual, gate and the linear over 8-bit rows with adapters, against the definitions in 64 bits, at the
sizes, layouts and values where they can go wrong."""

import math

import pytest
import torch

from oracle import quant as oracle
from oracle.attention import HALF_STEP

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
HALVES = [torch.bfloat16, torch.float16]
NAN, INF = float("nan"), float("inf")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _within(got, want, bound, what=""):
    got = got.cpu().double()
    assert got.shape == want.shape, what
    assert not torch.isnan(got).any(), what
    wrong = (got - want).abs() - bound
    assert not got.numel() or wrong.max().item() <= 0, (what, wrong.max().item(), (got - want).abs().max().item())


def _in_eight(rows, y, wrong, what=""):
    scales, scales_off, values, off = oracle.eight_bits(y, wrong)
    assert rows.values.dtype == torch.float8_e4m3fn and rows.scales.dtype == torch.float32
    _within(rows.scales, scales, scales_off, what)
    _within(rows.values.float(), values, off, what)


def _in_type(got, y, wrong, dtype, what=""):
    assert got.dtype == dtype
    off = y.abs() * wrong
    _within(got, y, off + (y.abs() + off) * HALF_STEP[dtype] + (2.0**-25 if dtype == torch.float16 else 2.0**-110), what)


SIZES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 511), (4, 512), (7, 513), (1, 1024), (67, 1024), (3, 1025), (5, 2048), (2, 2056), (3, 4096), (2, 5000), (2, 8192),
         (1, 8200), (2, 12289), (1, 32768), (2, 32769), (1, 70001), (1000, 96)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", SIZES)
def test_rows_of_every_width(dtype, rows, width):
    from nanovllm_voxcpm_amd.quant_ops import add_rms_norm, quantize_rows, silu_mul

    print(dtype, rows, width, flush=True)
    g = _gen(rows * 100003 + width)
    x, other = (torch.randn(rows, width, generator=g).to(dtype) for _ in range(2))
    weight = 1 + 0.3 * torch.randn(width, generator=g)
    _in_eight(quantize_rows(x.cuda()), x.double(), 0.0)
    for residual in (None, other):
        for w in (weight, weight.to(dtype)):
            total, y, wrong = oracle.add_rms_norm(x, w, residual, 1e-5)
            on = None if residual is None else residual.cuda()
            got, s = add_rms_norm(x.cuda(), w.cuda(), residual=on, eps=1e-5)
            assert torch.equal(s.cpu(), total)
            _in_type(got, y, wrong, dtype)
            got, s = add_rms_norm(x.cuda(), w.cuda(), residual=on, eps=1e-5, quantize=True)
            assert torch.equal(s.cpu(), total)
            _in_eight(got, y, wrong)
    gate_up = torch.cat([3 * x, other], dim=1)
    y, wrong = oracle.silu_mul(gate_up)
    _in_type(silu_mul(gate_up.cuda()), y, wrong, dtype)
    _in_eight(silu_mul(gate_up.cuda(), quantize=True), y, wrong)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_other_strides_and_at_odd_places(dtype):
    """Columns of a wider buffer, rows at any element, a row that all rows share; sums in place of either input and between other columns, whose neighbours stay."""
    from nanovllm_voxcpm_amd.quant_ops import add_rms_norm, quantize_rows, silu_mul

    g = _gen(5)
    for width in (64, 1003, 2040, 9000):
        wide = torch.randn(9, 2 * width + 5, generator=g).to(dtype).cuda()
        weight = torch.randn(width, generator=g).cuda()
        x, other = wide[:, 3 : 3 + width], wide[:, width + 4 : 2 * width + 4]
        for a in (x, x[:1].expand(9, width)):
            want = quantize_rows(a.contiguous())
            got = quantize_rows(a)
            assert torch.equal(got.values.float(), want.values.float()) and torch.equal(got.scales, want.scales)
            want, total = add_rms_norm(a.contiguous(), weight, residual=other.contiguous())
            got, s = add_rms_norm(a, weight, residual=other)
            assert torch.equal(got, want) and torch.equal(s, total)
        both = wide[:, 1 : 2 * width + 1]
        assert torch.equal(silu_mul(both), silu_mul(both.contiguous()))
        # sums into x, into the residual, and into columns of a buffer
        for place in ("x", "residual", "between"):
            buffer = wide.clone()
            a, b = buffer[:, 3 : 3 + width], buffer[:, width + 4 : 2 * width + 4]
            home = torch.full((9, width + 3), 7.0, dtype=dtype, device="cuda")
            to = {"x": a, "residual": b, "between": home[:, 1 : 1 + width]}[place]
            want, total = add_rms_norm(x, weight, residual=other, quantize=True)
            got, s = add_rms_norm(a, weight, residual=b, quantize=True, sum_out=to)
            assert s is to and torch.equal(s, total) and torch.equal(got.values.float(), want.values.float()) and torch.equal(got.scales, want.scales)
            if place == "between":
                assert (home[:, 0] == 7).all() and (home[:, 1 + width :] == 7).all()
            else:
                kept = torch.ones(2 * width + 5, dtype=torch.bool)
                kept[3 if place == "x" else width + 4 :][:width] = False
                assert torch.equal(buffer[:, kept.cuda()], wide[:, kept.cuda()])


def test_rows_of_zeros_small_numbers_and_values_that_are_none():
    from nanovllm_voxcpm_amd.quant_ops import add_rms_norm, quantize_rows, silu_mul

    x = torch.zeros(6, 40)
    x[1, 3] = 1e-35  # the least scale holds
    x[2, 4], x[2, 5] = 3e38, -1.0
    x[3, 7], x[3, 8] = NAN, 2.0
    x[4, 1], x[4, 2] = INF, 5.0
    x[5] = torch.linspace(-448, 448, 40)
    got = quantize_rows(x.cuda())
    values, scales = got.values.float().cpu(), got.scales.cpu()
    assert scales[0] == 2.0**-100 and (values[0] == 0).all()
    assert scales[1] == 2.0**-100 and values[1, 3] == torch.tensor(1e-35 * 2.0**100).to(torch.float8_e4m3fn).float()
    assert values[2, 4] == 448 and values[2, 5] == 0
    assert scales[3].isnan() and values[3].isnan().all()
    assert scales[4] == INF and values[4, 1].isnan() and values[4, 2] == 0
    assert scales[5] == 1 and torch.equal(values[5], x[5].to(torch.float8_e4m3fn).float())
    # e4m3 numbers come back as they are, whatever their row's power of two
    numbers = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    numbers = numbers[~numbers.isnan()]
    for power in (-60, -3, 0, 9, 90):
        back = quantize_rows((numbers * 2.0**power)[None].cuda())
        assert torch.equal(back.values.float().cpu()[0], numbers) and back.scales.item() == 2.0**power
    # the norm of zeros is zeros, a NaN row is NaN and its neighbours are not
    y, _ = add_rms_norm(x.cuda(), torch.ones(40).cuda())
    assert (y[0] == 0).all() and y[3].isnan().all() and not y[5].isnan().any()
    eight, _ = add_rms_norm(x.cuda(), torch.ones(40).cuda(), quantize=True)
    assert (eight.values[0].float() == 0).all() and eight.scales[0] == 2.0**-100 and eight.values[3].float().isnan().all() and eight.scales[3].isnan()
    # gates far out: silu is 0 on the left and its argument on the right, -inf gives NaN as the formula does
    gate = torch.tensor([[-1e4, 1e4, -90.0, 0.0, -INF, INF]])
    y = silu_mul(torch.cat([gate, torch.ones(1, 6)], dim=1).cuda()).cpu()[0]
    assert y[0] == 0 and y[1] == 1e4 and abs(y[2]) < 1e-36 and y[3] == 0 and y[4].isnan() and y[5] == INF


def test_rows_that_are_none_launch_nothing():
    from nanovllm_voxcpm_amd.quant_ops import QuantizedRows, add_rms_norm, quantize_rows, quantized_linear, silu_mul

    none = torch.empty(0, 64, device="cuda")
    rows = quantize_rows(none)
    assert rows.values.shape == (0, 64) and rows.scales.shape == (0,)
    assert add_rms_norm(none, torch.ones(64).cuda(), residual=none)[0].shape == (0, 64)
    assert silu_mul(none).shape == (0, 32)
    weight = quantize_rows(torch.randn(5, 64).cuda())
    assert quantized_linear(rows, weight).shape == (0, 5)
    assert quantized_linear(weight, QuantizedRows(rows.values, rows.scales)).shape == (5, 0)


# ---- the linear ------------------------------------------------------------------------------------------------------


def _rows8(g, n, k, scale=1.0):
    x = torch.randn(n, k, generator=g) * scale
    scales = (x.abs().amax(-1) / 448).clamp(min=2.0**-100)
    return (x / scales[:, None]).to(torch.float8_e4m3fn), scales


def _call(x, w, on="cuda", **kw):
    from nanovllm_voxcpm_amd.quant_ops import QuantizedRows, quantized_linear

    move = lambda v: [t.to(on) for t in v] if isinstance(v, (list, tuple)) and v and torch.is_tensor(v[0]) else v.to(on) if torch.is_tensor(v) else v  # noqa: E731
    return quantized_linear(QuantizedRows(*(t.to(on) for t in x)), QuantizedRows(*(t.to(on) for t in w)), **{n: move(v) for n, v in kw.items()})


def _adapters(g, slots, rank, k, columns, dtype, scale=1.0):
    a = [(torch.randn(slots, rank, k, generator=g) * scale / math.sqrt(k)).to(dtype) for _ in columns]
    b = [(torch.randn(slots, n, rank, generator=g) * scale / math.sqrt(rank)).to(dtype) for n in columns]
    return a, b


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,k,n", [(1, 16, 1), (1, 1024, 1536), (3, 48, 17), (16, 128, 16), (17, 144, 33), (31, 1008, 130), (33, 2064, 64), (64, 256, 257), (65, 1024, 96),
                                   (130, 4096, 48), (200, 8208, 32), (257, 112, 300), (513, 640, 384), (1030, 272, 520)])
def test_linear_of_every_size(dtype, t, k, n):
    print(dtype, t, k, n, flush=True)
    g = _gen(t * 7 + k * 3 + n)
    x, w = _rows8(g, t, k), _rows8(g, n, k, k**-0.5)
    for bias in (None, torch.randn(n, generator=g).to(dtype)):
        want, bound = oracle.linear(*x, *w, bias=bias, dtype=dtype)
        got = _call(x, w, bias=bias, dtype=dtype)
        assert got.dtype == dtype
        _within(got, want, bound)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rank", [1, 5, 8, 16, 24, 32, 64, 72, 130, 256])
@pytest.mark.parametrize("t,k,columns", [(1, 64, [32, 16, 16]), (7, 144, [5, 1, 40]), (40, 272, [64]), (150, 128, [33, 100]), (300, 160, [136, 8])])
def test_adapters_beside_the_linear(dtype, rank, t, k, columns):
    print(dtype, rank, t, k, columns, flush=True)
    g = _gen(rank * 31 + t)
    slots, n = 6, sum(columns)
    x, w = _rows8(g, t, k), _rows8(g, n, k, k**-0.5)
    a, b = _adapters(g, slots, rank, k, columns, dtype)
    # adapters in any order, some rows without one, ids outside the slots
    of = torch.randint(-1, slots, (t,), generator=g, dtype=torch.int32)
    of[t // 2] = slots
    of[-1] = 2**31 - 1 if t % 2 else -(2**31)
    of[0] = 3
    want, bound = oracle.linear(*x, *w, a=a, b=b, slots=of, dtype=dtype)
    got = _call(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of)
    _within(got, want, bound)
    # a row without an adapter is the base product's, bit for bit
    base = _call(x, w, dtype=dtype)
    without = (of < 0) | (of >= slots)
    assert torch.equal(got.cpu()[without], base.cpu()[without])


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,slots", [(64, 64), (256, 200), (700, 3), (2100, 40)])
def test_many_adapters_and_long_runs(dtype, t, slots):
    print(dtype, t, slots, flush=True)
    g = _gen(t)
    k, columns, rank = 128, [48, 80], 16
    x, w = _rows8(g, t, k), _rows8(g, 128, k, k**-0.5)
    a, b = _adapters(g, slots, rank, k, columns, dtype)
    every = torch.arange(t, dtype=torch.int32) % slots
    runs = torch.div(torch.arange(t, dtype=torch.int32), max(1, t // 5), rounding_mode="floor") % slots
    runs[t // 3 : t // 3 + 40] = -1
    one = torch.full((t,), slots - 1, dtype=torch.int32)
    none = torch.full((t,), -1, dtype=torch.int32)
    for of in (every, runs, one, none):
        want, bound = oracle.linear(*x, *w, a=a, b=b, slots=of, dtype=dtype)
        _within(_call(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of), want, bound)


def test_columns_between_targets_and_outputs_in_a_wider_buffer():
    """Targets that leave columns free; y in columns of a buffer whose others stay as they were, rows at odd elements."""
    g = _gen(9)
    t, k, n, dtype = 37, 96, 150, torch.bfloat16
    x, w = _rows8(g, t, k), _rows8(g, n, k, k**-0.5)
    a, b = _adapters(g, 4, 16, k, [30, 50], dtype)
    of = torch.randint(-1, 4, (t,), generator=g, dtype=torch.int32)
    want, bound = oracle.linear(*x, *w, a=a, b=b, columns=[7, 90], slots=of, dtype=dtype)
    for first, width in ((0, n), (1, n + 5), (8, n + 10)):
        home = torch.full((t, width), 7.0, dtype=dtype, device="cuda")
        y = home[:, first : first + n]
        got = _call(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of, lora_columns=[7, 90], out=y)
        assert got is y
        _within(y, want, bound)
        assert (home[:, :first] == 7).all() and (home[:, first + n :] == 7).all()


def test_rows_and_weights_that_are_views():
    g = _gen(10)
    t, k, n = 50, 160, 70
    wide, w = _rows8(g, t, 3 * k), _rows8(g, n, k, k**-0.5)
    x = wide[0].cuda()[:, k : 2 * k]  # rows 480 bytes apart
    want, bound = oracle.linear(wide[0][:, k : 2 * k], wide[1], *w)
    from nanovllm_voxcpm_amd.quant_ops import QuantizedRows, quantized_linear

    weight = QuantizedRows(w[0].cuda(), w[1].cuda())
    _within(quantized_linear(QuantizedRows(x, wide[1].cuda()), weight), want, bound)
    # one row for everybody
    same = x[:1].expand(t, k)
    one = quantized_linear(QuantizedRows(same, wide[1].cuda()), weight)
    want, bound = oracle.linear(wide[0][:1, k : 2 * k].expand(t, k), wide[1], *w)
    _within(one, want, bound)


@pytest.mark.parametrize("t", [5, 100, 600])
def test_values_that_are_none_stay_in_their_rows_and_columns(t):
    g = _gen(11)
    k, n, dtype = 80, 90, torch.bfloat16  # (K ends inside a tile: what lies there is another column's NaN)
    x, w = _rows8(g, t, k), _rows8(g, n, k, k**-0.5)
    a, b = _adapters(g, 3, 16, k, [n], dtype)
    of = torch.arange(t, dtype=torch.int32) % 4 - 1
    want, bound = oracle.linear(*x, *w, a=a, b=b, slots=of, dtype=dtype)
    x[0][2, 0], w[0][17, 0] = NAN, NAN
    a[0][1, 3, 5] = NAN  # reaches rows of slot 1
    b[0][2, 40, 7] = NAN  # reaches column 40 of rows of slot 2
    got = _call(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of).cpu()
    bad = torch.zeros(t, n, dtype=torch.bool)
    bad[2], bad[:, 17], bad[of == 1] = True, True, True
    bad[of == 2, 40] = True
    assert torch.equal(got.isnan(), bad)
    assert ((got.double() - want).abs() <= bound)[~bad].all()


def test_adapters_of_large_and_small_numbers():
    """The intermediate is held to more than 16 bits and not in fp16: adapters whose products lie beyond fp16's range, or far below its normal numbers."""
    g = _gen(12)
    t, k, n = 33, 128, 48
    for dtype in HALVES:
        for up in (2.0**10, 2.0**-12):
            x, w = _rows8(g, t, k, 100.0), _rows8(g, n, k, k**-0.5 * 0.01)
            a, b = _adapters(g, 2, 8, k, [n], dtype)
            a, b = [v * up for v in a], [(v.float() / up * 0.01).to(dtype) for v in b]
            of = torch.arange(t, dtype=torch.int32) % 2
            want, bound = oracle.linear(*x, *w, a=a, b=b, slots=of, dtype=dtype)
            _within(_call(x, w, dtype=dtype, lora_a=a, lora_b=b, token_to_slot=of), want, bound)


def test_two_calls_at_once_and_another_stream():
    """Calls on two streams share nothing; a call works on the stream that is current."""
    g = _gen(13)
    t, k, n, dtype = 300, 512, 256, torch.bfloat16
    cases = []
    for i in range(2):
        x, w = _rows8(g, t, k), _rows8(g, n, k, k**-0.5)
        a, b = _adapters(g, 4, 16, k, [n], dtype)
        of = torch.randint(-1, 4, (t,), generator=g, dtype=torch.int32)
        kw = dict(lora_a=[v.cuda() for v in a], lora_b=[v.cuda() for v in b], token_to_slot=of.cuda())
        cases.append(([v.cuda() for v in x], [v.cuda() for v in w], kw))
    want = [_call(x, w, dtype=dtype, **kw) for x, w, kw in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, (s, (x, w, kw)) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(_call(x, w, dtype=dtype, **kw))
    torch.cuda.synchronize()
    for many, one in zip(got, want):
        assert all(torch.equal(v, one) for v in many)


def test_a_decoder_step_in_a_graph_follows_its_inputs():
    """norm, q|k|v, o, norm, gate|up, gate, down in one captured graph, replayed with other rows and other adapters, against the same calls by themselves."""
    from nanovllm_voxcpm_amd.quant_ops import add_rms_norm, quantize_rows, quantized_linear, silu_mul

    g = _gen(14)
    hidden, inter, t, slots, rank, dtype = 128, 256, 48, 5, 16, torch.bfloat16
    weights = {name: quantize_rows((torch.randn(n, k, generator=g) * k**-0.5).cuda()) for name, n, k in
               (("qkv", 192, hidden), ("o", hidden, hidden), ("gate_up", 2 * inter, hidden), ("down", hidden, inter))}
    lora = {}
    for name, columns, k in (("qkv", [128, 32, 32], hidden), ("o", [hidden], hidden), ("gate_up", [inter, inter], hidden), ("down", [hidden], inter)):
        a, b = _adapters(g, slots, rank, k, columns, dtype)
        lora[name] = dict(lora_a=[v.cuda() for v in a], lora_b=[v.cuda() for v in b])
    norms = [(1 + 0.1 * torch.randn(hidden, generator=g)).to(dtype).cuda() for _ in range(3)]

    def step(x, residual, of):
        rows, s = add_rms_norm(x, norms[0], residual=residual, quantize=True)
        qkv = quantized_linear(rows, weights["qkv"], token_to_slot=of, **lora["qkv"])
        y = quantized_linear(quantize_rows(qkv[:, :hidden]), weights["o"], token_to_slot=of, **lora["o"])
        rows, s = add_rms_norm(y, norms[1], residual=s, quantize=True, sum_out=s)
        rows = silu_mul(quantized_linear(rows, weights["gate_up"], token_to_slot=of, **lora["gate_up"]), quantize=True)
        y = quantized_linear(rows, weights["down"], token_to_slot=of, **lora["down"])
        return add_rms_norm(y, norms[2], residual=s)

    x, residual = (torch.zeros(t, hidden, dtype=dtype, device="cuda") for _ in range(2))
    of = torch.zeros(t, dtype=torch.int32, device="cuda")
    step(x, residual, of)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, residual, of)
    for replay in range(4):
        new = [torch.randn(t, hidden, generator=g).to(dtype).cuda() for _ in range(2)]
        slots_now = torch.randint(-1, slots, (t,), generator=g, dtype=torch.int32)
        if replay == 2:
            slots_now[:] = -1
        x.copy_(new[0]), residual.copy_(new[1]), of.copy_(slots_now.cuda())
        graph.replay()
        torch.cuda.synchronize()
        want = step(new[0], new[1], slots_now.cuda())
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
