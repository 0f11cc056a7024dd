"""Refusals of the 8-bit ops, the structs of their C entries, and the oracle against plain torch; no GPU."""

import ctypes as C

import pytest
import torch

from nanovllm_voxcpm_amd import _hip
from nanovllm_voxcpm_amd.quant_ops import QuantizedRows, add_rms_norm, quantize_rows, quantized_linear, silu_mul
from oracle import quant as oracle


def _eight(n, k):
    return QuantizedRows(torch.zeros(n, k, dtype=torch.float8_e4m3fn), torch.ones(n))


def test_rows_are_refused():
    x, w = torch.randn(4, 32), torch.ones(32)
    for bad in (torch.randn(32), torch.randn(2, 2, 32), torch.randn(4, 64)[:, ::2], torch.empty(4, 0), torch.zeros(4, 32, dtype=torch.int32), torch.zeros(4, 32, dtype=torch.float64)):
        with pytest.raises(ValueError):
            quantize_rows(bad)
        with pytest.raises(ValueError):
            add_rms_norm(bad, w)
        with pytest.raises(ValueError):
            silu_mul(bad)
    for weight in (torch.ones(31), torch.ones(1, 32), torch.ones(64)[::2], torch.ones(32, dtype=torch.float16)):
        with pytest.raises(ValueError):
            add_rms_norm(x, weight)
    for residual in (torch.randn(3, 32), torch.randn(4, 31), torch.randn(4, 32).half(), torch.randn(4, 64)[:, ::2]):
        with pytest.raises(ValueError):
            add_rms_norm(x, w, residual=residual)
    with pytest.raises(ValueError, match="eps"):
        add_rms_norm(x, w, eps=-1e-6)
    with pytest.raises(ValueError, match="eps"):
        add_rms_norm(x, w, eps=float("nan"))
    with pytest.raises(ValueError, match="no residual"):
        add_rms_norm(x, w, sum_out=torch.empty(4, 32))
    with pytest.raises(ValueError, match="as wide as"):
        silu_mul(torch.randn(4, 33))
    buffer = torch.randn(4, 40)
    for sum_out in (torch.empty(4, 31), torch.empty(4, 32).half(), buffer[:, 1:33], torch.empty(1, 32).expand(4, 32)):
        with pytest.raises(ValueError):
            add_rms_norm(x, w, residual=buffer[:, :32], sum_out=sum_out)
    with pytest.raises(ValueError, match="overlaps weight"):
        add_rms_norm(x[:1], buffer[0, :32], residual=x[1:2], sum_out=buffer[:1, 8:40])


def test_rows_on_the_host_have_no_fallback():
    for call in (lambda: quantize_rows(torch.randn(4, 32)), lambda: add_rms_norm(torch.randn(4, 32), torch.ones(32)), lambda: silu_mul(torch.randn(4, 32)),
                 lambda: quantized_linear(_eight(3, 32), _eight(5, 32))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_linears_are_refused():
    rows, weight = _eight(3, 32), _eight(8, 32)
    for bad in (QuantizedRows(torch.zeros(3, 32), torch.ones(3)), QuantizedRows(rows.values[0], torch.ones(3)), _eight(3, 24), _eight(3, 0), QuantizedRows(rows.values, torch.ones(2)),
                QuantizedRows(rows.values, torch.ones(3).double()), QuantizedRows(rows.values, torch.ones(6)[::2]), QuantizedRows(_eight(3, 64).values[:, 8:40], torch.ones(3)),
                QuantizedRows(_eight(3, 40).values[:, :32], torch.ones(3)), QuantizedRows(_eight(3, 64).values[:, ::2], torch.ones(3))):
        with pytest.raises(ValueError):
            quantized_linear(bad, weight)
        if bad.values.dim() == 2:
            with pytest.raises(ValueError):
                quantized_linear(rows, bad)
    with pytest.raises(ValueError, match="takes 48"):
        quantized_linear(rows, _eight(8, 48))
    with pytest.raises(ValueError, match="dtype"):
        quantized_linear(rows, weight, dtype=torch.float32)
    for bias in (torch.zeros(8), torch.zeros(7).bfloat16(), torch.zeros(16).bfloat16()[::2]):
        with pytest.raises(ValueError, match="bias"):
            quantized_linear(rows, weight, bias=bias)
    for out in (torch.empty(3, 7).bfloat16(), torch.empty(3, 8), torch.empty(8, 3).bfloat16().t(), torch.empty(1, 8).bfloat16().expand(3, 8)):
        with pytest.raises(ValueError):
            quantized_linear(rows, weight, out=out)
    with pytest.raises(ValueError, match="overlaps"):
        bias = torch.zeros(64).bfloat16()
        quantized_linear(rows, weight, bias=bias[:8], out=bias[4:28].view(3, 8))


def test_adapters_are_refused():
    rows, weight = _eight(3, 32), _eight(8, 32)
    of = torch.zeros(3, dtype=torch.int32)
    a, b = [torch.zeros(2, 4, 32).bfloat16()], [torch.zeros(2, 8, 4).bfloat16()]
    good = dict(lora_a=a, lora_b=b, token_to_slot=of)
    for name in good:
        with pytest.raises(ValueError, match="together"):
            quantized_linear(rows, weight, **{n: v for n, v in good.items() if n != name})
    with pytest.raises(ValueError, match="lora_columns"):
        quantized_linear(rows, weight, lora_columns=[0])
    for change in (dict(lora_a=[], lora_b=[]), dict(lora_a=a * 2), dict(lora_a=a * 9, lora_b=[torch.zeros(2, 1, 4).bfloat16()] * 9), dict(lora_a=[a[0].float()]), dict(lora_b=[b[0].half()]),
                   dict(lora_a=[torch.zeros(2, 4, 48).bfloat16()]), dict(lora_b=[torch.zeros(2, 9, 4).bfloat16()]), dict(lora_b=[torch.zeros(3, 8, 4).bfloat16()]),
                   dict(lora_b=[torch.zeros(2, 8, 5).bfloat16()]), dict(lora_a=[torch.zeros(2, 0, 32).bfloat16()], lora_b=[torch.zeros(2, 8, 0).bfloat16()]),
                   dict(lora_a=[torch.zeros(2, 257, 32).bfloat16()], lora_b=[torch.zeros(2, 8, 257).bfloat16()]), dict(lora_a=[a[0].transpose(0, 1).contiguous().transpose(0, 1)]),
                   dict(lora_a=[torch.zeros(1025, 1, 32).bfloat16()], lora_b=[torch.zeros(1025, 8, 1).bfloat16()]), dict(lora_columns=[1]), dict(lora_columns=[-1]), dict(lora_columns=[0, 4]),
                   dict(lora_a=a * 2, lora_b=[torch.zeros(2, 4, 4).bfloat16()] * 2, lora_columns=[0, 3]), dict(token_to_slot=of.long()), dict(token_to_slot=of[:2]),
                   dict(token_to_slot=torch.zeros(6, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError):
            quantized_linear(rows, weight, **{**good, **change})


def test_tensors_that_wait_for_a_gradient_are_refused():
    x = torch.randn(4, 32, requires_grad=True)
    for call in (lambda: quantize_rows(x), lambda: add_rms_norm(x, torch.ones(32)), lambda: add_rms_norm(torch.randn(4, 32), torch.ones(32, requires_grad=True)), lambda: silu_mul(x),
                 lambda: quantized_linear(_eight(3, 32), _eight(8, 32), bias=torch.zeros(8, dtype=torch.bfloat16, requires_grad=True))):
        with pytest.raises(RuntimeError, match="no backward"):
            call()


def _rows_args(**kw):
    args = _hip.MloraRowsArgs()
    for name, value in dict(x=16, out=16, weight=16, scales=16, num_rows=2, width=32, dtype=_hip.DTYPE_BF16, **kw).items():
        setattr(args, name, value)
    return args


def _project_args(**kw):
    args = _hip.MloraProjectArgs()
    values = dict(x=16, w=16, x_scales=16, w_scales=16, y=16, x_row=32, w_row=32, y_row=8, num_rows=2, k=32, n=8, dtype=_hip.DTYPE_BF16, num_slices=1, r=4, num_slots=2,
                  token_to_slot=16, workspace=16, workspace_bytes=1 << 20)
    for name, value in {**values, **kw}.items():
        if name != "slices":
            setattr(args, name, value)
    for i, s in enumerate(kw.get("slices", [(16, 16, 8, 0)])):
        args.slices[i] = _hip.MloraSlice(*s)
    return args


def test_the_c_entries_refuse_before_they_launch():
    lib = _hip.load()
    for entry in (lib.mlora_add_rms_norm, lib.mlora_silu_mul, lib.mlora_quantize_rows):
        assert entry(None) == -1
        for bad in (dict(num_rows=-1), dict(width=-1), dict(width=0), dict(dtype=7), dict(x=None), dict(out=None), dict(num_rows=1 << 24), dict(num_rows=1 << 22, width=8193), dict(width=1 << 30)):
            args = _rows_args()
            for name, value in bad.items():
                setattr(args, name, value)
            assert entry(C.byref(args)) < 0, bad
        args = _rows_args()
        args.num_rows = 0
        assert entry(C.byref(args)) == 0
    args = _rows_args(residual=16)
    for entry in (lib.mlora_add_rms_norm, lib.mlora_silu_mul, lib.mlora_quantize_rows):
        assert entry(C.byref(args)) < 0  # (a residual without a place for the sum, or where there is none)
    args = _rows_args()
    args.weight = None
    assert lib.mlora_add_rms_norm(C.byref(args)) < 0
    args.scales = None
    assert lib.mlora_quantize_rows(C.byref(args)) < 0
    assert lib.mlora_project(None) == -1
    for bad in (dict(num_rows=-1), dict(k=-16), dict(n=-1), dict(k=24), dict(k=0), dict(dtype=_hip.DTYPE_F32), dict(x=None), dict(w=None), dict(y=None), dict(x_scales=None), dict(w_scales=None),
                dict(x=24), dict(w=8), dict(x_row=40), dict(w_row=8), dict(num_slices=9), dict(num_slices=-1), dict(r=0), dict(r=257), dict(num_slots=0), dict(num_slots=1025),
                dict(token_to_slot=None), dict(workspace=None), dict(workspace=24), dict(workspace_bytes=31), dict(slices=[(None, 16, 8, 0)]), dict(slices=[(16, None, 8, 0)]),
                dict(slices=[(24, 16, 8, 0)]), dict(slices=[(16, 16, 9, 0)]), dict(slices=[(16, 16, 0, 0)]), dict(slices=[(16, 16, 4, -1)]), dict(slices=[(16, 16, 4, 5)]),
                dict(num_slices=2, slices=[(16, 16, 4, 0), (16, 16, 4, 3)]), dict(num_rows=(1 << 20) + 1), dict(n=(1 << 22) + 1), dict(k=(1 << 22) + 16)):
        assert lib.mlora_project(C.byref(_project_args(**bad))) < 0, bad
    for nothing in (dict(num_rows=0), dict(n=0)):
        assert lib.mlora_project(C.byref(_project_args(**nothing))) == 0
    assert lib.mlora_project_workspace_bytes(C.byref(_project_args())) >= 2 * 8 * 4
    assert lib.mlora_project_workspace_bytes(C.byref(_project_args(num_slices=0))) == 0
    assert lib.mlora_project_workspace_bytes(None) == 0


def test_the_oracle_is_torch_in_64_bits():
    g = torch.Generator().manual_seed(1)
    x, residual = torch.randn(5, 48, generator=g).double(), torch.randn(5, 48, generator=g).double()
    weight = torch.randn(48, generator=g).double()
    total, y, _ = oracle.add_rms_norm(x.float(), weight.float(), residual.float(), 1e-5)
    want = torch.nn.functional.rms_norm(total.double(), (48,), weight.float().double(), 1e-5)
    assert torch.allclose(y, want, rtol=1e-13)
    y, _ = oracle.silu_mul(torch.cat([x, residual], dim=1))
    assert torch.allclose(y, torch.nn.functional.silu(x) * residual, rtol=1e-13)
    scales, _, values, _ = oracle.eight_bits(x, 0.0)
    assert torch.allclose(values * scales[:, None], x) and torch.allclose(values.abs().amax(-1), torch.full((5,), 448.0).double())
    a, b = [torch.randn(3, 4, 48, generator=g)], [torch.randn(3, 6, 4, generator=g)]
    w = torch.randn(10, 48, generator=g)
    y, bound = oracle.linear(x, torch.ones(5), w, torch.ones(10), bias=torch.ones(10), a=a, b=b, columns=[2], slots=torch.tensor([0, -1, 2, 3, 1]))
    want = x @ w.double().T + 1
    for t, s in ((0, 0), (2, 2), (4, 1)):
        want[t, 2:8] += b[0][s].double() @ (a[0][s].double() @ x[t])
    assert torch.allclose(y, want, rtol=1e-12) and (bound > 0).all()


def test_base_weights_that_stay_as_they_are():
    from nanovllm_voxcpm_amd.layers.lora import LoRALinear

    for layer, error, match in ((LoRALinear(32, 8), ValueError, "fp16 and bf16"), (LoRALinear(40, 8).half(), ValueError, "multiple of 16"), (LoRALinear(32, 8).half(), RuntimeError, "GPU")):
        with pytest.raises(error, match=match):
            layer.quantize_base_()
        assert not layer.base_in_8_bits and layer.weight is not None and "weight_values" not in layer.state_dict()


@torch.no_grad()
def test_a_sharded_row_parallel_linear_adds_its_bias_once(monkeypatch):
    """The ops stand in by their definitions: on the first rank with the bias, on the others without."""
    from nanovllm_voxcpm_amd.layers import lora as layers

    def quantize(x):
        scales, _, values, _ = oracle.eight_bits(x.double(), 0.0)
        return QuantizedRows(values.to(torch.float8_e4m3fn), scales.float())

    def linear(rows, weight, *, bias=None, dtype=None, **adapters):
        assert not adapters
        return oracle.linear(rows.values.float(), rows.scales, weight.values.float(), weight.scales, bias, dtype=dtype)[0].to(dtype)

    monkeypatch.setattr(layers, "quantize_rows", quantize)
    monkeypatch.setattr(layers, "quantized_linear", linear)
    monkeypatch.setattr(layers.LoRARowParallelLinear, "check_base_for_8_bits", lambda self: None)
    x, sums = torch.randn(3, 32).half(), []
    for rank in (0, 1):
        layer = layers.LoRARowParallelLinear(32, 8, bias=True).half()
        layer.weight.copy_(torch.ones(8, 32))
        layer.bias.copy_(torch.full((8,), 64.0))
        layer.tp_size, layer.tp_rank = 2, rank
        layer.quantize_base_()
        sums.append(layer(x))
    assert ((sums[0] - sums[1]).float() - 64).abs().max() <= 0.07  # (fp16 up to 128 and below 64: two halves of steps of 2^-4)


def test_sizes_beyond_32_bits_are_refused():
    wide, many = torch.empty(1, 2**31 + 512, dtype=torch.bfloat16, device="meta"), torch.empty(2**31 + 512, 16, dtype=torch.bfloat16, device="meta")
    for x in (wide, many):
        for call in (lambda: quantize_rows(x), lambda: silu_mul(x), lambda: add_rms_norm(x, torch.ones(1))):
            with pytest.raises(ValueError, match="larger than"):
                call()
        eight = QuantizedRows(torch.empty(x.shape, dtype=torch.float8_e4m3fn, device="meta"), torch.empty(x.size(0), device="meta"))
        for rows, weight in ((eight, _eight(5, 16)), (_eight(5, 16), eight)):
            with pytest.raises(ValueError, match="larger than"):
                quantized_linear(rows, weight)
