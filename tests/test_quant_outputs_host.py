"""Tensors that the 8-bit ops write must not wait for a gradient, which would not know of it; no GPU."""

import pytest
import torch
from torch.autograd import forward_ad

from nanovllm_voxcpm_amd.quant_ops import QuantizedRows, add_rms_norm, quantized_linear


def _calls(kind):
    make = {"leaf": lambda *shape, dtype: torch.empty(*shape, dtype=dtype, requires_grad=True), "result": lambda *shape, dtype: torch.empty(*shape, dtype=dtype, requires_grad=True) * 1}[kind]
    eight = lambda n: QuantizedRows(torch.zeros(n, 32, dtype=torch.float8_e4m3fn), torch.ones(n))  # noqa: E731
    return [lambda: add_rms_norm(torch.randn(4, 32), torch.ones(32), residual=torch.randn(4, 32), sum_out=make(4, 32, dtype=torch.float32)),
            lambda: quantized_linear(eight(3), eight(8), out=make(3, 8, dtype=torch.bfloat16))]


@pytest.mark.parametrize("kind", ["leaf", "result"])
def test_outputs_that_wait_for_a_gradient_are_refused(kind):
    for call in _calls(kind):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):  # (nothing waits there)
            call()


def test_outputs_that_carry_a_tangent_are_refused():
    with forward_ad.dual_level():
        to = forward_ad.make_dual(torch.empty(4, 32), torch.ones(4, 32))
        with pytest.raises(RuntimeError, match="tangent"):
            add_rms_norm(torch.randn(4, 32), torch.ones(32), residual=torch.randn(4, 32), sum_out=to)
