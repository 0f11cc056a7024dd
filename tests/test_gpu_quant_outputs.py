"""Tensors that the 8-bit ops write must not wait for a gradient: also where the usual call, in C++, would serve the rest."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_sum_in_place_of_a_tensor_that_waits_for_a_gradient_is_refused():
    from nanovllm_voxcpm_amd.quant_ops import QuantizedRows, add_rms_norm, quantize_rows, quantized_linear

    held = torch.randn(4, 64, device="cuda").requires_grad_()
    before = held.detach().clone()
    for x, residual in ((held.detach(), torch.randn(4, 64, device="cuda")), (torch.randn(4, 64, device="cuda"), held.detach())):
        with pytest.raises(RuntimeError, match="no backward"):
            add_rms_norm(x, torch.ones(64, device="cuda"), residual=residual, sum_out=held)
        assert torch.equal(held, before)
    rows = quantize_rows(torch.randn(4, 64, device="cuda"))
    out = torch.zeros(4, 4, device="cuda", dtype=torch.bfloat16).requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        quantized_linear(rows, QuantizedRows(*rows), out=out)
    with torch.no_grad():
        quantized_linear(rows, QuantizedRows(*rows), out=out)
        total = add_rms_norm(held, torch.ones(64, device="cuda"), residual=held, sum_out=held)[1]
    assert total is held and torch.equal(held, before + before) and out.abs().max() > 0
