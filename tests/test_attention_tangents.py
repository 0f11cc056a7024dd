"""The attention calls have no derivative of either kind: a tensor that carries a tangent is refused, not stripped of it (host side)."""

import pytest
import torch
from torch.autograd import forward_ad

from nanovllm_voxcpm_amd.attention_ops import decode_attention, prompt_attention, rotate_qk

ROTATE = dict(q=(5, 4, 64), k=(5, 2, 64), cos_sin=(9, 64), q_weight=(64,), k_weight=(64,), v=(5, 2, 64))
DECODE = dict(q=(3, 4, 64), k_cache=(5, 16, 2, 64), v_cache=(5, 16, 2, 64))
PROMPT = dict(q=(7, 4, 64), k=(7, 2, 64), v=(7, 2, 64))


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32)


CALLS = {
    "rotate": (rotate_qk, ROTATE, dict(positions=_ints(*range(5)), k_cache=torch.zeros(2, 16, 2, 64), v_cache=torch.zeros(2, 16, 2, 64), slot_mapping=_ints(*range(5)))),
    "decode": (decode_attention, DECODE, dict(block_tables=torch.zeros(3, 2, dtype=torch.int32), context_lens=_ints(1, 2, 3))),
    "prompt": (prompt_attention, PROMPT, dict(cu_seqlens=_ints(0, 3, 7))),
}


@pytest.mark.parametrize("call,name", [(c, n) for c, (_, tensors, _) in CALLS.items() for n in tensors])
def test_a_tensor_with_a_tangent_or_a_gradient_to_come_is_refused(call, name):
    fn, tensors, rest = CALLS[call]
    plain = {n: torch.zeros(shape) for n, shape in tensors.items()}
    with forward_ad.dual_level():
        dual = {**plain, name: forward_ad.make_dual(plain[name], torch.ones_like(plain[name]))}
        with pytest.raises(RuntimeError, match="no backward"):
            fn(**dual, **rest)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no backward"):  # (no_grad is of the backward direction)
            fn(**dual, **rest)
        with pytest.raises(RuntimeError, match="GPU"):
            fn(**plain, **rest)
    with pytest.raises(RuntimeError, match="no backward"):
        fn(**{**plain, name: plain[name].clone().requires_grad_()}, **rest)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        fn(**{**plain, name: plain[name].clone().requires_grad_()}, **rest)
