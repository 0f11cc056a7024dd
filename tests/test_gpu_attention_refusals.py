"""What the attention calls refuse or take on the GPU, where the C++ host path looks first."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _rotation(t=21, heads=4, kv_heads=2, dim=64, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(t, h, dim, generator=g).to(dtype).cuda() for h in (heads, kv_heads, kv_heads))
    table = torch.randn(50, dim, generator=g).cuda()
    return dict(q=q, k=k, v=v, positions=torch.arange(t, device="cuda"), cos_sin=table, slot_mapping=torch.arange(t, device="cuda") * 2)


def test_caches_between_one_another_are_written_and_on_one_another_refused():
    from nanovllm_voxcpm_amd.attention_ops import rotate_qk

    apart = [torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    want, _ = rotate_qk(**_rotation(), k_cache=apart[0], v_cache=apart[1])
    both = torch.zeros(3, 2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    side = torch.zeros(3, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
    heads = torch.zeros(2, 3, 2, 16, 64, dtype=torch.bfloat16, device="cuda").transpose(2, 3)
    for k_cache, v_cache in ((both[:, 0], both[:, 1]), (side[..., 64:], side[..., :64]), (heads[0], heads[1])):
        got, _ = rotate_qk(**_rotation(), k_cache=k_cache, v_cache=v_cache)
        assert torch.equal(got, want) and torch.equal(k_cache, apart[0]) and torch.equal(v_cache, apart[1])
    with pytest.raises(ValueError, match="k_cache overlaps v_cache"):
        rotate_qk(**_rotation(), k_cache=apart[0], v_cache=apart[0])
    room = torch.zeros(20000, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="rows or heads of v_cache"):
        rotate_qk(**_rotation(), k_cache=apart[0], v_cache=room.as_strided((3, 16, 2, 64), (2048, 64, 64, 1)))


def test_a_tensor_with_a_tangent_is_refused():
    from torch.autograd import forward_ad

    from nanovllm_voxcpm_amd.attention_ops import decode_attention, prompt_attention, rotate_qk

    call = _rotation()
    q, k, v, table = call["q"], call["k"], call["v"], call["cos_sin"]
    starts = torch.tensor([0, q.size(0)], dtype=torch.int32, device="cuda")
    cache, blocks = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(21, 1, dtype=torch.int32, device="cuda")
    with forward_ad.dual_level():
        for name in ("q", "k", "v"):
            with pytest.raises(RuntimeError, match="tangent"):
                rotate_qk(**{**call, name: forward_ad.make_dual(call[name], torch.ones_like(call[name]))}, k_cache=cache, v_cache=torch.zeros_like(cache))
            tensors = dict(q=q, k=k, v=v)
            tensors[name] = forward_ad.make_dual(tensors[name], torch.ones_like(tensors[name]))
            with pytest.raises(RuntimeError, match="tangent"):
                prompt_attention(**tensors, cu_seqlens=starts)
        with pytest.raises(RuntimeError, match="tangent"):
            decode_attention(forward_ad.make_dual(q, torch.ones_like(q)), cache, cache, blocks, blocks[:, 0])
        prompt_attention(q, k, v, starts)
        with torch.inference_mode():
            prompt_attention(forward_ad.make_dual(q, torch.ones_like(q)), k, v, starts)
    with pytest.raises(RuntimeError, match="no backward"):
        rotate_qk(q, k, call["positions"], table.clone().requires_grad_())
