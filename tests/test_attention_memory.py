"""Which tensors of an attention call may share memory (host arithmetic on views; a call that passes its checks ends at the missing GPU)."""

import itertools
import random

import pytest
import torch

from nanovllm_voxcpm_amd import attention_ops
from nanovllm_voxcpm_amd.attention_ops import rotate_qk


def _call(**change):
    t, h, hk, d = 5, 4, 2, 64
    return {**dict(q=torch.zeros(t, h, d), k=torch.zeros(t, hk, d), v=torch.zeros(t, hk, d), positions=torch.zeros(t, dtype=torch.int32), cos_sin=torch.zeros(9, d),
                   k_cache=torch.zeros(3, 16, hk, d), v_cache=torch.zeros(3, 16, hk, d), slot_mapping=torch.arange(t)), **change}


def _ends(text, **change):
    with pytest.raises(ValueError if text else RuntimeError, match=text or "GPU"):
        rotate_qk(**_call(**change))


def test_an_output_on_a_cache_is_refused():
    pages = torch.zeros(3, 16, 2, 64)
    for cache in ("k_cache", "v_cache"):
        _ends(f"k_out overlaps {cache}", k_out=pages[1, 3:8], **{cache: pages})
        _ends(f"q_out overlaps {cache}", q_out=pages.view(-1, 4, 64)[7:12], **{cache: pages})


def test_an_output_beside_a_cache_in_one_allocation_is_not():
    room = torch.zeros(3, 16, 6, 64)
    _ends(None, k_cache=room[:, :, :2], v_cache=room[:, :, 2:4], k_out=room[1, 3:8, 4:])
    _ends("k_out overlaps v_cache", k_cache=room[:, :, :2], v_cache=room[:, :, 2:4], k_out=room[1, 3:8, 3:5])
    flat = torch.zeros(3 * 16 * 2 * 64 + 5 * 4 * 64)
    _ends(None, k_cache=flat[: 3 * 16 * 2 * 64].view(3, 16, 2, 64), q_out=flat[3 * 16 * 2 * 64 :].view(5, 4, 64))


def _places(t):
    size = t.element_size()
    return {t.data_ptr() + size * sum(i * s for i, s in zip(index, t.stride())) + b
            for index in itertools.product(*(range(n) for n in t.shape)) for b in range(size)}


def test_overlap_against_all_places():
    pick, seen = random.Random(3), {True: 0, False: 0}
    memory = torch.zeros(400, dtype=torch.float16)
    for _ in range(3000):
        views = []
        for dims in (3, pick.choice([3, 4])):
            shape = [pick.randint(1, 4) for _ in range(dims)]
            stride = [pick.choice([1, 2, 3, 4, 6, 8, 12, 16, 24]) for _ in range(dims)]
            reach = sum((n - 1) * s for n, s in zip(shape, stride))
            views.append(torch.as_strided(memory, shape, stride, pick.randint(0, 399 - reach)))
        meet = bool(_places(views[0]) & _places(views[1]))
        seen[meet] += 1
        assert attention_ops._overlap(*views) == meet, [(v.shape, v.stride(), v.storage_offset()) for v in views]
    assert min(seen.values()) > 300


def test_which_caches_lie_on_one_another():
    pages, both, side = torch.zeros(4, 16, 2, 64), torch.zeros(3, 2, 16, 2, 64), torch.zeros(3, 16, 2, 128)
    for k_cache, v_cache, meet in ((pages, pages, True), (pages[:3], pages[1:], True), (both[:, 0], both[:, 1], False), (side[..., :64], side[..., 64:], False),
                                   (side[..., :64], side[..., 63:127], True), (pages[:2], pages[2:], False)):
        assert attention_ops._overlap(k_cache, v_cache) == meet
        _ends(None, k_cache=k_cache, v_cache=v_cache)  # (on the host nothing is written)


def test_written_tensors_whose_rows_lie_on_one_another_are_refused():
    row = torch.zeros(4000)
    _ends("q_out share memory", q_out=row.as_strided((5, 4, 64), (128, 64, 1)))
    _ends("k_out share memory", k_out=row.as_strided((5, 2, 64), (64, 64, 1)))
    _ends("rows or heads of k_cache", k_cache=row.as_strided((3, 16, 2, 64), (64, 64, 64, 1)))
    _ends("rows or heads of v_cache", v_cache=torch.zeros(7000).as_strided((3, 16, 2, 64), (2047, 128, 64, 1)))
    _ends(None, q_out=torch.zeros(4, 5, 64).transpose(0, 1))  # (heads outside rows)
    _ends(None, k_cache=torch.zeros(3, 2, 16, 64).transpose(1, 2), v_cache=torch.zeros(16, 3, 2, 64).transpose(0, 1))


def test_own_overlap_against_all_places():
    pick, seen = random.Random(4), {True: 0, False: 0}
    memory = torch.zeros(400, dtype=torch.float16)
    for _ in range(2000):
        shape = [pick.randint(1, 4) for _ in range(4)]
        t = torch.as_strided(memory, shape, [pick.choice([1, 2, 3, 4, 5, 8, 12, 16, 24, 30]) for _ in range(4)])
        on_itself = len(_places(t)) < t.numel() * t.element_size()
        seen[on_itself] += 1
        if on_itself:
            with pytest.raises(ValueError, match="share memory"):
                attention_ops._rows_apart(t, "t")
        else:
            attention_ops._rows_apart(t, "t")
    assert min(seen.values()) > 300
