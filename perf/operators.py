"""The attention block between the LoRA linears, as measurable cases.

A decoder layer's q|k|v linear hands over one packed row per token and its o linear takes one row of attention outputs.
Between them lie three operators:

* ``rotate`` - the RMS norms of every query and key head (where the model has them), the rotation by position, and the
  new keys and values into the pages of the cache.
* ``decode`` - one new token per running sequence over a paged cache.
* ``prompt`` - whole prompts, or chunks of prompts behind cached tokens, with or without a sliding window and a few first
  tokens that stay visible; also short batches in which every token sees every other.

Head layouts are the synthetic decoder's (16 query heads, 2 key-value heads of 64) and a wider one (32, 8 of 128); batches
are those of the decode, prefill and chunked-prefill benchmarks (64 and 201 streams, 16 prompts of 9392 tokens, chunks of
2048 tokens), contexts reach from one token to 131072.
"""

from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed() -> list[dict]:
    small, wide = dict(heads=16, kv_heads=2, dim=64), dict(heads=32, kv_heads=8, dim=128)
    return [
        # one running request: launches are all there is
        dict(name="rotate_1_token", kind="rotate", tokens=1, **small, dtype="bf16", norms=False, rotary=64, interleaved=False,
             page=256, unstored=0, reach=4096),
        # the prefill benchmark's 16 prompts in one batch, heads normed
        dict(name="rotate_9392_tokens", kind="rotate", tokens=9392, **small, dtype="bf16", norms=True, rotary=64, interleaved=False,
             page=256, unstored=0, reach=1024),
        # a wider model that rotates half of every head in neighbouring pairs, far positions, a batch padded by 189 rows
        dict(name="rotate_8381_tokens_wide", kind="rotate", tokens=8381, **wide, dtype="fp16", norms=True, rotary=64, interleaved=True,
             page=64, unstored=189, reach=131072),
        # one request in the middle of its answer
        dict(name="decode_1_stream", kind="decode", sequences=1, empty=0, longest=900, **small, dtype="bf16", page=256, window=0, sinks=0),
        # the end-to-end benchmark's decode batch
        dict(name="decode_64_streams", kind="decode", sequences=64, empty=0, longest=2048, **small, dtype="bf16", page=256, window=0, sinks=0),
        # a window of 1024 and four first tokens; the batch is padded to its graph's size by seven empty rows
        dict(name="decode_208_streams_window", kind="decode", sequences=208, empty=7, longest=8192, **small, dtype="fp16", page=16,
             window=1024, sinks=4),
        # a few very long contexts of a wider model: the work lies along the cache
        dict(name="decode_3_streams_long", kind="decode", sequences=3, empty=0, longest=131072, **wide, dtype="bf16", page=64, window=0, sinks=0),
        # one short prompt by itself
        dict(name="prompt_37_tokens", kind="prompt", sequences=1, tokens=37, cached=0, **small, dtype="bf16", page=0, causal=True,
             window=0, sinks=0),
        # the prefill benchmark: 16 prompts packed one behind the other
        dict(name="prompt_9392_tokens", kind="prompt", sequences=16, tokens=9392, cached=0, **small, dtype="bf16", page=0, causal=True,
             window=0, sinks=0),
        # chunked prefill: two chunks of 2048 tokens behind what their prompts have in the cache already
        dict(name="prompt_2_chunks_cached", kind="prompt", sequences=2, tokens=4096, cached=28001, **small, dtype="fp16", page=256,
             causal=True, window=0, sinks=0),
        # a long prompt of a wider model with a window of 2048 and four first tokens
        dict(name="prompt_16384_tokens_window", kind="prompt", sequences=1, tokens=16384, cached=0, **wide, dtype="bf16", page=0, causal=True,
             window=2048, sinks=4),
        # the estimator's batches: short sequences in which every token sees every other, in fp32
        dict(name="prompt_64_estimators_fp32", kind="prompt", sequences=64, tokens=833, cached=0, **small, dtype="fp32", page=0,
             causal=False, window=0, sinks=0),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random) -> dict:
    most = [work(c) for c in listed()]
    while True:
        case = _draw(rng)
        cost = work(case)
        if cost["bytes"] <= max(w["bytes"] for w in most) and cost["flops"] <= max(w["flops"] for w in most) and _held(case) <= 2 << 30:
            return case


def _draw(rng: random.Random) -> dict:
    kind = rng.choice(["rotate", "decode", "prompt"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 7, 8, 16) if g * kv_heads <= 32])
    shape = dict(heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 64, 128]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    page = rng.choice([16, 64, 256])
    window, sinks = rng.choice([(0, 0), (0, 0), (_log_int(rng, 64, 4096), rng.choice([0, 1, 4, 100]))])
    if kind == "rotate":
        tokens = _log_int(rng, 1, 9392)
        return dict(kind=kind, tokens=tokens, **shape, norms=rng.random() < 0.5, rotary=rng.choice([shape["dim"], shape["dim"] // 2]),
                    interleaved=rng.random() < 0.3, page=page, unstored=rng.randint(0, tokens // 8), reach=_log_int(rng, 64, 131072))
    if kind == "decode":
        sequences = _log_int(rng, 1, 256)
        return dict(kind=kind, sequences=sequences, empty=rng.randint(0, sequences // 8), longest=_log_int(rng, 1, 131072), **shape, page=page,
                    window=window, sinks=sinks)
    tokens = _log_int(rng, 1, 16384)
    sequences = _log_int(rng, 1, min(64, tokens))
    causal = rng.random() < 0.8
    paged = causal and rng.random() < 0.5
    return dict(kind=kind, sequences=sequences, tokens=tokens, cached=_log_int(rng, 1, 65536) if paged else 0, **shape, page=page if paged else 0,
                causal=causal, window=window if causal else 0, sinks=sinks if causal else 0)


# ---- batches: the lengths belong to the case, values and pages to the seed ---------------------------


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(new tokens, visible tokens) of every sequence."""
    pick = random.Random(case["sequences"] * 1000003 + case.get("tokens", 0) + case.get("longest", 0))
    n = case["sequences"]
    if case["kind"] == "decode":
        contexts = [max(1, round(case["longest"] * pick.uniform(0.05, 1.0))) for _ in range(n)]
        contexts[pick.randrange(n)] = case["longest"]
        for i in pick.sample(range(n), case["empty"]):
            contexts[i] = 0
        return [1] * n, contexts
    share = [pick.uniform(0.12, 1.88) for _ in range(n)]
    left = case["tokens"] - n
    new = [1 + int(left * s / sum(share)) for s in share]
    new[-1] += case["tokens"] - sum(new)
    cached = [round(case["cached"] * pick.uniform(0.5, 1.5)) for _ in range(n)]
    return new, [a + b for a, b in zip(new, cached)]


def _visible(case: dict, new: int, total: int) -> tuple[int, int]:
    """(query-key pairs, keys that any query sees) of one sequence."""
    at = np.arange(total - new, total, dtype=np.int64)  # the queries' positions
    if not case.get("causal", True):
        return new * total, total
    low = np.maximum(at + 1 - case["window"], 0) if case["window"] else np.zeros_like(at)
    first = np.minimum(low, case["sinks"])
    return int((first + at + 1 - low).sum()), int(first[-1] + total - low[0]) if low[0] > first[-1] else total


def _held(case: dict) -> int:
    """Bytes of the keys and values that the state holds (a window hides most of a long cache)."""
    if case["kind"] == "rotate":
        return 0
    return 2 * sum(_lengths(case)[1]) * case["kv_heads"] * case["dim"] * SIZES[case["dtype"]]


def work(case: dict) -> dict:
    e, d, h, hk = SIZES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "rotate":
        t, r = case["tokens"], case["rotary"]
        stored = t - case["unstored"]
        cells = t * (h + hk) * d + stored * hk * d + t * h * d + stored * 2 * hk * d  # q, k and the stored rows' v in; q and the stored rows out
        return {"bytes": cells * e + 4 * min(t, case["reach"]) * r + 12 * t, "flops": t * (h + hk) * (3 * r + (4 * d if case["norms"] else 0))}
    new, totals = _lengths(case)
    pairs = keys = 0
    for n, total in zip(new, totals):
        if total:
            p, k = _visible(case, n, total)
            pairs, keys = pairs + p, keys + k
    blocks = 4 * keys // case["page"] if case["page"] else 0
    return {"bytes": 2 * sum(new) * h * d * e + 2 * keys * hk * d * e + blocks + 4 * len(new), "flops": 4 * pairs * h * d}


# ---- states ------------------------------------------------------------------------------------------


def _normal(gen: torch.Generator, *shape: int, dtype: torch.dtype, scale: float = 1.0) -> torch.Tensor:
    t = torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)
    return t if scale == 1.0 else t.mul_(scale)


def _tables(gen: torch.Generator, totals: list[int], page: int) -> tuple[torch.Tensor, int]:
    """A block table with the pages of every sequence, and how many pages the cache has: all that are used and some more."""
    counts = [-(-t // page) for t in totals]
    pool = sum(counts) + 3
    order = torch.randperm(pool, generator=gen, device=DEVICE).to(torch.int32).cpu().numpy()
    table = np.full((len(totals), max(1, max(counts))), -1, dtype=np.int32)
    at = 0
    for row, c in enumerate(counts):
        table[row, :c] = order[at:at + c]
        at += c
    return torch.from_numpy(table).to(DEVICE), pool


def _starts(lengths: list[int]) -> torch.Tensor:
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device=DEVICE)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 17)
    dtype, d, h, hk, page = DTYPES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"], case["page"]
    if case["kind"] == "rotate":
        t, half, reach = case["tokens"], case["rotary"] // 2, case["reach"]
        stored = t - case["unstored"]
        angles = torch.arange(reach, device=DEVICE, dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
        pool = -(-t // page) + 2
        slots = torch.randperm(pool * page, generator=gen, device=DEVICE)[:t].to(torch.int32)
        slots[stored:] = -1
        weights = [1.0 + _normal(gen, d, dtype=torch.float32, scale=0.1) for _ in range(2)] if case["norms"] else [None, None]
        return dict(case=case, qkv=_normal(gen, t, (h + 2 * hk) * d, dtype=dtype),
                    positions=torch.randint(0, reach, (t,), generator=gen, device=DEVICE, dtype=torch.int32),
                    cos_sin=torch.cat([angles.cos(), angles.sin()], dim=1).float(), slots=slots,
                    q_weight=None if weights[0] is None else weights[0].to(dtype), k_weight=None if weights[1] is None else weights[1].to(dtype),
                    k_cache=_normal(gen, pool, page, hk, d, dtype=dtype), v_cache=_normal(gen, pool, page, hk, d, dtype=dtype))
    new, totals = _lengths(case)
    state = dict(case=case, q=_normal(gen, sum(new), h, d, dtype=dtype, scale=1.5), new=new, totals=totals)
    if page:
        state["block_tables"], pool = _tables(gen, totals, page)
        state["k"], state["v"] = (_normal(gen, pool, page, hk, d, dtype=dtype) for _ in range(2))
        state["context_lens"] = torch.tensor(totals, dtype=torch.int32, device=DEVICE)
    else:
        state["k"], state["v"] = (_normal(gen, sum(totals), hk, d, dtype=dtype) for _ in range(2))
    if case["kind"] == "prompt":
        state["starts"] = _starts(new)
    return state


# ---- one pass ----------------------------------------------------------------------------------------


def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state: dict):
    folder = os.path.join(os.getcwd(), "nanovllm-voxcpm_amd")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    from nanovllm_voxcpm_amd.attention_ops import decode_attention, prompt_attention, rotate_qk

    case = state["case"]
    if case["kind"] == "rotate":
        t, d, h, hk = case["tokens"], case["dim"], case["heads"], case["kv_heads"]
        q, k, v = state["qkv"].split([h * d, hk * d, hk * d], dim=1)
        q, _ = rotate_qk(q.view(t, h, d), k.view(t, hk, d), state["positions"], state["cos_sin"], q_weight=state["q_weight"],
                         k_weight=state["k_weight"], interleaved=case["interleaved"], v=v.view(t, hk, d), k_cache=state["k_cache"],
                         v_cache=state["v_cache"], slot_mapping=state["slots"])
        return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    if case["kind"] == "decode":
        return decode_attention(state["q"], state["k"], state["v"], state["block_tables"], state["context_lens"], window=case["window"],
                                sinks=case["sinks"])
    return prompt_attention(state["q"], state["k"], state["v"], state["starts"], block_tables=state.get("block_tables"),
                            context_lens=state.get("context_lens"), causal=case["causal"], window=case["window"], sinks=case["sinks"])


def _plain_rotation(x, cos, sin, weight, interleaved):
    """x [T, heads, D] in 32 bits, cos and sin [T, 1, rotary / 2]."""
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    half = cos.size(-1)
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _run_plain(state: dict):
    case = state["case"]
    d, h, hk = case["dim"], case["heads"], case["kv_heads"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "rotate":
        t, half = case["tokens"], case["rotary"] // 2
        q, k, v = (part.view(t, -1, d) for part in state["qkv"].split([h * d, hk * d, hk * d], dim=1))
        turn = state["cos_sin"][state["positions"]].unsqueeze(1)
        cos, sin = turn[..., :half], turn[..., half:]
        q = _plain_rotation(q.float(), cos, sin, state["q_weight"], case["interleaved"]).to(dtype)
        k = _plain_rotation(k.float(), cos, sin, state["k_weight"], case["interleaved"]).to(dtype)
        stored = t - case["unstored"]
        at = state["slots"][:stored].long()
        state["k_cache"].view(-1, hk, d)[at] = k[:stored]
        state["v_cache"].view(-1, hk, d)[at] = v[:stored]
        return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    scale = d ** -0.5
    if case["kind"] == "decode":
        b, longest = case["sequences"], max(1, max(state["totals"]))
        pages = state["block_tables"].clamp(min=0).long()
        # a few rows at a time: the gathered keys and values of a step stay below a quarter of a GB
        rows = max(1, (1 << 26) // (pages.size(1) * case["page"] * hk * d))
        out = torch.empty(b, h, d, device=DEVICE, dtype=dtype)
        for i in range(0, b, rows):
            chosen = pages[i:i + rows]
            n = chosen.size(0)
            k = state["k"][chosen].view(n, -1, hk, d)[:, :longest].permute(0, 2, 3, 1).float().contiguous()
            v = state["v"][chosen].view(n, -1, hk, d)[:, :longest].transpose(1, 2).float().contiguous()
            q = state["q"][i:i + rows].view(n, hk, h // hk, d).float()
            lens = state["context_lens"][i:i + rows].long()[:, None]
            key = torch.arange(longest, device=DEVICE)[None]
            seen = key < lens
            if case["window"]:
                seen = seen & ((key >= lens - case["window"]) | (key < case["sinks"]))
            seen = seen[:, None, None, :]
            scores = (torch.matmul(q, k) * scale).masked_fill(~seen, float("-inf"))
            top = scores.amax(-1, keepdim=True)
            p = torch.exp(scores - torch.where(top == float("-inf"), torch.zeros_like(top), top)) * seen
            total = p.sum(-1, keepdim=True)
            o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
            out[i:i + rows] = o.view(n, h, d).to(dtype)
        return out
    out = torch.empty_like(state["q"])
    at = before = 0
    for row, (new, total) in enumerate(zip(state["new"], state["totals"])):
        if case["page"]:
            chosen = state["block_tables"][row, :-(-total // case["page"])].long()
            k, v = (state[name][chosen].view(-1, hk, d)[:total] for name in ("k", "v"))
        else:
            k, v = (state[name][before:before + total] for name in ("k", "v"))
        k, v = k.permute(1, 2, 0).float().contiguous(), v.transpose(0, 1).float().contiguous()
        q = state["q"][at:at + new].view(new, hk, h // hk, d).permute(1, 2, 0, 3).float()
        step = max(1, (1 << 28) // (h * total))  # the scores of a step stay at a GB
        for i in range(0, new, step):
            n = min(step, new - i)
            end = total - new + i + n if case["causal"] else total
            scores = torch.matmul(q[:, :, i:i + n].reshape(hk, -1, d), k[:, :, :end]).view(hk, h // hk, n, end) * scale
            if case["causal"]:
                place = torch.arange(total - new + i, total - new + i + n, device=DEVICE)[:, None]
                key = torch.arange(end, device=DEVICE)[None]
                seen = key <= place
                if case["window"]:
                    seen = seen & ((key > place - case["window"]) | (key < case["sinks"]))
                scores = scores.masked_fill_(~seen, float("-inf"))
            p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
            o = torch.matmul(p.view(hk, -1, end), v[:, :end]).view(hk, h // hk, n, d) / p.sum(-1, keepdim=True)
            out[at + i:at + i + n] = o.permute(2, 0, 1, 3).reshape(n, h, d).to(dtype)
        at, before = at + new, before + total
    return out


# ---- the definition in 64 bits -----------------------------------------------------------------------


def exact(case: dict, seed: int):
    d, h, hk = case["dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "prompt" and sum(n * t for n, t in zip(*_lengths(case))) * h * d > 3 << 40:
        return None  # (every score is computed here, what a window hides too)
    s = prepare(case, seed)
    group = h // hk
    if case["kind"] == "rotate":
        t, r = case["tokens"], case["rotary"]
        x = s["qkv"].double().view(t, h + 2 * hk, d)
        if case["norms"]:
            scale = torch.cat([s["q_weight"].double().expand(h, d), s["k_weight"].double().expand(hk, d)])
            lengths = (x[:, :h + hk] ** 2).sum(-1, keepdim=True) / d + 1e-6
            x[:, :h + hk] = x[:, :h + hk] / lengths.sqrt() * scale
        i = torch.arange(r // 2, device=DEVICE)
        first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
        turn = s["cos_sin"][s["positions"].long()].double()
        number = torch.complex(x[:, :h + hk][..., first], x[:, :h + hk][..., second]) * torch.complex(turn[:, :r // 2], turn[:, r // 2:])[:, None]
        x[:, :h + hk, first], x[:, :h + hk, second] = number.real, number.imag
        k, v = s["k_cache"].double(), s["v_cache"].double()
        slots = s["slots"].long()
        kept = slots >= 0
        page, place = slots[kept] // case["page"], slots[kept] % case["page"]
        k[page, place], v[page, place] = x[kept, h:h + hk], x[kept, h + hk:]
        return {"q": x[:, :h].contiguous(), "k_cache": k, "v_cache": v}
    out = torch.zeros(s["q"].shape, device=DEVICE, dtype=torch.float64)
    row_of = base = 0
    for b, (new, total) in enumerate(zip(s["new"], s["totals"])):
        position = torch.arange(total - new, total, device=DEVICE)
        if case["page"]:
            j = torch.arange(total, device=DEVICE)
            where = s["block_tables"][b].long()[j // case["page"]] * case["page"] + j % case["page"]
        else:
            where = base + torch.arange(total, device=DEVICE)
        for g in range(hk if total else 0):
            keys = s["k"].view(-1, hk, d)[where, g].double()
            values = s["v"].view(-1, hk, d)[where, g].double()
            rows = max(1, (1 << 27) // (total * group))
            for i in range(0, new, rows):
                p = position[i:i + rows, None]
                at = slice(row_of + i, row_of + i + p.size(0))
                j = torch.arange(total, device=DEVICE)[None, :]
                hidden = torch.zeros(p.size(0), total, dtype=torch.bool, device=DEVICE)
                if case.get("causal", True):
                    hidden |= j > p
                    if case["window"]:
                        hidden |= (p - j >= case["window"]) & (j >= case["sinks"])
                for head in range(g * group, (g + 1) * group):
                    score = s["q"][at, head].double() @ keys.T.contiguous() / math.sqrt(d)
                    score[hidden] = -math.inf
                    out[at, head] = torch.softmax(score, dim=1) @ values
        row_of, base = row_of + new, base + total
    return out
