"""A decoder whose base weights are held in 8 bits, as measurable cases: the four operators between its attention calls.

Every linear of such a decoder takes rows in 8 bits (e4m3, one fp32 scale a row) and weights in 8 bits (one scale an output
column), and adds the adapters of the batch's requests in the same call.  What makes the rows:

* ``norm`` - the residual stream takes a linear's output, and the RMS norm of the sum is the next linear's input.
* ``gate`` - silu(gate) * up, the input of the down projection.
* ``rows`` - an attention output as it is, the input of the o projection.
* ``project`` - the linear itself: 8-bit product, scales, bias, and per row the low-rank update of its request's adapter.

Sizes are those of the decode, prefill and mixed benchmarks (hidden 1024, SwiGLU 4096, q|k|v 1024|256|256, ranks 8..64, 64 to
256 streams, 16 prompts of 9392 tokens, 8192 tokens over 128 adapters) and of a model twice as wide.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
TOP = 448.0  # the largest e4m3 number
LEAST = 2.0**-100  # no row's scale is smaller (rows of zeros)


def listed() -> list[dict]:
    return [
        # one running request: a launch is all there is
        dict(name="norm_1_token", kind="norm", tokens=1, width=1024, dtype="bf16", residual=True, eight=True),
        # the prefill benchmark's 16 prompts between two layers
        dict(name="norm_9392_tokens", kind="norm", tokens=9392, width=1024, dtype="bf16", residual=True, eight=True),
        # prompts of a wider model whose next linear is one in 16 bits
        dict(name="norm_3001_tokens_wide", kind="norm", tokens=3001, width=2048, dtype="fp16", residual=True, eight=False),
        # the end-to-end benchmark's decode batch, in front of the down projection
        dict(name="gate_64_tokens", kind="gate", tokens=64, width=4096, dtype="bf16", eight=True),
        # the prefill benchmark there
        dict(name="gate_9392_tokens", kind="gate", tokens=9392, width=4096, dtype="bf16", eight=True),
        # attention outputs of a ragged decode batch of a wider model
        dict(name="rows_201_tokens", kind="rows", tokens=201, width=2048, dtype="fp16"),
        # an estimator's fp32 features
        dict(name="rows_8192_tokens_fp32", kind="rows", tokens=8192, width=1024, dtype="fp32"),
        # q|k|v of one running request with its adapter
        dict(name="project_1_token", kind="project", tokens=1, sequences=1, width=1024, columns="1024+256+256", slots=8, rank=32, dtype="bf16",
             without=0.0, bias=False),
        # gate|up of the end-to-end benchmark's decode batch: 64 streams, 32 adapters
        dict(name="project_64_tokens", kind="project", tokens=64, sequences=64, width=1024, columns="4096+4096", slots=32, rank=32, dtype="bf16",
             without=0.0, bias=False),
        # down of a wider model, a ragged batch, one stream in ten without an adapter
        dict(name="project_201_tokens_wide", kind="project", tokens=201, sequences=201, width=8192, columns="2048", slots=48, rank=64, dtype="fp16",
             without=0.1, bias=True),
        # gate|up of the prefill benchmark: 16 prompts, 8 adapters, a quarter of the prompts without one
        dict(name="project_9392_tokens", kind="project", tokens=9392, sequences=16, width=1024, columns="4096+4096", slots=8, rank=64, dtype="bf16",
             without=0.25, bias=False),
        # down of the mixed benchmark: 128 adapters, two chunks of 2048 tokens and 4096 decodes
        dict(name="project_8192_tokens_mixed", kind="project", tokens=8192, sequences=4098, width=4096, columns="1024", slots=128, rank=64,
             dtype="bf16", without=0.0, bias=False),
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
    kind = rng.choice(["norm", "gate", "rows", "project", "project", "project"])
    tokens = _log_int(rng, 1, 9392)
    if kind != "project":
        # (a shard of a model need not be a multiple of anything)
        width = 16 * _log_int(rng, 4, 512) if rng.random() < 0.75 else _log_int(rng, 65, 8191)
        case = dict(kind=kind, tokens=tokens, width=width, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        if kind == "norm":
            case["residual"] = rng.random() < 0.8
        if kind != "rows":
            case["eight"] = rng.random() < 0.7
        return case
    width = 16 * _log_int(rng, 8, 512)
    columns = [rng.choice([16, 64, 1]) * _log_int(rng, 4, 128) for _ in range(rng.choice([1, 2, 3]))]
    slots = rng.choice([0, _log_int(rng, 1, 128), _log_int(rng, 1, 128)])
    return dict(kind=kind, tokens=tokens, sequences=rng.choice([tokens, _log_int(rng, 1, min(64, tokens))]), width=width,
                columns="+".join(map(str, columns)), slots=slots, rank=rng.choice([8, 16, 32, 64]) if slots else 0,
                dtype=rng.choice(["bf16", "bf16", "fp16"]), without=rng.choice([0.0, 0.1, 0.5]) if slots else 0.0, bias=rng.random() < 0.3)


def _columns(case: dict) -> list[int]:
    return [int(n) for n in case["columns"].split("+")]


def _held(case: dict) -> int:
    """Bytes of adapters that the state holds, used in this batch or not, and of the plain form's largest intermediate."""
    if case["kind"] != "project":
        return 0
    return case["slots"] * case["rank"] * (sum(_columns(case)) + len(_columns(case)) * case["width"]) * 2 + 4 * case["tokens"] * case["slots"] * case["rank"]


def _slots(case: dict) -> list[int]:
    """Slot of every token: the adapters belong to the case, their values to the seed."""
    pick = random.Random(case["tokens"] * 1000003 + case["sequences"])
    n, tokens = case["sequences"], case["tokens"]
    if n == tokens:
        lengths = [1] * n
    elif n > 64:  # a mixed batch: two chunks, then decodes
        chunk = (tokens - (n - 2)) // 2
        lengths = [chunk, tokens - (n - 2) - chunk] + [1] * (n - 2)
    else:
        share = [pick.uniform(0.12, 1.88) for _ in range(n)]
        lengths = [1 + int((tokens - n) * s / sum(share)) for s in share]
        lengths[-1] += tokens - sum(lengths)
    found = []
    for length in lengths:
        found += [-1 if not case["slots"] or pick.random() < case["without"] else pick.randrange(case["slots"])] * length
    return found


def work(case: dict) -> dict:
    t, k = case["tokens"], case["width"]
    if case["kind"] == "project":
        e, columns = SIZES[case["dtype"]], _columns(case)
        slots = _slots(case)
        used, rows = len(set(slots) - {-1}), sum(s >= 0 for s in slots)
        adapters = case["rank"] * (len(columns) * k + sum(columns))
        n = sum(columns)
        return {"bytes": t * k + 4 * t + n * k + 4 * n + t * n * e + used * adapters * e + 4 * t + (n * e if case["bias"] else 0),
                "flops": 2 * t * n * k + 2 * rows * adapters}
    e = SIZES[case["dtype"]]
    out = t * k + 4 * t if case.get("eight", True) else t * k * e
    if case["kind"] == "norm":
        return {"bytes": t * k * e * (3 if case["residual"] else 1) + k * e + out, "flops": t * k * (7 if case["eight"] else 5)}
    if case["kind"] == "gate":
        return {"bytes": 2 * t * k * e + out, "flops": t * k * 8}
    return {"bytes": t * k * e + out, "flops": 3 * t * k}


# ---- states ------------------------------------------------------------------------------------------


def _normal(gen: torch.Generator, *shape: int, dtype: torch.dtype, scale: float = 1.0) -> torch.Tensor:
    t = torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)
    return t if scale == 1.0 else t.mul_(scale)


def _in_eight(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of fp32 numbers as e4m3 numbers and a scale a row."""
    scales = (x.abs().amax(-1) / TOP).clamp(min=LEAST)
    return (x / scales[:, None]).to(torch.float8_e4m3fn), scales


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 23)
    t, k, dtype = case["tokens"], case["width"], DTYPES[case["dtype"]]
    if case["kind"] == "norm":
        # (a residual stream is wider than what a layer adds to it, and some of its columns wider than others)
        spread = torch.exp(0.7 * _normal(gen, k, dtype=torch.float32))
        x = _normal(gen, t, k, dtype=dtype)
        residual = (_normal(gen, t, k, dtype=torch.float32) * spread * 3.0).to(dtype) if case["residual"] else None
        return dict(case=case, x=x, residual=residual, weight=(1.0 + _normal(gen, k, dtype=torch.float32, scale=0.2)).to(dtype))
    if case["kind"] == "gate":
        return dict(case=case, x=_normal(gen, t, 2 * k, dtype=dtype, scale=1.5))
    if case["kind"] == "rows":
        return dict(case=case, x=_normal(gen, t, k, dtype=dtype))
    columns, slots, rank = _columns(case), case["slots"], case["rank"]
    n = sum(columns)
    x, x_scales = _in_eight(_normal(gen, t, k, dtype=torch.float32))
    w, w_scales = _in_eight(_normal(gen, n, k, dtype=torch.float32, scale=k ** -0.5))
    state = dict(case=case, x=x, x_scales=x_scales, w=w, w_scales=w_scales, bias=_normal(gen, n, dtype=dtype) if case["bias"] else None)
    if slots:
        state["a"] = [_normal(gen, slots, rank, k, dtype=dtype, scale=0.02) for _ in columns]
        state["b"] = [_normal(gen, slots, m, rank, dtype=dtype, scale=0.04) for m in columns]
        state["slots"] = torch.tensor(_slots(case), dtype=torch.int32, device=DEVICE)
    return state


# ---- one pass ----------------------------------------------------------------------------------------


def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state: dict):
    folder = os.path.join(os.getcwd(), "nanovllm-voxcpm_amd")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    from nanovllm_voxcpm_amd.quant_ops import QuantizedRows, add_rms_norm, quantize_rows, quantized_linear, silu_mul

    case = state["case"]
    if case["kind"] == "norm":
        rows, total = add_rms_norm(state["x"], state["weight"], residual=state["residual"], quantize=case["eight"])
        out = {"values": rows.values, "scales": rows.scales} if case["eight"] else {"values": rows}
        return {**out, "sum": total} if case["residual"] else out
    if case["kind"] == "gate":
        rows = silu_mul(state["x"], quantize=case["eight"])
        return {"values": rows.values, "scales": rows.scales} if case["eight"] else {"values": rows}
    if case["kind"] == "rows":
        rows = quantize_rows(state["x"])
        return {"values": rows.values, "scales": rows.scales}
    return quantized_linear(QuantizedRows(state["x"], state["x_scales"]), QuantizedRows(state["w"], state["w_scales"]), bias=state["bias"],
                            dtype=DTYPES[case["dtype"]], lora_a=state.get("a"), lora_b=state.get("b"), token_to_slot=state.get("slots"))


def _run_plain(state: dict):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "project":
        x = state["x"].float()
        y = torch.matmul(x, state["w"].float().t()) * state["x_scales"][:, None] * state["w_scales"]
        if case["slots"]:
            # every adapter's intermediate for every row, and of them the row's own
            slot_of = torch.arange(case["slots"], device=DEVICE, dtype=torch.int32).repeat_interleave(case["rank"])
            mine = state["slots"][:, None] == slot_of
            updates = []
            for a, b in zip(state["a"], state["b"]):
                h = torch.matmul(x, a.view(-1, case["width"]).float().t()) * state["x_scales"][:, None]
                updates.append(torch.matmul(h * mine, b.transpose(1, 2).reshape(-1, b.size(1)).float()))
            y = y + torch.cat(updates, dim=1)
        if state["bias"] is not None:
            y = y + state["bias"].float()
        return y.to(dtype)
    out = {}
    x = state["x"].float()
    if case["kind"] == "norm":
        if state["residual"] is not None:
            out["sum"] = (x + state["residual"].float()).to(dtype)
            x = out["sum"].float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * state["weight"].float()
    elif case["kind"] == "gate":
        gate, up = x[:, :case["width"]], x[:, case["width"]:]
        y = gate / (1 + torch.exp(-gate)) * up
    else:
        y = x
    if case.get("eight", True):
        out["values"], out["scales"] = _in_eight(y)
    else:
        out["values"] = y.to(dtype)
    return out


# ---- the definition in 64 bits -----------------------------------------------------------------------


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["kind"] == "project":
        x = x * s["x_scales"].double().unsqueeze(1)
        y = torch.addmm(torch.zeros((), dtype=torch.float64, device=DEVICE), x, (s["w"].double() * s["w_scales"].double().unsqueeze(1)).t().contiguous())
        if s["bias"] is not None:
            y += s["bias"].double()
        held = torch.tensor(_slots(case), device=DEVICE)
        for slot in sorted(set(_slots(case)) - {-1}):
            rows = torch.nonzero(held == slot).flatten()
            first = 0
            for a, b in zip(s["a"], s["b"]):
                y[rows, first:first + b.size(1)] += x[rows] @ a[slot].double().t() @ b[slot].double().t()
                first += b.size(1)
        return y
    out = {}
    if case["kind"] == "norm":
        if case["residual"]:
            # (the sum is held in the element type, and it is its norm that is taken)
            out["sum"] = x + s["residual"].double()
            x = out["sum"].float().to(s["x"].dtype).double()
        length = torch.sqrt(torch.linalg.vector_norm(x, dim=1).square() / case["width"] + 1e-6)
        x = x * s["weight"].double() / length.unsqueeze(1)
    elif case["kind"] == "gate":
        x = torch.sigmoid(x[:, :case["width"]]) * x[:, :case["width"]] * x[:, case["width"]:]
    if case.get("eight", True):
        # (before the rounding to 8 bits)
        out["scales"] = torch.clamp(x.abs().max(dim=1).values / TOP, min=LEAST)
        x = x / out["scales"].unsqueeze(1)
    out["values"] = x
    return out
