"""A decoder's linears with base weights in 8 bits, and the rows between them, executed by the HIP library.

Rows and weights in 8 bits are ``QuantizedRows``: e4m3 numbers and one fp32 scale a row (of a weight: an output column).
``quantize_rows`` makes them of any rows, ``add_rms_norm`` (residual sum and RMS norm; reference: nanovllm_voxcpm/layers/layernorm.py) and
``silu_mul`` (reference: nanovllm_voxcpm/layers/activation.py) of what stands in front of a linear, or leave it in the element type;
``quantized_linear`` multiplies them and adds, row by row, the low-rank update of the row's adapter (reference:
nanovllm_voxcpm/layers/lora.py, the forward of the LoRA linears, whose base weights have 16 bits).

All four enqueue work on torch's current stream and neither synchronise nor read device data on the host, so they may be captured into a
graph.  They have no derivatives: call them under ``torch.no_grad()`` or ``torch.inference_mode()``.  Element types are fp32, fp16 and bf16 for
rows, fp16 and bf16 for linears.
"""

from __future__ import annotations

from typing import NamedTuple, Sequence

import torch
from torch.autograd import forward_ad

from nanovllm_voxcpm_amd import _hip
from nanovllm_voxcpm_amd.attention_ops import _overlap, _rows_apart

__all__ = ["QuantizedRows", "add_rms_norm", "quantize_rows", "quantized_linear", "silu_mul"]


class QuantizedRows(NamedTuple):
    """Row r stands for ``values[r] * scales[r]``."""

    values: torch.Tensor  # [rows, width] float8_e4m3fn
    scales: torch.Tensor  # [rows] fp32

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return (self.values.float() * self.scales[:, None]).to(dtype)


def _no_grad(*tensors: torch.Tensor | None) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("the 8-bit ops have no backward: call them under torch.no_grad() or torch.inference_mode()")
    if not torch.is_inference_mode_enabled() and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("the 8-bit ops have no backward, nor a forward derivative: a tensor carries a tangent")


MOST_FEATURES = 2**22  # of a linear, in or out
_MOST = 2**31 - 1  # (sizes are 32-bit numbers in the library, which refuses what it does not serve below that)


def _rows(t: torch.Tensor, name: str, like: torch.Tensor | None = None) -> None:
    if t.dim() != 2:
        raise ValueError(f"{name} must be [rows, width], got shape {tuple(t.shape)}")
    if max(t.shape) > _MOST:
        raise ValueError(f"{name} {tuple(t.shape)} is larger than a call takes")
    if t.size(1) < 1:
        raise ValueError(f"{name} has rows without elements")
    if t.numel() and t.stride(1) != 1 and t.size(1) != 1:
        raise ValueError(f"the elements of a row of {name} must lie side by side")
    if like is None:
        _hip.dtype_code(t.dtype)
        return
    if t.device != like.device:
        raise ValueError(f"{name} lives on {t.device}, x on {like.device}")
    if t.dtype != like.dtype:
        raise ValueError(f"{name} has element type {t.dtype}, x has {like.dtype}")
    if t.shape != like.shape:
        raise ValueError(f"{name} {tuple(t.shape)} and x {tuple(like.shape)} differ")


def _outputs(x: torch.Tensor, width: int, quantize: bool) -> tuple[torch.Tensor, torch.Tensor | None]:
    shape = (x.size(0), width)
    if not quantize:
        return torch.empty(shape, dtype=x.dtype, device=x.device), None
    return torch.empty(shape, dtype=torch.float8_e4m3fn, device=x.device), torch.empty(x.size(0), dtype=torch.float32, device=x.device)


def quantize_rows(x: torch.Tensor) -> QuantizedRows:
    """Rows of ``x [rows, width]`` in 8 bits: scale = max(max|x| / 448, 2^-100), values = e4m3(x / scale).

    A row with a NaN is NaN altogether; one with an infinity has an infinite scale.  Of a weight ``[out, in]`` this makes what ``quantized_linear`` takes.
    """
    fast = _hip.load_fastcall()
    if fast is not None:  # the usual call, checked and enqueued in C++
        result = fast.rows(_hip.entry_point("mlora_quantize_rows"), x, 1, True, None, None, 0.0, None)
        if result is not None:
            return QuantizedRows(result[0], result[1])
    _rows(x, "x")
    _no_grad(x)
    values, scales = _outputs(x, x.size(1), True)
    _hip.rows("mlora_quantize_rows", x, values, scales, x.size(1))
    return QuantizedRows(values, scales)


def add_rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    *,
    residual: torch.Tensor | None = None,
    eps: float = 1e-6,
    quantize: bool = False,
    sum_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor | QuantizedRows, torch.Tensor]:
    """(norm, sum): sum = x + residual, rounded to the element type, and norm = sum * rsqrt(mean(sum^2) + eps) * weight, for every row of
    ``x``, ``residual [rows, width]``.

    ``weight``: ``[width]``, of x's element type or fp32.  ``quantize``: the norm in 8 bits, else in the element type; fp32 in between, one
    rounding.  The sum goes to ``sum_out`` where given (x or the residual itself are fine), else to a new tensor; without a residual
    it is x itself and nothing is written.
    """
    fast = _hip.load_fastcall()
    if fast is not None and weight is not None:
        result = fast.rows(_hip.entry_point("mlora_add_rms_norm"), x, 1, quantize, weight, residual, eps, sum_out)
        if result is not None:
            return QuantizedRows(result[0], result[1]) if quantize else result[0], x if residual is None else result[2]
    _rows(x, "x")
    _no_grad(x, weight, residual, sum_out)
    if weight.device != x.device:
        raise ValueError(f"weight lives on {weight.device}, x on {x.device}")
    if weight.dtype not in (x.dtype, torch.float32) or weight.shape != (x.size(1),) or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous vector of {x.size(1)} elements, fp32 or {x.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    total = x
    if residual is not None:
        _rows(residual, "residual", x)
        total = torch.empty(x.shape, dtype=x.dtype, device=x.device) if sum_out is None else sum_out
        if sum_out is not None:
            _rows(sum_out, "sum_out", x)
            _rows_apart(sum_out, "sum_out")
            for t, name in ((x, "x"), (residual, "residual")):
                if not (sum_out.data_ptr() == t.data_ptr() and sum_out.stride() == t.stride()) and _overlap(sum_out, t):
                    raise ValueError(f"sum_out overlaps {name}")
            if _overlap(sum_out, weight):
                raise ValueError("sum_out overlaps weight")
    elif sum_out is not None:
        raise ValueError("sum_out is for a sum: there is no residual")
    out, scales = _outputs(x, x.size(1), quantize)
    _hip.rows("mlora_add_rms_norm", x, out, scales, x.size(1), residual=residual, total=None if residual is None else total, weight=weight, eps=float(eps))
    return (QuantizedRows(out, scales) if quantize else out), total


def silu_mul(gate_up: torch.Tensor, *, quantize: bool = False) -> torch.Tensor | QuantizedRows:
    """silu(gate) * up for rows gate | up of ``gate_up [rows, 2 * width]``, silu(g) = g / (1 + exp(-g)); in 8 bits with ``quantize``, else in the
    element type; fp32 in between, one rounding."""
    fast = _hip.load_fastcall()
    if fast is not None:
        result = fast.rows(_hip.entry_point("mlora_silu_mul"), gate_up, 2, quantize, None, None, 0.0, None)
        if result is not None:
            return QuantizedRows(result[0], result[1]) if quantize else result[0]
    _rows(gate_up, "gate_up")
    _no_grad(gate_up)
    if gate_up.size(1) % 2:
        raise ValueError(f"gate_up has {gate_up.size(1)} columns: gate and up are as wide as each other")
    width = gate_up.size(1) // 2
    out, scales = _outputs(gate_up, width, quantize)
    _hip.rows("mlora_silu_mul", gate_up, out, scales, width)
    return QuantizedRows(out, scales) if quantize else out


def _quantized(rows: QuantizedRows, name: str, device: torch.device | None = None) -> None:
    values, scales = rows
    if values.dtype != torch.float8_e4m3fn or values.dim() != 2:
        raise ValueError(f"values of {name} must be float8_e4m3fn [rows, width], got {values.dtype} {tuple(values.shape)}")
    if max(values.shape) > _MOST:
        raise ValueError(f"{name} {tuple(values.shape)} is larger than a call takes")
    if values.size(1) < 1 or values.size(1) % 16:
        raise ValueError(f"rows of {name} have {values.size(1)} elements, which is no multiple of 16")
    if values.numel() and (values.stride(1) != 1 or values.data_ptr() % 16 or (values.size(0) > 1 and values.stride(0) % 16)):
        raise ValueError(f"rows of {name} must start on 16 bytes, with elements side by side")
    if scales.dtype != torch.float32 or scales.shape != (values.size(0),) or not scales.is_contiguous():
        raise ValueError(f"scales of {name} must be a contiguous fp32 vector of {values.size(0)} elements")
    if scales.device != values.device:
        raise ValueError(f"values of {name} live on {values.device}, its scales on {scales.device}")
    if device is not None and values.device != device:
        raise ValueError(f"{name} lives on {values.device}, x on {device}")


def _adapters(a: Sequence[torch.Tensor], b: Sequence[torch.Tensor], columns: Sequence[int] | None, width: int, out: int, dtype: torch.dtype, device: torch.device) -> list[int]:
    if len(a) != len(b) or not a or (columns is not None and len(columns) != len(a)):
        raise ValueError(f"{len(a)} lora_a and {len(b)} lora_b" + ("" if columns is None else f" for {len(columns)} lora_columns"))
    if len(a) > _hip.MAX_SLICES:
        raise ValueError(f"{len(a)} adapter targets, at most {_hip.MAX_SLICES} are served")
    slots, rank = (a[0].shape[:2] if a[0].dim() == 3 else (0, 0))
    if slots < 1 or rank < 1 or slots > _hip.MAX_SLOTS or rank > _hip.MAX_RANK:
        raise ValueError(f"lora_a must be [slots, rank, in], up to {_hip.MAX_SLOTS} slots of rank {_hip.MAX_RANK}, got shape {tuple(a[0].shape)}")
    first, end = [], 0
    for i, (a_of, b_of) in enumerate(zip(a, b)):
        if a_of.shape != (slots, rank, width) or b_of.dim() != 3 or b_of.size(0) != slots or b_of.size(2) != rank or b_of.size(1) < 1:
            raise ValueError(f"lora_a {tuple(a_of.shape)} and lora_b {tuple(b_of.shape)} of target {i} must be [{slots}, {rank}, {width}] and [{slots}, columns, {rank}]")
        for t, name in ((a_of, "lora_a"), (b_of, "lora_b")):
            if t.dtype != dtype or t.device != device or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} of target {i} must be contiguous, on 16 bytes, {dtype} on {device}, got {t.dtype} on {t.device}")
        first.append(end if columns is None else int(columns[i]))
        if first[-1] < end or first[-1] + b_of.size(1) > out:
            raise ValueError(f"columns {first[-1]} to {first[-1] + b_of.size(1)} of target {i} do not lie behind those of the one before it, inside {out}")
        end = first[-1] + b_of.size(1)
    return first


def quantized_linear(
    rows: QuantizedRows,
    weight: QuantizedRows,
    *,
    bias: torch.Tensor | None = None,
    dtype: torch.dtype = torch.bfloat16,
    lora_a: Sequence[torch.Tensor] | None = None,
    lora_b: Sequence[torch.Tensor] | None = None,
    token_to_slot: torch.Tensor | None = None,
    lora_columns: Sequence[int] | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``x W^T + bias`` of rows ``x [T, in]`` and a weight ``W [out, in]`` in 8 bits, and ``(x A[s]^T) B[s]^T`` beside it for the adapter s =
    ``token_to_slot[t]`` of every row.

    ``dtype``: fp16 or bf16, of the result, the bias ``[out]`` and the adapters.  ``lora_a``, ``lora_b``: buffers ``[slots, rank, in]`` and ``[slots,
    columns, rank]`` of every target (q, k and v of a stacked projection), whose columns lie one behind the other, or from ``lora_columns`` on;
    ``token_to_slot``: int32 ``[T]``, ids outside the slots stand for rows without an adapter.  Sums are fp32, the result is rounded
    once.  ``in`` is a multiple of 16 and rows start on 16 bytes; up to 2^20 rows a call, ``in`` and ``out`` up to 2^22.
    """
    fast = _hip.load_fastcall()
    if fast is not None and out is None and lora_columns is None:
        result = fast.linear8(_hip.entry_point("mlora_project"), _hip.entry_point("mlora_project_workspace_bytes"), rows[0], rows[1], weight[0], weight[1], bias, dtype,
                              lora_a, lora_b, token_to_slot)
        if result is not None:
            return result
    _quantized(rows, "rows")
    _quantized(weight, "weight", rows.values.device)
    x, w = rows.values, weight.values
    device, width, columns = x.device, x.size(1), w.size(0)
    if w.size(1) != width:
        raise ValueError(f"rows have {width} elements, the weight {tuple(w.shape)} takes {w.size(1)}")
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"dtype must be float16 or bfloat16, got {dtype}")
    if bias is not None and (bias.shape != (columns,) or bias.dtype != dtype or bias.device != device or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous vector of {columns} elements, {dtype} on {device}")
    given = [t is not None for t in (lora_a, lora_b, token_to_slot)]
    if any(given) and not all(given):
        raise ValueError("lora_a, lora_b and token_to_slot are given together or not at all")
    first: list[int] = []
    a, b = list(lora_a or ()), list(lora_b or ())
    _no_grad(*rows, *weight, bias, *a, *b, out)
    if all(given):
        first = _adapters(a, b, lora_columns, width, columns, dtype, device)
        if token_to_slot.dtype != torch.int32 or token_to_slot.shape != (x.size(0),) or not token_to_slot.is_contiguous() or token_to_slot.device != device:
            raise ValueError(f"token_to_slot must be a contiguous int32 vector of {x.size(0)} elements on {device}")
    elif lora_columns is not None:
        raise ValueError("lora_columns is for adapters: there are none")
    if out is None:
        out = torch.empty(x.size(0), columns, dtype=dtype, device=device)
    else:
        if out.shape != (x.size(0), columns) or out.dtype != dtype or out.device != device or (out.numel() and out.stride(1) != 1 and columns != 1):
            raise ValueError(f"out must be {dtype} [{x.size(0)}, {columns}] on {device}, with rows side by side")
        _rows_apart(out, "out")
        for t in (*rows, *weight, bias, token_to_slot, *a, *b):
            if t is not None and _overlap(out, t):
                raise ValueError("out overlaps one of the inputs")
    _hip.project(x, rows.scales, w, weight.scales, bias, out, a, b, first, token_to_slot)
    return out
