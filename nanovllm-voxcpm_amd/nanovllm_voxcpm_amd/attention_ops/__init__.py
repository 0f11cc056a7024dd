"""The attention block between the q|k|v and the o linear, executed by the HIP library.

``rotate_qk`` norms and rotates the query and key heads of a batch and writes keys and values into the pages of a cache
(reference: nanovllm_voxcpm/layers/rotary_embedding.py, layers/attention.py:10-50); ``decode_attention`` attends with one new
token per sequence to such a cache, ``prompt_attention`` with any number of rows per sequence to packed keys or to a cache
(reference: nanovllm_voxcpm/layers/attention.py:70-105).

All three enqueue work on torch's current stream and neither synchronise nor read device data on the host, so they may be
captured into a graph.  They have no derivatives: call them under ``torch.no_grad()`` or ``torch.inference_mode()``.
Element types are fp32, fp16 and bf16, head sizes multiples of 8 up to 256; index vectors are int32 (positions and slots may
be int64).  The rotary size, columns of the table of ``rotate_qk``, is a multiple of 16 up to the head size, or 0.  Tensors may be strided views as long as a head's elements lie side by side.

Attention is fast at head sizes 64 and 128 with rows that start on 16 bytes.  Every other call is right but runs on a kernel that reads
its keys one at a time: short sequences do well there, long ones take longer than a product, a softmax and a product of torch's would
(3 streams of 131072 keys, 8 heads of 96, 97 ms and 4; 64 of 2048 1.2 ms and 0.4).  A table of blocks wider than the longest sequence costs
decode a second launch where its width alone asks for one (64 streams of up to 2048 keys 12.9 us, 15.8 in tables of twice that).
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from nanovllm_voxcpm_amd import _hip

__all__ = ["decode_attention", "prompt_attention", "rotary_table", "rotate_qk"]


def rotary_table(rotary_dim: int, num_positions: int, *, base: float = 10000.0, factors: torch.Tensor | list[float] | None = None,
                 scale: float = 1.0, device: torch.device | str | None = None) -> torch.Tensor:
    """The fp32 table ``[num_positions, rotary_dim]`` of ``rotate_qk``: cosines, then sines, of position * base ** (-2 i / rotary_dim) /
    factors[i] (``factors``: one per pair, for long-context models), times ``scale``.  ``rotate_qk`` takes sizes that are multiples of 16.  Angles are computed in 64 bits: in 32
    those of far positions are off by thousandths."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be an even number, got {rotary_dim}")
    if num_positions < 1:
        raise ValueError(f"num_positions must be positive, got {num_positions}")
    half = rotary_dim // 2
    inverse = float(base) ** (-torch.arange(half, dtype=torch.float64) / half)
    if factors is not None:
        factors = torch.as_tensor(factors, dtype=torch.float64).cpu()
        if factors.shape != (half,):
            raise ValueError(f"factors must hold one value for each of the {half} pairs, got shape {tuple(factors.shape)}")
        inverse = inverse / factors
    angles = torch.arange(num_positions, dtype=torch.float64)[:, None] * inverse[None, :]
    return (torch.cat([angles.cos(), angles.sin()], dim=1) * scale).float().to(device or "cpu")


def _heads(t: torch.Tensor, name: str, like: torch.Tensor | None = None) -> None:
    if t.dim() != 3:
        raise ValueError(f"{name} must be [rows, heads, head size], got shape {tuple(t.shape)}")
    if t.numel() and t.stride(2) != 1 and t.size(2) != 1:
        raise ValueError(f"the elements of a head of {name} must lie side by side")
    _same(t, name, like)


def _same(t: torch.Tensor, name: str, like: torch.Tensor | None) -> None:
    if like is None:
        return
    if t.device != like.device:
        raise ValueError(f"{name} lives on {t.device}, q on {like.device}")
    if t.dtype != like.dtype:
        raise ValueError(f"{name} has element type {t.dtype}, q has {like.dtype}")


def _index(t: torch.Tensor, name: str, device: torch.device, least: int, dtypes=(torch.int32,)) -> None:
    if t.dtype not in dtypes or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {' or '.join(str(d).replace('torch.', '') for d in dtypes)} vector")
    if t.device != device:
        raise ValueError(f"{name} lives on {t.device}, q on {device}")
    if t.numel() < least:
        raise ValueError(f"{name} has {t.numel()} entries, {least} are needed")


def _cache(k: torch.Tensor, v: torch.Tensor, kv_heads: int | None, q: torch.Tensor, names=("k_cache", "v_cache")) -> None:
    for t, name in ((k, names[0]), (v, names[1])):
        if t.dim() != 4:
            raise ValueError(f"{name} must be [blocks, rows of a block, heads, head size], got shape {tuple(t.shape)}")
        if t.numel() and t.stride(3) != 1 and t.size(3) != 1:
            raise ValueError(f"the elements of a head of {name} must lie side by side")
        _same(t, name, q)
    if k.shape != v.shape:
        raise ValueError(f"{names[0]} {tuple(k.shape)} and {names[1]} {tuple(v.shape)} differ")
    if k.size(1) < 1:
        raise ValueError(f"{names[0]} has blocks without rows")
    if k.size(3) != q.size(2) or (kv_heads is not None and k.size(2) != kv_heads):
        raise ValueError(f"{names[0]} {tuple(k.shape)} does not hold heads of size {q.size(2)}" + (f", {kv_heads} of them" if kv_heads is not None else ""))


def _no_grad(*tensors: torch.Tensor | None) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("the attention ops have no backward: call them under torch.no_grad() or torch.inference_mode()")
    if not torch.is_inference_mode_enabled() and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("the attention ops have no backward, nor a forward derivative: a tensor carries a tangent")


def _memory(t: torch.Tensor) -> tuple[int, int, int, int]:
    """First byte of a strided tensor and the one behind its last; bytes from row to row and of a row's extent."""
    size, shape, strides = t.element_size(), t.shape, t.stride()
    if 0 in shape:
        return 0, 0, 0, 0
    width = 1 + sum((n - 1) * s for n, s in zip(shape[1:], strides[1:]))
    start = t.data_ptr()
    return start, start + size * ((shape[0] - 1) * strides[0] + width), size * strides[0], size * width


def _beside(a: tuple[int, int, int, int], b: tuple[int, int, int, int]) -> bool:
    """Whether two tensors' memory is plainly apart: one behind the other, or columns of one buffer, rows as far apart in both."""
    if a[1] <= b[0] or b[1] <= a[0]:
        return True
    row = a[2]
    if row != b[2] or row <= 0:
        return False
    apart = (b[0] - a[0]) % row
    return a[3] <= apart and apart + b[3] <= row


def _reaches(terms: list[tuple[int, int, int]], target: int, tries: list[int]) -> bool:
    """Whether sum c x = target for some whole numbers x, terms (c, least x, largest x) of falling c > 0.  Strides nest as a rule, so that one or
    two x are possible at every term; after ``tries[0]`` of them the answer is yes."""
    if not terms:
        return target == 0
    (c, lo, hi), rest = terms[0], terms[1:]
    least, most = sum(r * x for r, x, _ in rest), sum(r * x for r, _, x in rest)
    for x in range(max(lo, -((most - target) // c)), min(hi, (target - least) // c) + 1):
        tries[0] -= 1
        if tries[0] < 0 or _reaches(rest, target - c * x, tries):
            return True
    return False


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether an element of one tensor lies on one of the other.  (Views may lie between one another without: heads of the packed rows of a linear.)"""
    at, bt = _memory(a), _memory(b)
    if _beside(at, bt):
        return False
    # an address of a less one of b, by bytes
    terms = {1: [1 - b.element_size(), a.element_size() - 1]}
    for t, end, sign in ((a, 1, 1), (b, 0, -1)):
        for n, s in zip(t.shape, t.stride()):
            if n > 1 and s:
                terms.setdefault(s * t.element_size(), [0, 0])[end] += sign * (n - 1)
    return _reaches([(c, *terms[c]) for c in sorted(terms, reverse=True)], bt[0] - at[0], [10000])


def _rows_apart(t: torch.Tensor, name: str) -> None:
    """A written tensor's elements must not lie on one another (an expanded view, rows closer than they are long)."""
    if t.is_contiguous() or not t.numel():
        return
    terms = sorted(((s, n - 1) for n, s in zip(t.shape, t.stride()) if n > 1), reverse=True)
    reach = 0  # of the dimensions of smaller strides
    for i in range(len(terms) - 1, -1, -1):
        stride, most = terms[i]
        # (where strides do not nest: a step along some dimension that the others take back)
        if stride <= reach or stride == 0:
            for j in range(len(terms)):
                one = [(s, 1 if n == j else -m, m) for n, (s, m) in enumerate(terms) if s]
                if terms[j][0] == 0 or _reaches(one, 0, [10000]):
                    raise ValueError(f"rows or heads of {name} share memory")
            return
        reach += stride * most


def _result(out: torch.Tensor | None, source: torch.Tensor, name: str) -> torch.Tensor:
    """The caller's output, or a new one; it may be the source's own memory with the same strides."""
    if out is None:
        return torch.empty(source.shape, dtype=source.dtype, device=source.device)
    if out.shape != source.shape:
        raise ValueError(f"{name} has shape {tuple(out.shape)}, {tuple(source.shape)} is needed")
    _heads(out, name, source)
    _rows_apart(out, name)
    if not (out.data_ptr() == source.data_ptr() and out.stride() == source.stride()) and _overlap(out, source):
        raise ValueError(f"{name} overlaps its input")
    return out


def rotate_qk(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    *,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    v: torch.Tensor | None = None,
    k_cache: torch.Tensor | None = None,
    v_cache: torch.Tensor | None = None,
    slot_mapping: torch.Tensor | None = None,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Norm and rotate the heads of ``q [T, heads, D]`` and ``k [T, kv_heads, D]`` and store k and v in a cache, in one launch.

    ``q_weight``, ``k_weight`` (``[D]``, the element type of q or fp32): RMS norm of every head first, x * rsqrt(mean(x^2) + eps) *
    weight; None leaves the heads as they are.  The first ``cos_sin.size(1)`` elements of a head are then turned by row
    ``positions[t]`` of the table (``rotary_table``), in pairs (i, i + half) or, ``interleaved``, (2 i, 2 i + 1).  Everything is
    computed in fp32 and rounded once.  A position outside the table gives NaN.

    With ``k_cache``, ``v_cache [blocks, rows of a block, kv_heads, D]``, ``v`` and ``slot_mapping [T]`` the new k and v of token t go to row
    ``slot_mapping[t]`` of the cache, counted over all blocks; a negative slot (padding) or one behind the last block is
    not stored.  No two tokens may share a slot, and no two rows of the caches memory.

    Returns (q, k): in ``q_out`` and ``k_out`` where given (an input itself is fine; the caches and the other tensors are not), else new
    tensors; k is None with a cache and without ``k_out``, since the cache has it.
    """
    fast = _hip.load_fastcall()
    if fast is not None and q_out is None and k_out is None:  # the usual call, checked and enqueued in C++
        result = fast.rotate(_hip.entry_point("mlora_rotate_qk"), q, k, positions, cos_sin, q_weight, k_weight, eps, interleaved, v, k_cache, v_cache, slot_mapping)
        if result is not None:
            return result
    _heads(q, "q")
    _heads(k, "k", q)
    _no_grad(q, k, v, q_weight, k_weight, cos_sin)
    rows, dim = q.size(0), q.size(2)
    if k.size(0) != rows or k.size(2) != dim:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in rows or head size")
    _index(positions, "positions", q.device, rows, (torch.int32, torch.int64))
    if cos_sin.dim() != 2 or cos_sin.dtype != torch.float32 or (cos_sin.numel() and cos_sin.stride(1) != 1):
        raise ValueError("cos_sin must be an fp32 [positions, rotary size] table with rows side by side")
    if cos_sin.device != q.device:
        raise ValueError(f"cos_sin lives on {cos_sin.device}, q on {q.device}")
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is None:
            continue
        if w.device != q.device:
            raise ValueError(f"{name} lives on {w.device}, q on {q.device}")
        if w.dtype not in (q.dtype, torch.float32) or w.shape != (dim,) or not w.is_contiguous():
            raise ValueError(f"{name} must be a contiguous vector of {dim} elements, fp32 or {q.dtype}")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("q_weight and k_weight must have the same element type")
    cached = [t is not None for t in (v, k_cache, v_cache, slot_mapping)]
    if any(cached) and not all(cached):
        raise ValueError("v, k_cache, v_cache and slot_mapping are given together or not at all")
    if all(cached):
        _heads(v, "v", q)
        if v.shape != k.shape:
            raise ValueError(f"v {tuple(v.shape)} and k {tuple(k.shape)} differ")
        _cache(k_cache, v_cache, k.size(1), q)
        for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
            _rows_apart(t, name)
        _index(slot_mapping, "slot_mapping", q.device, rows, (torch.int32, torch.int64))
    q_out = _result(q_out, q, "q_out")
    if k_out is not None or not all(cached):
        k_out = _result(k_out, k, "k_out")
    lies = {id(t): _memory(t) for t in (q, k, v, q_out, k_out, k_cache, v_cache) if t is not None}
    for out, name, others in ((q_out, "q_out", (k, v, k_out)), (k_out, "k_out", (q, v))):
        if out is None:
            continue
        for t, of in (*((t, "another of the tensors") for t in others), (k_cache, "k_cache"), (v_cache, "v_cache")):
            if t is not None and not _beside(lies[id(out)], lies[id(t)]) and _overlap(out, t):
                raise ValueError(f"{name} overlaps {of}")
    if all(cached) and q.is_cuda and not _beside(lies[id(k_cache)], lies[id(v_cache)]) and _overlap(k_cache, v_cache):  # (of host tensors nothing is written)
        raise ValueError("k_cache overlaps v_cache")
    _hip.rotate_qk(q, k, v, q_out, k_out, k_cache, v_cache, positions, slot_mapping, cos_sin, q_weight, k_weight, float(eps), bool(interleaved))
    return q_out, k_out


def _masks(window: int, sinks: int) -> None:
    if window < 0 or sinks < 0:
        raise ValueError(f"window and sinks must not be negative, got {window} and {sinks}")


def _table(block_tables: torch.Tensor, context_lens: torch.Tensor, sequences: int, device: torch.device) -> None:
    if block_tables.dim() != 2 or block_tables.dtype != torch.int32 or (block_tables.numel() and block_tables.size(1) > 1 and block_tables.stride(1) != 1):
        raise ValueError("block_tables must be an int32 [sequences, blocks] table with rows side by side")
    if block_tables.device != device:
        raise ValueError(f"block_tables lives on {block_tables.device}, q on {device}")
    if block_tables.size(0) < sequences:
        raise ValueError(f"block_tables has {block_tables.size(0)} rows for {sequences} sequences")
    _index(context_lens, "context_lens", device, sequences)


def _output(out: torch.Tensor | None, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.shape != q.shape:
        raise ValueError(f"out has shape {tuple(out.shape)}, {tuple(q.shape)} is needed")
    _heads(out, "out", q)
    _rows_apart(out, "out")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if _overlap(out, t):
            raise ValueError(f"out overlaps {name}")
    return out


def _shared_heads(heads: int, kv_heads: int) -> None:
    if heads and (kv_heads < 1 or heads % kv_heads):
        raise ValueError(f"{heads} query heads do not share {kv_heads} key-value heads evenly")


def decode_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    *,
    scale: float | None = None,
    window: int = 0,
    sinks: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of one new token per sequence, ``q [sequences, heads, D]``, over the first ``context_lens[s]`` rows (the new token's among
    them) of the pages ``block_tables[s]`` of ``k_cache``, ``v_cache [blocks, rows of a block, kv_heads, D]``.

    ``scale``: of the scores, D ** -0.5 by default.  ``window``: only the last ``window`` rows are seen (0: all), and the
    first ``sinks`` beside them.  A sequence of no rows (padding) gives 0.  Lengths beyond the table's pages end there; the rows of a page
    id outside the cache are not seen.  What lies in rows that are not seen does not matter.
    """
    fast = _hip.load_fastcall()
    if fast is not None and out is None:
        result = fast.decode(_hip.entry_point("mlora_decode_attention"), _hip.entry_point("mlora_decode_attention_workspace_bytes"), q, k_cache, v_cache,
                             block_tables, context_lens, scale, window, sinks)
        if result is not None:
            return result
    _heads(q, "q")
    _cache(k_cache, v_cache, None, q)
    _no_grad(q, k_cache, v_cache)
    _shared_heads(q.size(1), k_cache.size(2))
    _masks(window, sinks)
    _table(block_tables, context_lens, q.size(0), q.device)
    out = _output(out, q, k_cache, v_cache)
    _hip.decode_attention(q, out, k_cache, v_cache, block_tables, context_lens, q.size(2) ** -0.5 if scale is None else float(scale), window, sinks)
    return out


def prompt_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    cu_seqlens_k: torch.Tensor | None = None,
    block_tables: torch.Tensor | None = None,
    context_lens: torch.Tensor | None = None,
    causal: bool = True,
    scale: float | None = None,
    window: int = 0,
    sinks: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of packed sequences: rows ``cu_seqlens[s] : cu_seqlens[s + 1]`` of ``q [T, heads, D]`` are the last rows of sequence s.
    (Starts that decrease are read as they are: nothing outside the tensors is touched, but not every row need be written.)

    Keys and values lie packed, ``k``, ``v [rows, kv_heads, D]`` with sequence s at ``cu_seqlens_k[s] : cu_seqlens_k[s + 1]`` (``cu_seqlens`` by
    default), or, with ``block_tables`` and ``context_lens``, in the pages of a cache, ``[blocks, rows of a block, kv_heads, D]``, as in
    ``decode_attention``.  ``causal``: a row sees its own key and those in front of it, with ``window`` only the last ``window`` of
    them and the first ``sinks`` keys; without ``causal`` every row sees the whole sequence.  Rows that see nothing are 0, rows of
    ``out`` behind the last sequence are left as they are (a new ``out`` holds anything there).
    """
    fast = _hip.load_fastcall()
    if fast is not None and out is None:
        result = fast.prompt(_hip.entry_point("mlora_prompt_attention"), _hip.entry_point("mlora_prompt_attention_workspace_bytes"), q, k, v, cu_seqlens,
                             cu_seqlens_k, block_tables, context_lens, causal, scale, window, sinks)
        if result is not None:
            return result
    _heads(q, "q")
    _masks(window, sinks)
    if not causal and (window or sinks):
        raise ValueError("a window or sinks need causal order")
    _index(cu_seqlens, "cu_seqlens", q.device, 1)
    sequences = cu_seqlens.numel() - 1
    if (block_tables is None) != (context_lens is None):
        raise ValueError("block_tables and context_lens are given together or not at all")
    if block_tables is not None:
        if cu_seqlens_k is not None:
            raise ValueError("cu_seqlens_k is for packed keys: with block_tables context_lens says how many there are")
        _cache(k, v, None, q, ("k", "v"))
        _shared_heads(q.size(1), k.size(2))
        _table(block_tables, context_lens, sequences, q.device)
    else:
        _heads(k, "k", q)
        _heads(v, "v", q)
        if k.shape != v.shape or k.size(2) != q.size(2):
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be alike, with heads of size {q.size(2)}")
        _shared_heads(q.size(1), k.size(1))
        if cu_seqlens_k is not None:
            _index(cu_seqlens_k, "cu_seqlens_k", q.device, sequences + 1)
    _no_grad(q, k, v)
    out = _output(out, q, k, v)
    _hip.prompt_attention(q, out, k, v, cu_seqlens, cu_seqlens_k, block_tables, context_lens, bool(causal),
                          q.size(2) ** -0.5 if scale is None else float(scale), window, sinks)
    return out
