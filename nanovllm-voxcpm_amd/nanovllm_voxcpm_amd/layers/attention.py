"""Attention over a paged key-value cache, as a decoder layer calls it between its q|k|v and its o linear.

Stands where the reference's ``Attention`` layer stands (nanovllm_voxcpm/layers/attention.py:53-106: store the new keys and
values by slot, then attend, prompts packed one behind the other or one new token per sequence), with the rotation, and the norms of
query and key heads where a model has them, in the launch that stores.  ``AttentionBatch`` carries what the reference
keeps in its attention context (positions are the model's own there).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn as nn

from nanovllm_voxcpm_amd.attention_ops import decode_attention, prompt_attention, rotary_table, rotate_qk


@dataclass
class AttentionBatch:
    """Where the rows of a batch stand and where their keys and values lie.

    ``positions``, ``slot_mapping``: per row, its position in its sequence and its row in the cache counted over all blocks (-1:
    not stored, for padding).  ``block_tables``, ``context_lens``: per sequence, its blocks and its keys, the batch's rows among them.
    ``cu_seqlens``: first row of every sequence and the end of the last; None when every sequence has one row (decode).  ``end_position``: one more
    than the largest position, where the host knows it; a layer refuses a batch beyond its rotary table by it.  (A position that it does not
    speak of, copied into the tensors of a captured batch, say, turns by NaN there.)
    """

    positions: torch.Tensor
    slot_mapping: torch.Tensor
    block_tables: torch.Tensor
    context_lens: torch.Tensor
    cu_seqlens: torch.Tensor | None = None
    end_position: int | None = None


def build_attention_batch(new_tokens: list[int], cached_tokens: list[int], block_tables: list[list[int]], block_size: int, *,
                          device: torch.device | str, rows: int | None = None, blocks: int | None = None) -> AttentionBatch:
    """The batch in which sequence s brings ``new_tokens[s]`` rows behind ``cached_tokens[s]`` that are in the cache already, in the blocks
    ``block_tables[s]``.  A batch of one new token each attends in the decode form.  ``rows`` and ``blocks`` pad the batch to that many
    rows and table columns (graph buffers): padding rows of a decode batch are sequences without keys, those of prompts lie behind
    the last sequence, and neither is stored."""
    sequences = len(new_tokens)
    if len(cached_tokens) != sequences or len(block_tables) != sequences:
        raise ValueError(f"{sequences} sequences with {len(cached_tokens)} cached lengths and {len(block_tables)} block tables")
    if block_size < 1:
        raise ValueError(f"block_size must be positive, got {block_size}")
    decode = all(n == 1 for n in new_tokens)
    total = sum(new_tokens)
    width = max([len(b) for b in block_tables], default=0)
    rows, blocks = total if rows is None else rows, width if blocks is None else blocks
    if rows < total or blocks < width:
        raise ValueError(f"a batch of {total} rows and {width} blocks a sequence does not fit {rows} rows and {blocks} blocks")
    positions, slots = [], []
    for s, (new, cached, table) in enumerate(zip(new_tokens, cached_tokens, block_tables)):
        if new < 0 or cached < 0:
            raise ValueError(f"sequence {s} has {new} new and {cached} cached tokens")
        if (new + cached + block_size - 1) // block_size > len(table):
            raise ValueError(f"sequence {s} of {new + cached} tokens does not fit {len(table)} blocks of {block_size}")
        for p in range(cached, cached + new):
            positions.append(p)
            slots.append(table[p // block_size] * block_size + p % block_size)
    positions += [0] * (rows - total)
    slots += [-1] * (rows - total)
    entries = rows if decode else sequences
    tables = [table + [-1] * (blocks - len(table)) for table in block_tables] + [[-1] * blocks] * (entries - sequences)
    lens = [n + c for n, c in zip(new_tokens, cached_tokens)] + [0] * (entries - sequences)
    starts = [0]
    for n in new_tokens:
        starts.append(starts[-1] + n)
    # one copy: every part of the batch is a view of it
    parts = [positions, slots, lens, [] if decode else starts, [b for table in tables for b in table]]
    packed = torch.tensor([v for part in parts for v in part], dtype=torch.int32).to(device)
    views, at = [], 0
    for part in parts:
        views.append(packed[at : at + len(part)])
        at += len(part)
    return AttentionBatch(views[0], views[1], views[4].view(entries, blocks), views[2], None if decode else views[3],
                          max([n + c for n, c in zip(new_tokens, cached_tokens) if n], default=0))


def unserved_sizes(head_size: int, rotary_dim: int | None = None) -> str:
    """What keeps the attention calls from serving these head and rotary sizes; empty where nothing does."""
    if head_size < 8 or head_size % 8 or head_size > 256:
        return f"head_size = {head_size} is not a multiple of 8 up to 256"
    rotary_dim = head_size if rotary_dim is None else rotary_dim
    if rotary_dim < 0 or rotary_dim % 16 or rotary_dim > head_size:
        return f"rotary_dim = {rotary_dim} is not a multiple of 16 up to the head size {head_size}"
    return ""


class PagedAttention(nn.Module):
    """Rotation (with per-head norms of queries and keys where ``qk_norm``), cache store and attention of one layer.

    ``window``, ``sinks``: a row sees the last ``window`` keys and the first ``sinks`` (0: all).  ``rotary_dim``: elements of a head that
    are turned, all of them by default, 0 for none; a multiple of 16, as ``head_size`` is one of 8, up to 256.  The rotary table is fp32 whatever
    the module's type and is made once per device by ``prepare``, which the first call does too if nobody did (outside
    a graph capture, then)."""

    def __init__(self, num_heads: int, num_kv_heads: int, head_size: int, *, qk_norm: bool = False, eps: float = 1e-6, window: int = 0, sinks: int = 0,
                 scale: float | None = None, rotary_dim: int | None = None, max_position: int = 4096, base: float = 10000.0, interleaved: bool = False):
        super().__init__()
        if num_kv_heads < 1 or num_heads % num_kv_heads:
            raise ValueError(f"{num_heads} query heads do not share {num_kv_heads} key-value heads evenly")
        if unserved := unserved_sizes(head_size, rotary_dim):
            raise ValueError(unserved)
        self.num_heads, self.num_kv_heads, self.head_size = num_heads, num_kv_heads, head_size
        self.eps, self.window, self.sinks, self.scale = eps, window, sinks, scale
        self.rotary_dim = head_size if rotary_dim is None else rotary_dim
        self.max_position, self.base, self.interleaved = max_position, base, interleaved
        self.q_norm = nn.Parameter(torch.ones(head_size)) if qk_norm else None
        self.k_norm = nn.Parameter(torch.ones(head_size)) if qk_norm else None
        self._tables: dict[torch.device, torch.Tensor] = {}

    def prepare(self, device: torch.device | str, table: torch.Tensor | None = None) -> torch.Tensor:
        """Make, or install, the rotary table of a device (layers of a model may share one)."""
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if table is None:
            table = self._tables.get(device)
        if table is None:
            if self.rotary_dim:
                table = rotary_table(self.rotary_dim, self.max_position, base=self.base, device=device)
            else:
                table = torch.zeros(self.max_position, 0, device=device)
        self._tables[device] = table
        return table

    def forward(self, qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, batch: AttentionBatch) -> torch.Tensor:
        """qkv [rows, (heads + 2 kv heads) * head size], caches [blocks, block size, kv heads, head size] -> [rows, heads * head size]."""
        rows, size = qkv.size(0), self.head_size
        table = self._tables.get(qkv.device)
        if table is None:
            table = self.prepare(qkv.device)
        if batch.end_position is not None and batch.end_position > table.size(0) and self.rotary_dim:
            raise ValueError(f"position {batch.end_position - 1} of the batch lies behind the {table.size(0)} positions of the layer's rotary table (max_position)")
        heads = qkv.view(rows, self.num_heads + 2 * self.num_kv_heads, size)
        q, k, v = heads.split([self.num_heads, self.num_kv_heads, self.num_kv_heads], dim=1)
        q, _ = rotate_qk(q, k, batch.positions, table, q_weight=self.q_norm, k_weight=self.k_norm, eps=self.eps, interleaved=self.interleaved,
                         v=v, k_cache=k_cache, v_cache=v_cache, slot_mapping=batch.slot_mapping)
        if batch.cu_seqlens is None:
            out = decode_attention(q, k_cache, v_cache, batch.block_tables, batch.context_lens, scale=self.scale, window=self.window, sinks=self.sinks)
        else:
            out = prompt_attention(q, k_cache, v_cache, batch.cu_seqlens, block_tables=batch.block_tables, context_lens=batch.context_lens,
                                   scale=self.scale, window=self.window, sinks=self.sinks)
        return out.view(rows, self.num_heads * size)
