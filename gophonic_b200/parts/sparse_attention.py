"""Grouped-query causal attention that reads a part of the paged cache.

The layer is ``Attention`` with the same tensors.  Beside its keys the cache keeps the lowest and highest value of every key
channel of each full page of 64 tokens; a token takes from them, for each kv head, the pages whose keys could score highest
(``PageSelection``: how many, and which are always read) and attends to those alone, so what a token costs stops growing
with its context beyond them.  While every page would be listed, the layer runs as ``Attention`` does, bit for bit.
"""
from __future__ import annotations

from typing import Mapping

import torch

from .attention import Attention
from .base import KVRequest, Runtime


class SparseAttention(Attention):
    @classmethod
    def cache_request(cls, spec):
        return KVRequest(kv_heads=spec.kv_heads, head_dim=spec.head_dim, bounds=True)

    def __init__(self, spec, prefix: str, tensors: Mapping[str, torch.Tensor], runtime: Runtime):
        if spec.selection is None or spec.window:
            raise ValueError(f"{prefix}: attention that selects pages needs a page selection and has no window")
        super().__init__(spec, prefix, tensors, runtime)
        ops, d, sel = runtime.ops, spec.head_dim, spec.selection
        if not ops.page_attention_accepts(runtime.act_dtype, d):
            raise ValueError(f"{prefix}: no kernel attends to selected pages with heads of {d} in {runtime.act_dtype}")
        if sel.pages > ops.MAX_LISTED_PAGES:
            raise ValueError(f"{prefix}: {sel.pages} pages a token, at most {ops.MAX_LISTED_PAGES}")

    def prepare(self, capacity: int) -> None:
        if capacity > 64 * self.rt.ops.MAX_SELECTABLE_PAGES:
            raise ValueError(f"pages are selected of up to {64 * self.rt.ops.MAX_SELECTABLE_PAGES} tokens a sequence, the cache has room for {capacity}")
        super().prepare(capacity)

    def selects(self, max_q_len: int, max_kv_len: int) -> bool:
        sel = self.spec.selection
        return max_kv_len > 64 * sel.pages and (sel.prompts or max_q_len == 1)

    def plan(self, nseq: int, max_q_len: int, max_kv_len: int, sm_count: int):
        """Whether the step's rows select, else ``Attention``'s plan."""
        if self.selects(max_q_len, max_kv_len):
            return "selected pages"
        return super().plan(nseq, max_q_len, max_kv_len, sm_count)

    def key_splits(self, batch):
        if batch.plan_for(self) == "selected pages":     # rows of runs, a row a pass, which read everything
            return 1, None
        return super().key_splits(batch)

    def who_selects(self, batch):
        """Which sequences' rows select: True for all, False for none, else (their rows, the other sequences' rows) as numbers of rows a
        sequence.  A sequence's answer does not follow from the others': unless ``prompts``, those that bring a single token select,
        also beside the runs of others, and a run's rows do not, also where a pass holds one of them."""
        limit, runs = 64 * self.spec.selection.pages, not self.spec.selection.prompts
        if batch.plan_for(self) == "selected pages" and not (runs and batch.singles is not None and not all(batch.singles)):
            return True
        if not runs or batch.singles is None or batch.max_kv_len <= limit:
            return False
        key = ("single tokens that select", limit)      # every layer has the same answer
        if key not in batch.shared:
            some = [int(single and past + rows > limit) for single, (past, rows) in zip(batch.singles, batch.extents)]
            mine = torch.tensor(some, dtype=torch.int32, device=batch.seq_q_len.device) if any(some) else None
            batch.shared[key] = False if mine is None else (mine, batch.seq_q_len - mine)
        return batch.shared[key]

    def _attend(self, batch, qkv: torch.Tensor, cache) -> torch.Tensor:
        ops, s = self.rt.ops, self.spec
        who = self.who_selects(batch)
        # The pages that a run of tokens fills: its own later tokens may select them, and those of later steps will.  Single tokens
        # leave them to the end of the step (``Cache.keep_bounds``).
        fills = batch.max_q_len > 1 and cache is not None and cache.writable
        if who is False:
            ctx = super()._attend(batch, qkv, cache)
            if fills:
                self._bounds(batch, cache)
            return ctx
        if cache is None:
            raise ValueError("attention needs a key/value cache plane")
        if cache.k.dtype != qkv.dtype:
            raise ValueError(f"attention: cache holds {cache.k.dtype}, activations are {qkv.dtype}")
        rows, sel = qkv.shape[0], s.selection
        cos, sin, rot = self.position.kernel_args()
        ops.qk_norm_rope_kv_write(qkv, s.heads, s.kv_heads, s.head_dim, self.q_norm, self.k_norm, self.eps, cos, sin, rot, batch.row_pos,
                                  batch.row_seq, batch.seq_slot, cache.block_table, cache.k, cache.v, cache.writable)
        if fills:
            self._bounds(batch, cache)
        q = qkv[:, :self.q_dim]
        pages = batch.workspace(("selected pages", s.kv_heads, sel.pages), rows * s.kv_heads * sel.pages, torch.int32)
        pages = pages[:rows * s.kv_heads * sel.pages].view(rows, s.kv_heads, sel.pages)
        ctx = torch.empty((rows, self.q_dim), dtype=qkv.dtype, device=qkv.device)
        heads = (s.heads, s.kv_heads, s.head_dim)
        q_len, max_q_len = batch.seq_q_len, batch.max_q_len
        if who is not True:
            q_len, others = who
            # (rows of single tokens are left as they are, or, where all rows of a pass are single ones, written by both, these first)
            ops.attention(q, ctx, cache.k, cache.v, cache.block_table, batch.seq_slot, batch.seq_q_start, others, batch.seq_kv_len, batch.nseq,
                          max_q_len, *heads, float(s.scale))
            max_q_len = 1
        seqs = (batch.seq_slot, batch.seq_q_start, q_len, batch.seq_kv_len, batch.nseq, max_q_len)
        ops.select_pages(q, cache.bounds, cache.block_table, *seqs, *heads, pages, sel.first, sel.last)
        ops.attention_pages(q, ctx, cache.k, cache.v, cache.block_table, *seqs, *heads, float(s.scale), pages)
        return ctx

    def _bounds(self, batch, cache) -> None:
        self.rt.ops.page_bounds(cache.k, cache.bounds, cache.block_table, batch.seq_slot, batch.seq_q_len, batch.seq_kv_len, batch.nseq, batch.max_q_len)
