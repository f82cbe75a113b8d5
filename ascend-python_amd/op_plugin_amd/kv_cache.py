"""A key-value cache in pages: the pool of every layer, and which sequence holds which pages.

The state is three int32 tensors on the device, the page table, the sequences' lengths and a count per page, which the
npu_kv_* ops change in place, so a serving loop never waits for the host: ``extend`` gives the slots that
npu_mrope_scatter_kv writes and the positions it turns by, and the table and lengths go straight to npu_paged_attention and
npu_prompt_attention.
"""
from __future__ import annotations

import torch

from . import (npu_kv_compact, npu_kv_copy_pages, npu_kv_extend, npu_kv_fork, npu_kv_free)


class PagedKVCache:
    """layers pools of num_pages pages of page_size tokens, for up to max_seqs sequences of up to max_len tokens.

    dtype float16 / bfloat16, or int8: rows as npu_dynamic_quant gives them, with an fp32 scale per token and head.
    ``keys[l]`` and ``values[l]`` are [num_pages, page_size, kv_heads, head_dim]; ``key_scales[l]`` and
    ``value_scales[l]`` [num_pages, page_size, kv_heads], or None."""

    def __init__(self, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int, max_seqs: int,
                 max_len: int, dtype: torch.dtype = torch.bfloat16, device: str | torch.device = "cuda"):
        if dtype not in (torch.float16, torch.bfloat16, torch.int8):
            raise ValueError(f"PagedKVCache: dtype must be float16, bfloat16 or int8, got {dtype}")
        self.page_size, self.num_pages = page_size, num_pages
        shape = (num_pages, page_size, kv_heads, head_dim)
        self.keys = [torch.empty(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.values = [torch.empty(shape, dtype=dtype, device=device) for _ in range(layers)]
        quant = dtype == torch.int8
        scales = lambda: torch.empty(shape[:3], dtype=torch.float32, device=device) if quant else None  # noqa: E731
        self.key_scales = [scales() for _ in range(layers)]
        self.value_scales = [scales() for _ in range(layers)]
        width = -(-max_len // page_size)
        self.block_table = torch.full((max_seqs, width), -1, dtype=torch.int32, device=device)
        self.context_lens = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self.ref_count = torch.zeros(num_pages, dtype=torch.int32, device=device)

    def _pools(self) -> list[torch.Tensor]:
        return [t for group in (self.keys, self.values, self.key_scales, self.value_scales) for t in group if t is not None]

    def extend(self, seqs: torch.Tensor, cu_tokens: torch.Tensor, total: int):
        """Room for cu_tokens[i + 1] - cu_tokens[i] new tokens of seqs[i]: (slots, positions, missing).  missing is 0 on the
        device, or how many pages or table columns are missing: then nothing has changed and every slot is -1."""
        return npu_kv_extend(self.block_table, self.context_lens, self.ref_count, seqs, cu_tokens, total, self.page_size)

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> torch.Tensor:
        """children[i] becomes a copy of parents[i]: whole pages are shared, a started last page is copied."""
        return npu_kv_fork(self._pools(), self.block_table, self.context_lens, self.ref_count, parents, children,
                           self.page_size)

    def free(self, seqs: torch.Tensor) -> None:
        npu_kv_free(self.block_table, self.context_lens, self.ref_count, seqs, self.page_size)

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        npu_kv_copy_pages(self._pools(), src, dst)

    def rows(self, seqs: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """The page table's rows and the lengths of seqs, as the attention ops take them.  A sequence number that the other
        calls pass over (negative, or max_seqs and more: a batch's padding) has no tokens."""
        if self.context_lens.numel() == 0:
            return self.block_table.new_full((seqs.numel(), self.block_table.shape[1]), -1), self.context_lens.new_zeros(seqs.numel())
        held = seqs.clamp(0, self.context_lens.numel() - 1)
        at = held.long()
        return self.block_table[at], self.context_lens[at].masked_fill_(held != seqs, 0)

    def compact(self) -> torch.Tensor:
        """Moves the pages in use to the front of the pool; how many moved, on the device."""
        table, count, moved = npu_kv_compact(self._pools(), self.block_table, self.ref_count)
        # into the tensors that captured graphs and other holders of the state read
        self.block_table.copy_(table)
        self.ref_count.copy_(count)
        return moved
