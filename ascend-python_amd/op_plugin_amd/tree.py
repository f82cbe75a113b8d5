"""Trees of drafted tokens, as a step of decoding with drafts takes them.

A sequence's tree is its rows cu_tokens[i] .. cu_tokens[i + 1]: row 0 is the token drawn last, every other one a draft that follows
row parents[r] of its tree, a lower one.  One step, on the device throughout:

    slots, positions, missing = cache.extend(seqs, cu_tokens, total)
    seqs = torch.where(missing == 0, seqs, -1)                     # no room: nothing was added, every sequence is passed over
    mask, depth = tree_mask(parents, cu_tokens, words)             # once for all steps whose trees are alike
    positions = tree_positions(positions, cu_tokens, depth)
    x = quant_attention(..., slots, positions, ..., tree_mask=mask)  # in every layer
    sampled, logprobs = npu_sample(logits, uniform, temperature=..., top_k=..., top_p=..., min_p=...)
    path, accepted, next_tokens = cache.accept(seqs, cu_tokens, tokens, parents, sampled)
"""
from __future__ import annotations

import torch


def _sequence_of(cu_tokens: torch.Tensor, total: int) -> torch.Tensor:
    """Of each row the number of its sequence (past the last: of the last)."""
    row = torch.arange(total, device=cu_tokens.device, dtype=cu_tokens.dtype)
    return (torch.searchsorted(cu_tokens, row, right=True) - 1).clamp(0, max(cu_tokens.numel() - 2, 0))


def tree_mask(parents: torch.Tensor, cu_tokens: torch.Tensor, words: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """parents [T] int32 -> (mask [T, words] int64, depth [T] int32): bit k of a row's mask is set where row k of its tree is the
    row itself or one of its ancestors; trees of up to 64 * words rows.  A parent that is not a lower row makes a root."""
    if words < 1:
        raise ValueError(f"tree_mask: masks need a word at least, got {words}")
    if parents.dim() != 1 or cu_tokens.dim() != 1 or cu_tokens.numel() < 1:
        raise ValueError(f"tree_mask: parents must be [T] and cu_tokens [sequences + 1], got {tuple(parents.shape)} and "
                         f"{tuple(cu_tokens.shape)}")
    total = parents.numel()
    row = torch.arange(total, device=parents.device)
    if total == 0 or cu_tokens.numel() == 1:
        return parents.new_zeros((total, words), dtype=torch.int64), torch.zeros_like(parents)
    first = cu_tokens[_sequence_of(cu_tokens, total)].long()
    own = (row - first).clamp(min=0)
    up = torch.where((parents >= 0) & (parents < own), first + parents, row)
    mask = torch.where(torch.arange(words, device=parents.device) == (own // 64)[:, None],
                       torch.ones_like(own)[:, None] << (own % 64)[:, None], 0)
    depth = (up != row).to(torch.int32)
    for _ in range((64 * words - 1).bit_length()):  # twice as many ancestors each time
        mask, depth, up = mask | mask[up], depth + depth[up], up[up]
    return mask, depth


def tree_positions(positions: torch.Tensor, cu_tokens: torch.Tensor, depth: torch.Tensor) -> torch.Tensor:
    """The positions of drafted tokens, the root's and its depth further: positions as ``PagedKVCache.extend`` gave them, one
    after another (-1, of a sequence that is passed over, stays)."""
    if positions.numel() == 0 or cu_tokens.numel() == 1:
        return positions.clone()
    root = positions[cu_tokens[_sequence_of(cu_tokens, positions.numel())].long().clamp(max=positions.numel() - 1)]
    return torch.where(positions >= 0, root + depth, positions)
