"""The quantized attention block of a decoder layer over a paged cache, built from the torch.ops.npu ops: what stands before
the MLP block of mlp.py.

    y, s    = RMSNorm(x; gamma, eps) -> per-token int8           npu_rms_norm_dynamic_quant
    q, k, v = W8A8(y, W_qkv; s, s_qkv)                           npu_quant_matmul
    q       = rotated q; rotated k and v into the cache          npu_mrope_scatter_kv
    o       = attention over the cache                           npu_prompt_attention, npu_paged_attention (one token each),
                                                                 or npu_tree_attention (trees of drafted tokens)
    out     = W8A8(int8(o), W_o; s_o)                            npu_dynamic_quant, npu_quant_matmul

q, k and v stay views of the projection's output.
"""
from __future__ import annotations

import torch

from . import (npu_dynamic_quant, npu_mrope_scatter_kv, npu_paged_attention, npu_prompt_attention, npu_quant_matmul,
               npu_rms_norm_dynamic_quant, npu_tree_attention)
from .kv_cache import PagedKVCache


def quant_attention(x: torch.Tensor, gamma: torch.Tensor, w_qkv: torch.Tensor, s_qkv: torch.Tensor, w_o: torch.Tensor,
                    s_o: torch.Tensor, cache: PagedKVCache, layer: int, seqs: torch.Tensor, cu_tokens: torch.Tensor | None,
                    slots: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, q_heads: int, *,
                    rows: tuple[torch.Tensor, torch.Tensor] | None = None, sections: list[int] | None = None,
                    rotary_mode: str = "half", window: int = 0, sinks: int = 0, eps: float = 1e-6,
                    tree_mask: torch.Tensor | None = None) -> torch.Tensor:
    """x [T, H] fp16/bf16: the new tokens of sequences ``seqs``, cu_tokens[i] .. cu_tokens[i + 1] of the i-th; cu_tokens
    None: one token each.  slots and positions as ``cache.extend`` gave them (positions [axes, T] with ``sections`` for
    images and video), once for all layers, and so is rows, ``cache.rows(seqs)`` after ``extend`` (None: taken here, in
    every layer again).  A sequence number that ``extend`` passes over sees nothing: its rows are 0.
    tree_mask: the rows of each sequence are a tree of drafted tokens (tree.tree_mask; positions by tree.tree_positions),
    with cu_tokens.
    w_qkv int8 [H, (q_heads + 2 * kv_heads) * head_dim], w_o int8 [q_heads * head_dim, H], as quant_mlp takes its
    weights.  -> [T, H]."""
    if tree_mask is not None and cu_tokens is None:
        raise ValueError("quant_attention: trees of drafted tokens need cu_tokens")
    kv_heads, head_dim = cache.keys[layer].shape[2:]
    y, s, _ = npu_rms_norm_dynamic_quant(x, gamma, eps)
    qkv = npu_quant_matmul(y, w_qkv, s_qkv, pertoken_scale=s, output_dtype=x.dtype)
    q, k, v = qkv.view(x.shape[0], q_heads + 2 * kv_heads, head_dim).split([q_heads, kv_heads, kv_heads], dim=1)
    scales = dict(key_scale=cache.key_scales[layer], value_scale=cache.value_scales[layer])
    q = npu_mrope_scatter_kv(positions, q, k, v, cos_sin, cache.keys[layer], cache.values[layer], slots,
                             mrope_section=sections, rotary_mode=rotary_mode, **scales)
    table, lens = rows if rows is not None else cache.rows(seqs)
    if tree_mask is not None:
        o, _ = npu_tree_attention(q, cache.keys[layer], cache.values[layer], cu_tokens, table, lens, tree_mask, window=window,
                                  sinks=sinks, **scales)
    elif cu_tokens is None:
        o, _ = npu_paged_attention(q, cache.keys[layer], cache.values[layer], table, lens, window=window, sinks=sinks, **scales)
    else:
        o, _ = npu_prompt_attention(q, cache.keys[layer], cache.values[layer], cu_tokens, block_table=table,
                                    context_lens=lens, window=window, sinks=sinks, **scales)
    y, s = npu_dynamic_quant(o.view(x.shape[0], q_heads * head_dim))
    return npu_quant_matmul(y, w_o, s_o, pertoken_scale=s, output_dtype=x.dtype)
