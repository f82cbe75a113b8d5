"""op_plugin_amd -- MI355X (gfx950) quantized-inference ops behind the torch_npu op names.

Importing this package loads ``_npu_ops.so``, which registers

* ``torch.ops.npu.npu_dynamic_quant(input, *, smooth_scales=None) -> (int8 y, fp32 scale)``
* ``torch.ops.npu.npu_quant_matmul(x1, x2, scale, *, offset=None, pertoken_scale=None,
  bias=None, output_dtype=None) -> Tensor``  (W8A8)
* ``torch.ops.npu.npu_weight_quant_batchmatmul(x, weight, antiquant_scale,
  antiquant_offset=None, quant_scale=None, quant_offset=None, bias=None,
  antiquant_group_size=0) -> Tensor``  (W4A16 / W8A16)
* ``torch.ops.npu.npu_convert_weight_to_int4pack(weight, inner_k_tiles=0) -> Tensor``
  (``inner_k_tiles=4``: straight to the NZ layout)
* ``torch.ops.npu.npu_format_cast(self, acl_format) -> Tensor``: an int4-packed or int8 weight between ND (2)
  and FRACTAL_NZ (29), the MFMA-tiled layouts ``npu_weight_quant_batchmatmul`` streams fastest
* ``torch.ops.npu.quantize_per_tensor(self, scale, zero_point, dtype)``,
  ``torch.ops.npu.quantize_per_channel(self, scales, zero_points, axis, dtype)`` and
  ``torch.ops.npu.dequantize(self)``: the reference's static quantization ops (plain int8 / uint8 / int32
  results for torch.qint8 / quint8 / qint32; dequantize is their cast to float32)
* ``torch.ops.npu.npu_rms_norm(self, gamma, epsilon=1e-6) -> (y, fp32 rstd)``
* ``torch.ops.npu.npu_swiglu(self, dim=-1) -> Tensor``
* ``torch.ops.npu.npu_rms_norm_dynamic_quant(self, gamma, epsilon=1e-6) -> (int8 q, fp32 scale, fp32 rstd)``
  and ``torch.ops.npu.npu_swiglu_dynamic_quant(self, dim=-1) -> (int8 q, fp32 scale)``: RMSNorm / SwiGLU
  fused with npu_dynamic_quant of their 16-bit output (bit-identical to the unfused chain)
* ``torch.ops.npu.npu_quant_matmul_swiglu(x1, x2, scale, *, pertoken_scale=None, output_dtype=None) -> h``: the
  quantized MLP block's gate-up projection with the SwiGLU in the GEMM's epilogue, h =
  npu_swiglu(npu_quant_matmul(x1, x2, scale, pertoken_scale=..., output_dtype=...)) bit for bit (x2 [K, 2I] or
  its int8 NZ cast; no bias)
* ``torch.ops.npu.npu_quant_matmul_swiglu_quant(x1, x2, scale, *, pertoken_scale=None, output_dtype=None) -> (q,
  scale)``: the same followed by npu_dynamic_quant of h, bit for bit; the GEMM's epilogue stores each row's
  partial absmax, so the quantizer reads h once with no row reduction
* attention over a paged key-value cache (index tensors are int32 on the device):
  ``torch.ops.npu.npu_paged_attention(query, key_cache, value_cache, block_table, context_lens, *, key_scale=None,
  value_scale=None, scale=None, window=0, sinks=0) -> (out, lse)`` (one new token per sequence),
  ``torch.ops.npu.npu_prompt_attention(query, key, value, cu_seqlens_q, *, cu_seqlens_k=None, block_table=None,
  context_lens=None, key_scale=None, value_scale=None, scale=None, window=0, sinks=0) -> (out, lse)`` (ragged prompts or
  prompt chunks, causal, keys contiguous or paged),
  ``torch.ops.npu.npu_tree_attention(query, key_cache, value_cache, cu_seqlens_q, block_table, context_lens, tree_mask, *,
  key_scale=None, value_scale=None, scale=None, window=0, sinks=0) -> (out, lse)`` (trees of drafted tokens: a row sees the
  context and the rows of its own tree whose bits its mask [tokens, words] int64 has set)
* ``torch.ops.npu.npu_mrope(positions, query, key, cos_sin_cache, *, mrope_section=None, rotary_mode="half") -> (query,
  key)`` and ``torch.ops.npu.npu_mrope_scatter_kv(positions, query, key, value, cos_sin_cache, key_cache, value_cache,
  slot_mapping, *, key_scale=None, value_scale=None, mrope_section=None, rotary_mode="half") -> query``: rotary
  positions of one to four axes, alone or with the write into the cache (int8 with scales per token and head)
* the cache's pages: ``npu_kv_extend``, ``npu_kv_fork``, ``npu_kv_free``, ``npu_kv_copy_pages``, ``npu_kv_compact``
  (``op_plugin_amd.kv_cache.PagedKVCache`` holds their state), and ``torch.ops.npu.npu_kv_accept(caches, block_table,
  context_lens, ref_count, seqs, cu_tokens, tokens, parents, sampled, page_size) -> (path, accepted, next_tokens)``: of trees
  of drafted tokens the way that was drawn stays in the cache
* ``torch.ops.npu.npu_sample(logits, uniform, *, temperature=None, top_k=None, top_p=None, min_p=None) -> (tokens,
  logprobs)``: a token per row of logits from given uniform numbers, with settings per row

and exposes the same callables here, so code written as
``torch_npu.npu_quant_matmul(...)`` runs as ``op_plugin_amd.npu_quant_matmul(...)``
(the reference tests call ops this way, e.g.
test/test_custom_ops/test_npu_rms_norm.py:20).  The kernels are the HIP code of
``libqk_hip.so``; there is no fallback: if the native library is missing, the
import fails.
"""
from __future__ import annotations

import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libqk_hip.so")
OPS_PATH = os.path.join(_HERE, "_npu_ops.so")

if not (os.path.exists(LIB_PATH) and os.path.exists(OPS_PATH)):
    raise ImportError(
        "op_plugin_amd: native libraries are not built (expected "
        f"{LIB_PATH} and {OPS_PATH}); run `python ascend-python_amd/build.py` or "
        "`__graft_entry__.build()` first")

if not hasattr(torch.ops.npu, "npu_quant_matmul"):
    torch.ops.load_library(OPS_PATH)

npu_dynamic_quant = torch.ops.npu.npu_dynamic_quant
npu_quant_matmul = torch.ops.npu.npu_quant_matmul
npu_weight_quant_batchmatmul = torch.ops.npu.npu_weight_quant_batchmatmul
npu_convert_weight_to_int4pack = torch.ops.npu.npu_convert_weight_to_int4pack
npu_format_cast = torch.ops.npu.npu_format_cast
quantize_per_tensor = torch.ops.npu.quantize_per_tensor
quantize_per_channel = torch.ops.npu.quantize_per_channel
dequantize = torch.ops.npu.dequantize
npu_rms_norm = torch.ops.npu.npu_rms_norm
npu_swiglu = torch.ops.npu.npu_swiglu
npu_rms_norm_dynamic_quant = torch.ops.npu.npu_rms_norm_dynamic_quant
npu_swiglu_dynamic_quant = torch.ops.npu.npu_swiglu_dynamic_quant
npu_quant_matmul_swiglu = torch.ops.npu.npu_quant_matmul_swiglu
npu_quant_matmul_swiglu_quant = torch.ops.npu.npu_quant_matmul_swiglu_quant
npu_paged_attention = torch.ops.npu.npu_paged_attention
npu_prompt_attention = torch.ops.npu.npu_prompt_attention
npu_tree_attention = torch.ops.npu.npu_tree_attention
npu_mrope = torch.ops.npu.npu_mrope
npu_mrope_scatter_kv = torch.ops.npu.npu_mrope_scatter_kv
npu_kv_copy_pages = torch.ops.npu.npu_kv_copy_pages
npu_kv_fork = torch.ops.npu.npu_kv_fork
npu_kv_free = torch.ops.npu.npu_kv_free
npu_kv_extend = torch.ops.npu.npu_kv_extend
npu_kv_compact = torch.ops.npu.npu_kv_compact
npu_kv_accept = torch.ops.npu.npu_kv_accept
npu_sample = torch.ops.npu.npu_sample

# qk_abi.h constants
QK_F16, QK_BF16, QK_F32, QK_I8, QK_I32, QK_U8, QK_I4_NZ, QK_I8_NZ, QK_I8_NK = 1, 2, 3, 4, 5, 6, 16, 17, 18
ACL_FORMAT_ND, ACL_FORMAT_FRACTAL_NZ = 2, 29
QK_OK, QK_ERR_ARG, QK_ERR_UNSUPPORTED, QK_ERR_WORKSPACE, QK_ERR_LAUNCH = 0, -1, -2, -3, -4
QK_NOALLOC_SCRATCH_BYTES = 16 << 20

ABI_SYMBOLS = (
    "qk_last_error", "qk_abi_version", "qk_debug_set_plan", "qk_dynamic_quant", "qk_quant_matmul_workspace_size",
    "qk_quant_matmul", "qk_quant_matmul_nz_workspace_size", "qk_quant_matmul_nz", "qk_weight_quant_bmm_workspace_size",
    "qk_weight_quant_bmm", "qk_weight_quant_bmm_noalloc", "qk_int4_pack", "qk_weight_format_cast",
    "qk_quantize_per_tensor", "qk_quantize_per_channel", "qk_dequantize", "qk_rms_norm", "qk_rms_norm_quant",
    "qk_swiglu", "qk_swiglu_quant", "qk_quant_matmul_swiglu", "qk_quant_matmul_swiglu_quant_workspace_size",
    "qk_quant_matmul_swiglu_quant", "qk_paged_attention_workspace_size", "qk_paged_attention",
    "qk_prompt_attention_workspace_size", "qk_prompt_attention", "qk_tree_attention_workspace_size", "qk_tree_attention",
    "qk_mrope", "qk_kv_copy_pages",
    "qk_kv_fork_workspace_size", "qk_kv_fork", "qk_kv_free", "qk_kv_extend_workspace_size", "qk_kv_extend",
    "qk_kv_compact_workspace_size", "qk_kv_compact", "qk_kv_accept_workspace_size",
    "qk_kv_accept", "qk_sample_workspace_size", "qk_sample",
)


class KvCache(ctypes.Structure):
    """qk_kv_cache: the keys and values of one layer, as the C ABI takes them (strides in elements)."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("key", "value", "key_scale", "value_scale")] + \
               [(n, ctypes.c_int64) for n in (
                   "num_pages", "page_size", "kv_heads", "head_dim", "key_page_stride", "key_token_stride",
                   "key_head_stride", "value_page_stride", "value_token_stride", "value_head_stride",
                   "key_scale_page_stride", "key_scale_token_stride", "key_scale_head_stride",
                   "value_scale_page_stride", "value_scale_token_stride", "value_scale_head_stride")] + \
               [("dtype", ctypes.c_int)]


class Rows(ctypes.Structure):
    """qk_rows: where the rows of a cache tensor's tokens lie, in bytes."""
    _fields_ = [("base", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in (
        "page_stride", "token_stride", "piece_stride", "pieces", "piece_bytes")]


class Pages(ctypes.Structure):
    """qk_pages: a cache tensor as pages of page_bytes bytes, page_stride bytes apart."""
    _fields_ = [("base", ctypes.c_void_p), ("page_stride", ctypes.c_int64), ("page_bytes", ctypes.c_int64)]


_abi = None


def abi() -> ctypes.CDLL:
    """ctypes handle on libqk_hip.so with argtypes set (the C ABI of include/qk_abi.h)."""
    global _abi
    if _abi is None:
        L = ctypes.CDLL(LIB_PATH)
        P, I64, I, SZ = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t
        L.qk_last_error.restype = ctypes.c_char_p
        L.qk_last_error.argtypes = []
        L.qk_abi_version.restype = I
        L.qk_debug_set_plan.argtypes = [ctypes.c_char_p]
        L.qk_dynamic_quant.argtypes = [P, I, I64, I64, P, P, P, P]
        L.qk_quant_matmul_workspace_size.argtypes = [I64, I64, I64, I, ctypes.POINTER(SZ)]
        L.qk_quant_matmul.argtypes = [P, I64, P, I64, I64, I64, I64, I64, P, I64, P, I64, P, P, I, P, I, P, SZ, P]
        L.qk_quant_matmul_nz_workspace_size.argtypes = [I64, I64, I64, I, ctypes.POINTER(SZ)]
        L.qk_quant_matmul_nz.argtypes = [P, I64, P, I64, I64, I64, P, I64, P, I64, P, P, I, P, I, P, SZ, P]
        L.qk_weight_quant_bmm_workspace_size.argtypes = [I64, I64, I64, I, I64, ctypes.POINTER(SZ)]
        L.qk_weight_quant_bmm.argtypes = [P, I, P, I, P, P, I, I64, I64, I64, I64, P, I, P, I, P, SZ, P]
        L.qk_weight_quant_bmm_noalloc.argtypes = [P, I, P, I, P, P, I, I64, I64, I64, I64, P, I, P, I, P]
        L.qk_int4_pack.argtypes = [P, I, I64, I64, P, P]
        L.qk_weight_format_cast.argtypes = [P, I, P, I, I, I64, I64, P]
        L.qk_quantize_per_tensor.argtypes = [P, I, I64, ctypes.c_float, I64, P, I, P]
        L.qk_quantize_per_channel.argtypes = [P, I, I64, I64, I64, P, P, P, I, P]
        L.qk_dequantize.argtypes = [P, I, I64, P, P]
        F = ctypes.c_float
        L.qk_rms_norm.argtypes = [P, I, P, I64, I64, F, P, P, P]
        L.qk_rms_norm_quant.argtypes = [P, I, P, I64, I64, F, P, P, P, P]
        L.qk_swiglu.argtypes = [P, I, I64, I64, P, P]
        L.qk_swiglu_quant.argtypes = [P, I, I64, I64, P, P, P]
        L.qk_quant_matmul_swiglu.argtypes = [P, I64, P, I, I64, I64, I64, I64, P, I64, P, P, I, P]
        L.qk_quant_matmul_swiglu_quant_workspace_size.argtypes = [I64, I64, P]
        L.qk_quant_matmul_swiglu_quant.argtypes = [P, I64, P, I, I64, I64, I64, I64, P, I64, P, I, P, P, P, SZ, P]
        C, G, Z = ctypes.POINTER(KvCache), ctypes.POINTER(Pages), ctypes.POINTER(SZ)
        L.qk_paged_attention_workspace_size.argtypes = [I64, I64, C, I64, I64, I64, Z]
        L.qk_paged_attention.argtypes = [P, I, I64, I64, I64, I64, C, P, I64, I64, P, F, I64, I64, P, P, P, SZ, P]
        L.qk_prompt_attention_workspace_size.argtypes = [I64, I64, I64, C, I64, I64, I64, Z]
        L.qk_prompt_attention.argtypes = [P, I, I64, I64, I64, I64, I64, P, C, P, P, I64, I64, P, F, I64, I64, P, P, P,
                                          SZ, P]
        L.qk_tree_attention_workspace_size.argtypes = [I64, I64, I64, C, I64, I64, I64, Z]
        L.qk_tree_attention.argtypes = [P, I, I64, I64, I64, I64, I64, P, C, P, I64, I64, P, P, I64, I64, F, I64, I64, P, P,
                                        P, SZ, P]
        L.qk_mrope.argtypes = [P, P, P, I] + [I64] * 10 + [P, I64, I64, P, P, I, I64, I64, I, P, P, C, P, P]
        L.qk_kv_copy_pages.argtypes = [G, I64, I64, P, P, I64, P]
        L.qk_kv_fork_workspace_size.argtypes = [I64, Z]
        L.qk_kv_fork.argtypes = [G, I64, I64, I64, P, I64, I64, I64, P, P, P, P, I64, P, P, SZ, P]
        L.qk_kv_free.argtypes = [I64, I64, P, I64, I64, I64, P, P, P, I64, P]
        L.qk_kv_extend_workspace_size.argtypes = [I64, I64, Z]
        L.qk_kv_extend.argtypes = [I64, I64, P, I64, I64, I64, P, P, P, P, I64, I64, P, P, P, P, SZ, P]
        L.qk_kv_compact_workspace_size.argtypes = [I64, Z]
        L.qk_kv_compact.argtypes = [G, I64, I64, P, I64, I64, I64, P, P, P, P, P, SZ, P]
        L.qk_kv_accept.argtypes = [ctypes.POINTER(Rows), I64, I64, I64, P, I64, I64, I64, P, P, P, P, I64, I64, P, P, P, P, P, P,
                                   P, SZ, P]
        L.qk_kv_accept_workspace_size.argtypes = [I64, Z]
        L.qk_sample_workspace_size.argtypes = [I64, I64, I, Z]
        L.qk_sample.argtypes = [P, I, I64, I64, I64, P, P, P, P, P, P, P, P, SZ, P]
        for name in ABI_SYMBOLS:
            getattr(L, name).restype = I if name != "qk_last_error" else ctypes.c_char_p
        _abi = L
    return _abi


def get_npu_format(t: torch.Tensor) -> int:
    """Storage format of a tensor, as torch_npu.get_npu_format reports it: FRACTAL_NZ (29) for a weight that
    npu_format_cast(w, 29) or npu_convert_weight_to_int4pack(w, inner_k_tiles=4) returned (the format is recorded
    with its storage, not inferred from the shape), ND (2) for every other tensor."""
    return int(torch.ops.npu.get_npu_format(t))


def last_error() -> str:
    return abi().qk_last_error().decode()


def debug_set_plan(spec: str = "") -> None:
    """Force kernel choices of the planners (tests and tuning only; "" restores the planners' choices).

    Spec grammar: see PlanOverride in csrc/kernels/common.h, e.g. "w4_gemm=force" or
    "w4_stream=8:4:2,skinny_splits=4"."""
    rc = abi().qk_debug_set_plan(spec.encode())
    if rc != 0:
        raise ValueError(last_error())


__all__ = [
    "npu_dynamic_quant", "npu_quant_matmul", "npu_weight_quant_batchmatmul",
    "npu_convert_weight_to_int4pack", "npu_format_cast", "get_npu_format", "quantize_per_tensor",
    "quantize_per_channel", "dequantize", "npu_rms_norm", "npu_swiglu", "npu_rms_norm_dynamic_quant",
    "npu_swiglu_dynamic_quant", "npu_quant_matmul_swiglu", "npu_quant_matmul_swiglu_quant", "npu_paged_attention",
    "npu_prompt_attention", "npu_tree_attention", "npu_mrope", "npu_mrope_scatter_kv", "npu_kv_copy_pages", "npu_kv_fork", "npu_kv_free",
    "npu_kv_extend", "npu_kv_compact", "npu_kv_accept", "npu_sample", "abi", "last_error", "debug_set_plan", "LIB_PATH", "OPS_PATH",
]
