"""Forms of the attention ops that the contract offers besides those of test_gpu_attention: contiguous int8 keys, and one sequence
that fills every workgroup, whose parts are joined in more groups than a group has members."""
import math

import pytest
import torch

import attention_ref as R
from test_gpu_attention_paths import BF16, DEV, F16, _decode, _ints, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("n", [100000, 131071])
def test_decode_all_workgroups_on_one_sequence(ops, n, quant):  # noqa: F811
    """Some 768 parts of one sequence and head: 48 groups of 16, joined at once."""
    _decode(ops, [n], 2, 1, 64, 128, F16 if quant else BF16, quant)
    if n == 100000:
        _decode(ops, [n, 3, 0], 1, 1, 128, 64, BF16, quant, window=99000, sinks=5)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [16, 64, 80, 128, 256])
def test_prompt_contiguous_int8(ops, D, dtype):  # noqa: F811
    """int8 keys and values [tokens, heads, D] with scales [tokens, heads]: ragged, with keys of their own number, out of a fused
    tensor (strides of their own), NaN in the scales of rows between the sequences."""
    print(f"[case] contiguous int8 D={D} {dtype}", flush=True)
    g = torch.Generator().manual_seed(D)
    q_lens, k_lens, Hq, Hkv = [70, 1, 0, 33, 3], [170, 257, 5, 20, 3], 4, 2
    cu_q, cu_k = [0], [0]
    for a, b in zip(q_lens, k_lens):
        cu_q.append(cu_q[-1] + a)
        cu_k.append(cu_k[-1] + b)
    n = cu_k[-1] + 10
    both = torch.randint(-127, 128, (n, 2 * Hkv, D), generator=g).to(torch.int8)
    scales = 0.002 + 0.02 * torch.rand((n, 2 * Hkv), generator=g)
    scales[cu_k[-1]:] = math.nan
    q = torch.randn((cu_q[-1] + 2, Hq, D), generator=g).to(dtype)
    real = both.double() * scales.double()[..., None]
    for window, sinks in ((0, 0), (40, 3)):
        parts = [R.attend(q[cu_q[b]:cu_q[b + 1]].double(), real[cu_k[b]:cu_k[b + 1], :Hkv], real[cu_k[b]:cu_k[b + 1], Hkv:],
                          R.visible(q_lens[b], k_lens[b], window, sinks), 1 / math.sqrt(D)) for b in range(5)]
        parts.append(R.attend(q[cu_q[-1]:].double(), real[:0, :Hkv], real[:0, Hkv:], torch.zeros((2, 0), dtype=torch.bool), 1.0))
        ref = [torch.cat(x) for x in zip(*parts)]
        kv, sc = both.to(DEV), scales.to(DEV)
        out, lse = ops.npu_prompt_attention(q.to(DEV), kv[:, :Hkv], kv[:, Hkv:], _ints(cu_q), cu_seqlens_k=_ints(cu_k),
                                            key_scale=sc[:, :Hkv], value_scale=sc[:, Hkv:], window=window, sinks=sinks)
        R.check(out, lse, ref, dtype, max(k_lens), extra_values=int(dtype == F16))
