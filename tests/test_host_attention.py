"""Host side of the attention and cache ops, no GPU: schemas, shape inference and refusals (Meta tensors), the C ABI's checks
before any launch, the division by a page's size, and the oracle of the GPU tests against torch on small cases."""
import ctypes
import math
import random

import pytest
import torch

import attention_ref as R
import op_plugin_amd as q

BF16, F16, I8, I32 = torch.bfloat16, torch.float16, torch.int8, torch.int32


def _m(shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="meta")


def _cache(P=10, S=16, H=2, D=64, dtype=BF16):
    return _m((P, S, H, D), dtype), _m((P, S, H, D), dtype)


def test_registered():
    for name in ("npu_paged_attention", "npu_prompt_attention", "npu_mrope", "npu_mrope_scatter_kv", "npu_kv_copy_pages",
                 "npu_kv_fork", "npu_kv_free", "npu_kv_extend", "npu_kv_compact"):
        assert getattr(q, name) is getattr(torch.ops.npu, name) and name in q.__all__


def test_meta_shapes():
    k, v = _cache()
    out, lse = q.npu_paged_attention(_m((3, 8, 64)), k, v, _m((3, 5), I32), _m((3,), I32))
    assert out.shape == (3, 8, 64) and out.dtype == BF16 and lse.shape == (3, 8) and lse.dtype == torch.float32
    out, lse = q.npu_prompt_attention(_m((30, 8, 64)), _m((30, 2, 64)), _m((30, 2, 64)), _m((4,), I32), window=4, sinks=1)
    assert out.shape == (30, 8, 64) and lse.shape == (30, 8)
    k8, v8 = _cache(dtype=I8)
    s = _m((10, 16, 2), torch.float32)
    out, _ = q.npu_prompt_attention(_m((30, 8, 64)), k8, v8, _m((4,), I32), block_table=_m((3, 5), I32),
                                    context_lens=_m((3,), I32), key_scale=s, value_scale=s)
    assert out.shape == (30, 8, 64)
    a, b = q.npu_mrope(_m((3, 7), I32), _m((7, 4, 64)), _m((7, 2, 64)), _m((100, 64), torch.float32), mrope_section=[8, 12, 12])
    assert a.shape == (7, 4, 64) and b.shape == (7, 2, 64)
    a = q.npu_mrope_scatter_kv(_m((7,), I32), _m((7, 4, 64)), _m((7, 2, 64)), _m((7, 2, 64)), _m((100, 32), BF16), k, v,
                               _m((7,), I32), rotary_mode="interleave")
    assert a.shape == (7, 4, 64)
    t, n, c = _m((6, 5), I32), _m((6,), I32), _m((10,), I32)
    assert q.npu_kv_fork([k, v], t, n, c, _m((2,), I32), _m((2,), I32), 16).shape == (1,)
    q.npu_kv_free(t, n, c, _m((2,), I32), 16)
    slots, positions, missing = q.npu_kv_extend(t, n, c, _m((2,), I32), _m((3,), I32), 9, 16)
    assert slots.shape == positions.shape == (9,) and missing.shape == (1,)
    a, b, moved = q.npu_kv_compact([k, v], t, c)
    assert a.shape == (6, 5) and b.shape == (10,) and moved.shape == (1,)
    q.npu_kv_copy_pages([k, v], _m((3,), I32), _m((3,), I32))


def _refuses(call, text):
    with pytest.raises(RuntimeError, match=text):
        call()


def test_paged_attention_refusals():
    k, v = _cache()
    t, n = _m((3, 5), I32), _m((3,), I32)
    good = dict(query=_m((3, 8, 64)), key_cache=k, value_cache=v, block_table=t, context_lens=n)
    call = lambda **kw: q.npu_paged_attention(**{**good, **kw})  # noqa: E731
    call()
    _refuses(lambda: call(query=_m((3, 8, 64), torch.float32)), "float16 or bfloat16")
    _refuses(lambda: call(query=_m((3, 512))), "tokens, heads, head_dim")
    _refuses(lambda: call(query=_m((3, 8, 32))), "one head_dim")
    _refuses(lambda: call(query=_m((3, 7, 64))), "multiple of the keys'")
    _refuses(lambda: call(query=_m((4, 8, 64))), "one row per query")
    _refuses(lambda: call(query=_m((3, 8, 64), F16)), "int8 or Half")
    _refuses(lambda: call(value_cache=_m((10, 16, 2, 32))), "one shape")
    _refuses(lambda: call(value_cache=_m((10, 16, 2, 64), F16)), "one dtype")
    _refuses(lambda: call(key_cache=_m((10, 16, 128)), value_cache=_m((10, 16, 128))), "pages, page_size, heads")
    _refuses(lambda: call(key_cache=_m((10, 0, 2, 64)), value_cache=_m((10, 0, 2, 64))), "at least one token")
    _refuses(lambda: call(block_table=_m((3, 5), torch.int64)), "block_table must be int32")
    _refuses(lambda: call(context_lens=_m((3, 1), I32)), "context_lens must have 1")
    _refuses(lambda: call(context_lens=torch.zeros(3, dtype=I32)), "context_lens must be on")
    _refuses(lambda: call(window=-1), "must not be negative")
    _refuses(lambda: call(sinks=-1), "must not be negative")
    _refuses(lambda: call(scale=math.inf), "scale must be finite")
    _refuses(lambda: call(key_scale=_m((10, 16, 2), torch.float32)), "go with int8")
    k8, v8 = _cache(dtype=I8)
    _refuses(lambda: call(key_cache=k8, value_cache=v8), "go with int8")
    s = _m((10, 16, 2), torch.float32)
    call(key_cache=k8, value_cache=v8, key_scale=s, value_scale=s)
    _refuses(lambda: call(key_cache=k8, value_cache=v8, key_scale=s, value_scale=_m((10, 16, 1), torch.float32)), "must be float32")
    _refuses(lambda: call(key_cache=k.transpose(2, 3), value_cache=v.transpose(2, 3)), "last dimension")


def test_prompt_attention_refusals():
    k, v = _cache()
    good = dict(query=_m((30, 8, 64)), key=_m((30, 2, 64)), value=_m((30, 2, 64)), cu_seqlens_q=_m((4,), I32))
    call = lambda **kw: q.npu_prompt_attention(**{**good, **kw})  # noqa: E731
    call()
    _refuses(lambda: call(block_table=_m((3, 5), I32)), "go together")
    _refuses(lambda: call(cu_seqlens_k=_m((4,), I32), block_table=_m((3, 5), I32), context_lens=_m((3,), I32)), "either paged")
    _refuses(lambda: call(key=k, value=v), "tokens, heads, head_dim")
    _refuses(lambda: call(key=k, value=v, block_table=_m((2, 5), I32), context_lens=_m((3,), I32)), "one row per sequence")
    _refuses(lambda: call(cu_seqlens_k=_m((3,), I32)), "cu_seqlens_k must be")
    _refuses(lambda: call(cu_seqlens_q=_m((0,), I32)), "batch \\+ 1")
    _refuses(lambda: call(cu_seqlens_q=_m((1,), I32)), "without a sequence")
    _refuses(lambda: call(cu_seqlens_q=_m((4,), torch.int64)), "int32")


def test_mrope_refusals():
    good = dict(positions=_m((3, 7), I32), query=_m((7, 4, 64)), key=_m((7, 2, 64)), cos_sin_cache=_m((100, 64), torch.float32),
                mrope_section=[8, 12, 12])
    call = lambda **kw: q.npu_mrope(**{**good, **kw})  # noqa: E731
    call()
    _refuses(lambda: call(mrope_section=None), "need mrope_section")
    _refuses(lambda: call(mrope_section=[8, 12]), "must have 3 values")
    _refuses(lambda: call(mrope_section=[8, 12, 11]), "sum to rotary_dim / 2")
    _refuses(lambda: call(mrope_section=[-4, 18, 18]), "not be negative")
    _refuses(lambda: call(rotary_mode="neox"), "'half' or 'interleave'")
    _refuses(lambda: call(positions=_m((5, 7), I32), mrope_section=[8, 6, 6, 6, 6]), "1 to 4 axes")
    _refuses(lambda: call(positions=_m((3, 6), I32)), "one column per token")
    _refuses(lambda: call(cos_sin_cache=_m((100, 66), torch.float32)), "at most head_dim")
    _refuses(lambda: call(cos_sin_cache=_m((100, 31), torch.float32)), "must be even")
    _refuses(lambda: call(cos_sin_cache=_m((100, 64), F16)), "float32 or BFloat16")
    _refuses(lambda: call(key=_m((7, 2, 32))), "key must be")
    k, v = _cache()
    good = dict(positions=_m((7,), I32), query=_m((7, 4, 64)), key=_m((7, 2, 64)), value=_m((7, 2, 64)),
                cos_sin_cache=_m((100, 64), torch.float32), key_cache=k, value_cache=v, slot_mapping=_m((7,), I32))
    call = lambda **kw: q.npu_mrope_scatter_kv(**{**good, **kw})  # noqa: E731
    call()
    _refuses(lambda: call(slot_mapping=_m((6,), I32)), "one slot per token")
    _refuses(lambda: call(slot_mapping=_m((7,), torch.int64)), "int32")
    _refuses(lambda: call(value=_m((7, 1, 64))), "value must be as key")
    _refuses(lambda: call(key_cache=_m((10, 16, 4, 64)), value_cache=_m((10, 16, 4, 64))), "the key's heads")


def test_pages_refusals():
    k, v = _cache()
    t, n, c, two = _m((6, 5), I32), _m((6,), I32), _m((10,), I32), _m((2,), I32)
    _refuses(lambda: q.npu_kv_fork([k, _m((9, 16, 2, 64))], t, n, c, two, two, 16), "must have 10 pages")
    _refuses(lambda: q.npu_kv_fork([k], t, n, c, two, _m((3,), I32), 16), "one length")
    _refuses(lambda: q.npu_kv_fork([k], t, n, c, two, two, 0), "page_size must be positive")
    _refuses(lambda: q.npu_kv_fork([_m((10, 8, 8))[:, :, :4]], t, n, c, two, two, 16), "must be dense")
    _refuses(lambda: q.npu_kv_fork([_m((1, 8)).expand(10, 8)], t, n, c, two, two, 16), "overlap")
    _refuses(lambda: q.npu_kv_free(t, _m((5,), I32), c, two, 16), "one length per row")
    _refuses(lambda: q.npu_kv_free(t.t(), _m((5,), I32), c, two, 16), "contiguous")
    _refuses(lambda: q.npu_kv_extend(t, n, c, two, two, 9, 16), "one value more")
    _refuses(lambda: q.npu_kv_extend(t, n, c, two, _m((3,), I32), -1, 16), "not be negative")
    _refuses(lambda: q.npu_kv_compact([k], t, _m((10,), torch.int64)), "int32")
    _refuses(lambda: q.npu_kv_copy_pages([k], two, _m((3,), I32)), "one length")


def _abi_cache(**kw):
    c = q.KvCache(key=4096, value=4096, num_pages=10, page_size=16, kv_heads=2, head_dim=64, key_page_stride=2048,
                  key_token_stride=128, key_head_stride=64, value_page_stride=2048, value_token_stride=128,
                  value_head_stride=64, dtype=q.QK_BF16)
    for name, x in kw.items():
        setattr(c, name, x)
    return c


def test_abi_refusals():
    """Every check comes before a launch, so these run without a GPU (the pointers are never followed)."""
    L = q.abi()
    fake = ctypes.c_void_p(4096)

    def decode(c, dtype=q.QK_BF16, batch=3, heads=8, strides=(512, 64), width=5, window=0, query=fake, lens=fake):
        return L.qk_paged_attention(query, dtype, batch, heads, *strides, ctypes.byref(c) if c else None, fake, width, width,
                                    lens, 0.1, window, 0, fake, fake, None, 0, None)

    assert decode(None) == q.QK_ERR_ARG and "null cache" in q.last_error()
    assert decode(_abi_cache(), dtype=q.QK_F32) == q.QK_ERR_ARG
    assert decode(_abi_cache(dtype=q.QK_F16)) == q.QK_ERR_ARG and "int8 or of the tensors' dtype" in q.last_error()
    assert decode(_abi_cache(head_dim=60)) == q.QK_ERR_UNSUPPORTED and "multiple of 8" in q.last_error()
    assert decode(_abi_cache(head_dim=264)) == q.QK_ERR_UNSUPPORTED
    assert decode(_abi_cache(head_dim=72, dtype=q.QK_I8)) == q.QK_ERR_UNSUPPORTED and "multiple of 16" in q.last_error()
    assert decode(_abi_cache(dtype=q.QK_I8)) == q.QK_ERR_ARG and "key_scale" in q.last_error()
    assert decode(_abi_cache(page_size=0)) == q.QK_ERR_ARG
    assert decode(_abi_cache(num_pages=1 << 28)) == q.QK_ERR_UNSUPPORTED and "31 bits" in q.last_error()
    assert decode(_abi_cache(), heads=7) == q.QK_ERR_ARG and "multiple of kv_heads" in q.last_error()
    assert decode(_abi_cache(), batch=-1) == q.QK_ERR_ARG
    assert decode(_abi_cache(), width=1 << 30) == q.QK_ERR_UNSUPPORTED
    assert decode(_abi_cache(), window=-3) == q.QK_ERR_ARG
    assert decode(_abi_cache(), strides=(512, 63)) == q.QK_ERR_ARG and "strides" in q.last_error()
    assert decode(_abi_cache(), query=ctypes.c_void_p(4098)) == q.QK_ERR_ARG and "aligned" in q.last_error()
    assert decode(_abi_cache(key_token_stride=100)) == q.QK_ERR_ARG and "16 bytes" in q.last_error()
    assert decode(_abi_cache(key=4104)) == q.QK_ERR_ARG and "16-byte aligned" in q.last_error()
    assert decode(_abi_cache(), lens=None) == q.QK_ERR_ARG and "null pointer" in q.last_error()
    assert decode(_abi_cache(), batch=0) == q.QK_OK
    n = ctypes.c_size_t(0)
    assert L.qk_paged_attention_workspace_size(3, 8, ctypes.byref(_abi_cache()), 5, 0, 0, None) == q.QK_ERR_ARG
    assert L.qk_prompt_attention_workspace_size(-1, 3, 8, ctypes.byref(_abi_cache()), 5, 0, 0, ctypes.byref(n)) == q.QK_ERR_ARG
    c = _abi_cache(num_pages=1)
    prompt = lambda *mid: L.qk_prompt_attention(fake, q.QK_BF16, 9, 3, 8, 512, 64, *mid, 0.1, 0, 0, fake, None, None, 0, None)  # noqa: E731
    assert prompt(None, ctypes.byref(c), fake, None, 0, 0, None) == q.QK_ERR_ARG
    assert prompt(fake, ctypes.byref(c), fake, None, 5, 5, fake) == q.QK_ERR_ARG and "either paged" in q.last_error()
    assert prompt(fake, ctypes.byref(c), None, None, 0, 0, None) == q.QK_ERR_ARG and "cu_seqlens_k" in q.last_error()
    assert prompt(fake, ctypes.byref(_abi_cache()), fake, None, 0, 0, None) == q.QK_ERR_ARG and "one page" in q.last_error()
    pages = q.Pages(base=4096, page_stride=100, page_bytes=200)
    assert L.qk_kv_copy_pages(ctypes.byref(pages), 1, 5, fake, fake, 2, None) == q.QK_ERR_ARG
    assert L.qk_kv_free(5, 16, fake, 4, 8, 7, fake, fake, fake, 2, None) == q.QK_ERR_ARG and "overlap" in q.last_error()
    assert L.qk_kv_free(5, 16, fake, 4, 8, 8, fake, fake, fake, 65537, None) == q.QK_ERR_UNSUPPORTED
    assert L.qk_kv_fork(None, 0, 5, 16, fake, 4, 8, 8, fake, fake, fake, fake, 2, fake, None, 0, None) == q.QK_ERR_WORKSPACE
    assert L.qk_kv_extend(5, 16, fake, 4, 8, 8, fake, fake, fake, fake, 2, 9, fake, fake, fake, ctypes.c_void_p(4100), 1 << 20,
                          None) == q.QK_ERR_WORKSPACE and "256-byte" in q.last_error()


def test_page_division_rule():
    """(j * m) >> s with m = ceil(2^s / d), s = 31 + ceil(log2 d), is j // d for every j below 2^31."""
    rng = random.Random(0)
    for d in [1, 2, 3, 5, 7, 16, 48, 100, 127, 128, 129, 1000, 65535, 65537, (1 << 30) + 1, (1 << 31) - 1] + \
            [rng.randrange(1, 1 << 31) for _ in range(300)]:
        c = (d - 1).bit_length()
        s = 31 + c
        m = -(-(1 << s) // d)
        assert m < 1 << 32
        top = (1 << 31) - 1
        near = [x for k in (1, 2, top // d // 2, top // d) for x in (k * d - 1, k * d, k * d + 1)]
        for j in near + [0, 1, top] + [rng.randrange(0, 1 << 31) for _ in range(50)]:
            if 0 <= j <= top:
                assert (j * m) >> s == j // d


def test_oracle_attention():
    """The 64-bit oracle against torch's own on a causal case, and its masks against their definition."""
    g = torch.Generator().manual_seed(0)
    qq, k, v = (torch.randn((6, h, 8), generator=g, dtype=torch.float64) for h in (4, 2, 2))
    out, lse = R.attend(qq, k, v, R.visible(6, 6, 0, 0), 0.3)[:2]
    want = torch.nn.functional.scaled_dot_product_attention(
        qq.transpose(0, 1), k.repeat_interleave(2, 1).transpose(0, 1), v.repeat_interleave(2, 1).transpose(0, 1),
        is_causal=True, scale=0.3).transpose(0, 1)
    assert torch.allclose(out, want, rtol=1e-12, atol=1e-12)
    assert R.visible(2, 5, 2, 1).tolist() == [[True, False, True, True, False], [True, False, False, True, True]]
    assert R.visible(4, 2, 0, 0).tolist() == [[False, False], [False, False], [True, False], [True, True]]
    assert torch.isneginf(R.attend(qq, k, v, torch.zeros((6, 6), dtype=torch.bool), 0.3)[1]).all()


def test_oracle_rotation():
    x = torch.tensor([[[1.0, 2.0, 3.0, 4.0, 9.0]]], dtype=torch.float64)
    table = torch.tensor([[0.0, 0.5, 1.0, 0.25], [7.0, 7.0, 7.0, 7.0]])
    pos = torch.tensor([[0], [0]])
    y = R.rotate(x, pos, table, [1, 1], "half")
    assert y.flatten().tolist() == [1 * 0 - 3 * 1, 2 * 0.5 - 4 * 0.25, 3 * 0 + 1 * 1, 4 * 0.5 + 2 * 0.25, 9]
    y = R.rotate(x, pos, table, [1, 1], "interleave")
    assert y.flatten().tolist() == [1 * 0 - 2 * 1, 2 * 0 + 1 * 1, 3 * 0.5 - 4 * 0.25, 4 * 0.5 + 3 * 0.25, 9]


def test_oracle_pool():
    pool = R.Pool(torch.tensor([[3, -1], [-1, -1]]), torch.tensor([3, 0]), torch.tensor([0, 1, 0, 1]), 2)
    pool.table[0] = [3, 1]
    assert pool.fork([0], [1]) == ([(1, 0)], 0) and pool.table[1] == [3, 0] and pool.count == [1, 1, 0, 2]
    assert pool.extend([1], [1]) == ([1], [3], 0) and pool.lens == [3, 4]
    pool.free([0])
    assert pool.count == [1, 0, 0, 1]
    assert pool.compact() == ([[-1, -1], [1, 0]], [1, 1, 0, 0], [(3, 1)])
