"""Meta calls of the attention and cache ops refuse what a call on the device refuses in the C ABI, and nothing else: a traced
program fails where it is traced."""
import pytest
import torch

import op_plugin_amd as q
from test_host_attention import F16, I8, I32, _m, _refuses

BIG = 2 ** 31 - 1


def _decode(D=64, dtype=F16, P=10, S=16, H=2, Hq=8, k=None, width=5, tokens=3):
    k = _m((P, S, H, D), dtype) if k is None else k
    scale = dict(key_scale=_m(k.shape[:3], torch.float32), value_scale=_m(k.shape[:3], torch.float32)) if dtype == I8 else {}
    return lambda: q.npu_paged_attention(_m((tokens, Hq, D), F16), k, k, _m((tokens, width), I32), _m((tokens,), I32), **scale)


def _paged_prompt(D=64, dtype=F16, P=10, S=16, H=2, Hq=8, k=None, width=5, tokens=30):
    k = _m((P, S, H, D), dtype) if k is None else k
    scale = dict(key_scale=_m(k.shape[:3], torch.float32), value_scale=_m(k.shape[:3], torch.float32)) if dtype == I8 else {}
    return lambda: q.npu_prompt_attention(_m((tokens, Hq, D), F16), k, k, _m((4,), I32), block_table=_m((3, width), I32),
                                          context_lens=_m((3,), I32), **scale)


def _scatter(D=64, dtype=F16, P=10, S=16, H=2, Hq=8, k=None, tokens=7):
    k = _m((P, S, H, D), dtype) if k is None else k
    scale = dict(key_scale=_m(k.shape[:3], torch.float32), value_scale=_m(k.shape[:3], torch.float32)) if dtype == I8 else {}
    x = _m((tokens, H, D), F16)
    return lambda: q.npu_mrope_scatter_kv(_m((tokens,), I32), _m((tokens, Hq, D), F16), x, x, _m((100, 32), torch.float32), k, k,
                                          _m((tokens,), I32), **scale)


@pytest.mark.parametrize("form", [_decode, _paged_prompt, _scatter])
def test_cache_limits(form):
    for good in (dict(), dict(dtype=I8), dict(D=256), dict(D=72), dict(D=80, dtype=I8), dict(P=0),
                 dict(k=_m((10, 16, 2, 64 + 8), F16)[..., :64]), dict(k=_m((10, 2, 16, 64), F16).transpose(1, 2)),
                 dict(k=_m((10, 16, 2, 64 + 8), F16)[..., 8:]), dict(k=_m((1, 1, 1, 3 * 64 + 1), F16)[..., :64], H=1)):
        form(**good)()
    for D in (60, 264, 1000):
        _refuses(form(D=D), "head_dim must be")
    _refuses(form(D=72, dtype=I8), "multiple of 16")
    _refuses(form(k=_m((10, 16, 2, 64 + 4), F16)[..., :64]), "multiples of 16 bytes")
    _refuses(form(k=_m((10, 16, 2 * 64 + 4), F16)[..., :128].unflatten(-1, (2, 64))), "multiples of 16 bytes")
    _refuses(form(dtype=I8, k=_m((10, 16, 2, 64 + 8), I8)[..., :64]), "multiples of 16 bytes")
    _refuses(form(k=_m((10, 16, 2, 64 + 8), F16)[..., 4:68]), "16-byte aligned")
    _refuses(form(P=1 << 27), "31 bits")
    form(tokens=0)()


@pytest.mark.parametrize("form", [_decode, _paged_prompt])
def test_attention_limits(form):
    _refuses(form(width=1 << 28), "31 bits")
    _refuses(form(H=1, Hq=65536, tokens=30), "q_heads must be")
    _refuses(form(H=1, Hq=65535, tokens=40000), "launch limit")


def test_contiguous_keys():
    """Copied where their rows are not whole pieces, so only the sizes are refused; and nothing where there are no rows."""
    call = lambda k, tokens=30: lambda: q.npu_prompt_attention(_m((tokens, 8, k.shape[2]), F16), k, k, _m((4,), I32))  # noqa: E731
    call(_m((30, 2, 68), F16)[..., 4:])()
    call(_m((30, 64, 2), F16).transpose(1, 2))()
    call(_m((0, 2, 64), F16))()
    for D in (60, 264):
        _refuses(call(_m((30, 2, D), F16)), "head_dim must be")
        call(_m((0, 2, D), F16), 0)()
    with pytest.raises(RuntimeError, match="tokens, heads, head_dim"):
        q.npu_prompt_attention(_m((30, 8, 64), F16), _m((), F16), _m((), F16), _m((4,), I32))


def test_rotation_limits():
    call = lambda D, Hq=4, T=7: lambda: q.npu_mrope(_m((T,), I32), _m((T, Hq, D), F16), _m((T, 2, D), F16),  # noqa: E731
                                                    _m((100, 32), torch.float32))
    call(256)()
    call(60)()
    call(300, T=0)()
    _refuses(call(257), "head_dim must be 1..256")
    _refuses(call(64, Hq=65536), "invalid size")


def test_page_limits():
    t, n, c = _m((6, 5), I32), _m((6,), I32), _m((10,), I32)
    many = _m((65537,), I32)
    for page in (1 << 28, BIG):
        _refuses(lambda: q.npu_kv_free(t, n, c, _m((2,), I32), page), "31 bits")
    q.npu_kv_free(t, n, c, _m((65536,), I32), BIG // 10)
    _refuses(lambda: q.npu_kv_free(t, n, c, many, 16), "at most 65536")
    _refuses(lambda: q.npu_kv_fork([], t, n, c, many, many, 16), "at most 65536")
    _refuses(lambda: q.npu_kv_fork([], t, n, c, _m((2,), I32), _m((2,), I32), 1 << 28), "31 bits")
    _refuses(lambda: q.npu_kv_extend(t, n, c, many, _m((65538,), I32), 9, 16), "at most 65536")
    _refuses(lambda: q.npu_kv_extend(t, n, c, _m((2,), I32), _m((3,), I32), 2 ** 31, 16), "number of tokens")
