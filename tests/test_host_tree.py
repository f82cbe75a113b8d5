"""Host side of decoding with drafts, no GPU: masks and positions of trees, shape inference and refusals (Meta tensors), the C ABI's
checks before any launch."""
import ctypes
import random

import pytest
import torch

import op_plugin_amd as q
import tree_ref as T
from op_plugin_amd.kv_cache import PagedKVCache
from op_plugin_amd.tree import tree_mask, tree_positions
from test_host_attention import BF16, F16, I32, _cache, _m, _refuses

I64, F32 = torch.int64, torch.float32


def test_registered():
    for name in ("npu_tree_attention", "npu_kv_accept", "npu_sample"):
        assert getattr(q, name) is getattr(torch.ops.npu, name) and name in q.__all__


@pytest.mark.parametrize("sizes", [[1], [5, 0, 3], [64], [65, 1], [200, 7, 0], [0]])
def test_masks_and_positions(sizes):
    trees = T.trees(3, sizes)
    cu = [0]
    for n in sizes:
        cu.append(cu[-1] + n)
    words = max(1, -(-max(sizes) // 64))
    parents = torch.tensor([p for t in trees for p in t], dtype=I32)
    cu_t = torch.tensor(cu, dtype=I32)
    mask, depth = tree_mask(parents, cu_t, words)
    rows = [r for t in trees for r in T.ancestors(t)]
    assert torch.equal(mask, T.mask_words(rows, words)) and mask.dtype == I64
    assert depth.tolist() == [len(r) - 1 for r in rows] and depth.dtype == I32
    start = [random.Random(i).randrange(100) for i in range(len(sizes))]
    positions = torch.tensor([s + i for s, n in zip(start, sizes) for i in range(n)], dtype=I32)
    want = [s + len(r) - 1 for s, t in zip(start, trees) for r in T.ancestors(t)]
    assert tree_positions(positions, cu_t, depth).tolist() == want
    assert tree_positions(torch.full_like(positions, -1), cu_t, depth).tolist() == [-1] * len(want)


def test_mask_of_odd_parents():
    mask, depth = tree_mask(torch.tensor([5, 0, 2, -7, 3, 9], dtype=I32), torch.tensor([0, 6], dtype=I32))
    assert mask.squeeze(1).tolist() == [1, 3, 4, 8, 24, 32] and depth.tolist() == [0, 1, 0, 0, 1, 0]
    with pytest.raises(ValueError):
        tree_mask(torch.zeros(3, dtype=I32), torch.tensor([0, 3], dtype=I32), 0)
    with pytest.raises(ValueError):
        tree_mask(torch.zeros((3, 1), dtype=I32), torch.tensor([0, 3], dtype=I32))


def test_meta_shapes():
    k, v = _cache()
    out, lse = q.npu_tree_attention(_m((30, 8, 64)), k, v, _m((4,), I32), _m((3, 5), I32), _m((3,), I32), _m((30, 2), I64), window=4)
    assert out.shape == (30, 8, 64) and out.dtype == BF16 and lse.shape == (30, 8) and lse.dtype == F32
    out, lse = q.npu_tree_attention(_m((0, 8, 64)), k, v, _m((1,), I32), _m((0, 5), I32), _m((0,), I32), _m((0, 1), I64))
    assert out.shape == (0, 8, 64)
    tokens, lp = q.npu_sample(_m((7, 1000), F16), _m((7,), F32), temperature=_m((7,), F32), top_k=_m((7,), I32), top_p=_m((7,), F32),
                              min_p=_m((7,), F32))
    assert tokens.shape == lp.shape == (7,) and tokens.dtype == I32 and lp.dtype == F32
    path, accepted, nxt = q.npu_kv_accept([k, v, _m((10, 16, 2), F32)], _m((6, 5), I32), _m((6,), I32), _m((10,), I32), _m((2,), I32),
                                          _m((3,), I32), _m((9,), I32), _m((9,), I32), _m((9,), I32), 16)
    assert path.shape == (9,) and accepted.shape == nxt.shape == (2,) and path.dtype == accepted.dtype == nxt.dtype == I32


def test_tree_attention_refusals():
    k, v = _cache()
    good = dict(query=_m((30, 8, 64)), key_cache=k, value_cache=v, cu_seqlens_q=_m((4,), I32), block_table=_m((3, 5), I32),
                context_lens=_m((3,), I32), tree_mask=_m((30, 1), I64))
    call = lambda **kw: q.npu_tree_attention(**{**good, **kw})  # noqa: E731
    call()
    _refuses(lambda: call(query=_m((30, 8, 64), F32)), "float16 or bfloat16")
    _refuses(lambda: call(query=_m((30, 7, 64))), "multiple of the keys'")
    _refuses(lambda: call(query=_m((30, 8, 32))), "one head_dim")
    _refuses(lambda: call(query=_m((30, 8, 64), F16)), "int8 or Half")
    _refuses(lambda: call(tree_mask=_m((30,), I64)), "tree_mask must be int64")
    _refuses(lambda: call(tree_mask=_m((30, 1), I32)), "tree_mask must be int64")
    _refuses(lambda: call(tree_mask=_m((29, 1), I64)), "tree_mask must be int64")
    _refuses(lambda: call(tree_mask=_m((30, 0), I64)), "a word at least")
    _refuses(lambda: call(tree_mask=_m((30, 1), I64).expand(30, 2 ** 31 // 64 + 1)), "words")
    _refuses(lambda: call(tree_mask=torch.zeros((30, 1), dtype=I64)), "tree_mask must be on")
    _refuses(lambda: call(block_table=_m((4, 5), I32)), "one row per sequence")
    _refuses(lambda: call(context_lens=_m((2,), I32)), "one row per sequence")
    _refuses(lambda: call(cu_seqlens_q=_m((1,), I32), block_table=_m((0, 5), I32), context_lens=_m((0,), I32)), "rows without a sequence")
    _refuses(lambda: call(cu_seqlens_q=_m((4,), I64)), "cu_seqlens_q must be int32")
    _refuses(lambda: call(window=-1), "must not be negative")
    _refuses(lambda: call(scale=float("inf")), "scale must be finite")
    _refuses(lambda: call(key_scale=_m((10, 16, 2), F32), value_scale=_m((10, 16, 2), F32)), "go with int8")
    for D in (60, 264):
        k2, v2 = _cache(D=D)
        _refuses(lambda: call(query=_m((30, 8, D)), key_cache=k2, value_cache=v2), "head_dim must be")
    far = _m((1 << 27, 16, 2, 64))
    _refuses(lambda: call(key_cache=far, value_cache=far), "31 bits")


def test_sample_refusals():
    good = dict(logits=_m((7, 1000)), uniform=_m((7,), F32))
    call = lambda **kw: q.npu_sample(**{**good, **kw})  # noqa: E731
    call()
    _refuses(lambda: call(logits=_m((7, 1000), I32)), "float16, bfloat16 or float32")
    _refuses(lambda: call(logits=_m((7, 1000), torch.float64)), "float16, bfloat16 or float32")
    _refuses(lambda: call(logits=_m((7,))), "rows, vocabulary")
    _refuses(lambda: call(logits=_m((7, 0))), "vocabulary of 1 to")
    _refuses(lambda: call(logits=_m((7, (1 << 24) + 1))), "vocabulary of 1 to")
    _refuses(lambda: call(logits=_m((1 << 22, 2)), uniform=_m((1 << 22,), F32)), "number of rows")
    _refuses(lambda: call(uniform=_m((6,), F32)), "uniform must be")
    _refuses(lambda: call(uniform=_m((7,), BF16)), "uniform must be")
    _refuses(lambda: call(uniform=torch.zeros(7)), "uniform must be on")
    _refuses(lambda: call(temperature=_m((7, 1), F32)), "temperature must be")
    _refuses(lambda: call(top_k=_m((7,), I64)), "top_k must be")
    _refuses(lambda: call(top_p=_m((1,), F32)), "top_p must be")
    _refuses(lambda: call(min_p=_m((7,), F16)), "min_p must be")


def test_accept_refusals():
    k, v = _cache()
    good = dict(caches=[k, v], block_table=_m((6, 5), I32), context_lens=_m((6,), I32), ref_count=_m((10,), I32), seqs=_m((2,), I32),
                cu_tokens=_m((3,), I32), tokens=_m((9,), I32), parents=_m((9,), I32), sampled=_m((9,), I32), page_size=16)
    call = lambda **kw: q.npu_kv_accept(**{**good, **kw})  # noqa: E731
    call()
    call(caches=[])
    call(caches=[_m((10, 2, 16, 64)).transpose(1, 2), _m((10, 16, 4, 64))[:, :, 1:3], _m((10, 16, 3, 2, 64))])
    _refuses(lambda: call(caches=[_m((10, 16, 3, 4, 72))[:, :, :, :2, :64]]), "at one distance")
    _refuses(lambda: call(caches=[k, _m((9, 16, 2, 64))]), "every cache tensor must be")
    _refuses(lambda: call(caches=[_m((10, 8, 2, 64))]), "every cache tensor must be")
    _refuses(lambda: call(caches=[_m((10,))]), "every cache tensor must be")
    _refuses(lambda: call(caches=[torch.zeros((10, 16, 2))]), "a cache tensor must be on")
    _refuses(lambda: call(caches=[_m((1, 16, 2, 64)).expand(10, 16, 2, 64)]), "overlap")
    _refuses(lambda: call(caches=[_m((10, 16, 1, 64)).expand(10, 16, 2, 64)]), "at one distance")
    _refuses(lambda: call(page_size=0), "page_size must be positive")
    _refuses(lambda: call(cu_tokens=_m((2,), I32)), "one value more than seqs")
    _refuses(lambda: call(tokens=_m((9,), I64)), "tokens must be int32")
    _refuses(lambda: call(parents=_m((8,), I32)), "one length")
    _refuses(lambda: call(sampled=_m((9, 1), I32)), "sampled must have 1")
    _refuses(lambda: call(seqs=_m((70000,), I32), cu_tokens=_m((70001,), I32)), "at most")
    _refuses(lambda: call(block_table=_m((5, 6), I32).t()), "must be contiguous")


def test_cache_and_block():
    cache = PagedKVCache(2, 10, 16, 2, 64, max_seqs=4, max_len=50, device="meta")
    path, accepted, nxt = cache.accept(_m((2,), I32), _m((3,), I32), _m((9,), I32), _m((9,), I32), _m((9,), I32))
    assert path.shape == (9,) and accepted.shape == nxt.shape == (2,)
    from op_plugin_amd.attention import quant_attention
    with pytest.raises(ValueError, match="need cu_tokens"):
        quant_attention(None, None, None, None, None, None, cache, 0, None, None, None, None, None, 8, tree_mask=_m((9, 1), I64))


def test_abi_refusals():
    L = q.abi()
    size = ctypes.c_size_t(7)
    none = ctypes.c_void_p()
    one = ctypes.c_void_p(256)
    assert L.qk_sample_workspace_size(3, 0, q.QK_F32, ctypes.byref(size)) == q.QK_ERR_UNSUPPORTED
    assert L.qk_sample_workspace_size(3, 100, q.QK_I8, ctypes.byref(size)) == q.QK_ERR_ARG and "float16" in q.last_error()
    assert L.qk_sample_workspace_size(-1, 100, q.QK_F32, ctypes.byref(size)) == q.QK_ERR_ARG
    assert L.qk_sample_workspace_size(1 << 22, 100, q.QK_F32, ctypes.byref(size)) == q.QK_ERR_ARG and "at most" in q.last_error()
    assert L.qk_sample_workspace_size(3, 100, q.QK_F32, None) == q.QK_ERR_ARG
    assert L.qk_sample_workspace_size(0, 100, q.QK_F32, ctypes.byref(size)) == q.QK_OK and size.value == 0
    assert L.qk_sample_workspace_size(4, 200000, q.QK_BF16, ctypes.byref(size)) == q.QK_OK and size.value > 0
    sample = lambda x=one, dt=q.QK_BF16, rows=4, vocab=200000, stride=200000, u=one, t=one, ws=one, n=1 << 30: L.qk_sample(  # noqa: E731
        x, dt, rows, vocab, stride, u, none, none, none, none, t, one, ws, n, none)
    assert sample(rows=0) == q.QK_OK
    assert sample(x=none) == sample(u=none) == sample(t=none) == q.QK_ERR_ARG and "null" in q.last_error()
    assert sample(stride=-1) == q.QK_ERR_ARG
    assert sample(x=ctypes.c_void_p(257)) == q.QK_ERR_ARG
    assert sample(ws=none) == sample(n=100) == q.QK_ERR_WORKSPACE and "required" in q.last_error()
    assert sample(ws=ctypes.c_void_p(264)) == q.QK_ERR_WORKSPACE and "aligned" in q.last_error()
    c = q.KvCache(key=256, value=256, num_pages=4, page_size=16, kv_heads=2, head_dim=64, key_page_stride=2048, key_token_stride=128,
                  key_head_stride=64, value_page_stride=2048, value_token_stride=128, value_head_stride=64, dtype=q.QK_BF16)
    tree = lambda cu=one, table=one, lens=one, mask=one, words=1, stride=1, batch=2, tokens=9, scale=1.0, ws=one, n=1 << 40: (  # noqa: E731
        L.qk_tree_attention(one, q.QK_BF16, tokens, batch, 8, 512, 64, cu, ctypes.byref(c), table, 50, 50, lens, mask, words, stride,
                            scale, 0, 0, one, none, ws, n, none))
    assert tree(tokens=0) == q.QK_OK
    assert tree(cu=none) == tree(mask=none) == tree(lens=none) == tree(table=none) == q.QK_ERR_ARG and "null" in q.last_error()
    assert tree(words=0) == tree(words=1 << 40) == tree(stride=-1) == q.QK_ERR_ARG and "words" in q.last_error()
    assert tree(mask=ctypes.c_void_p(260)) == q.QK_ERR_ARG and "8-byte" in q.last_error()
    assert tree(batch=0) == q.QK_ERR_ARG and "without a sequence" in q.last_error()
    assert tree(scale=float("nan")) == q.QK_ERR_ARG
    assert tree(n=8) == tree(ws=none) == q.QK_ERR_WORKSPACE
    rows = (q.Rows * 1)(q.Rows(256, 2048, 128, 0, 1, 128))
    accept = lambda rows=rows, k=1, pages=10, S=16, n=2, total=9, tokens=one, path=one, ws=one, b=1 << 20: L.qk_kv_accept(  # noqa: E731
        rows, k, pages, S, one, 6, 5, 5, one, one, one, one, n, total, tokens, one, one, path, one, one, ws, b, none)
    assert accept(k=-1) == accept(rows=None) == q.QK_ERR_ARG
    assert accept(tokens=none) == accept(path=none) == q.QK_ERR_ARG and "null" in q.last_error()
    assert accept(S=0) == accept(total=-1) == accept(n=-1) == q.QK_ERR_ARG
    assert accept(n=70000) == q.QK_ERR_UNSUPPORTED
    assert accept(ws=none) == accept(b=8) == q.QK_ERR_WORKSPACE
    bad = (q.Rows * 1)(q.Rows(256, 2048, 128, 64, 2, 128))
    assert accept(rows=bad) == q.QK_ERR_ARG and "overlap" in q.last_error()
    assert accept(rows=(q.Rows * 1)(q.Rows(None, 2048, 128, 0, 1, 128))) == q.QK_ERR_ARG
    assert L.qk_kv_accept_workspace_size(2, None) == q.QK_ERR_ARG
