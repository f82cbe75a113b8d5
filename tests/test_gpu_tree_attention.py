"""npu_tree_attention against attention in 64 bits: trees of every size from none to several words of the mask, over contexts
from nothing to many parts, pages that end inside a tile, windows that cut the context by depth, masks that are no tree's,
and NaN in every place that no row sees."""
import math
import random

import pytest
import torch

import attention_ref as R
import tree_ref as T

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import op_plugin_amd
    return op_plugin_amd


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32)


def _run(ops, past, sizes, Hq=8, Hkv=2, D=64, page=16, dtype=BF16, quant=False, window=0, sinks=0, scale=None, rows=None, words=None,
         extra=0, order="snd", seed=0, times=1):
    """past[b]: tokens before the tree; sizes[b]: of the tree; rows: masks as sets, of random trees by default; extra: rows past
    the last sequence."""
    print(f"[case] tree past={past} sizes={sizes} Hq={Hq} Hkv={Hkv} D={D} page={page} {dtype} quant={quant} window={window} "
          f"sinks={sinks} words={words} extra={extra} {order}", flush=True)
    g = torch.Generator().manual_seed(seed)
    lens = [max(p + n, 0) for p, n in zip(past, sizes)]
    if rows is None:
        rows = [T.ancestors(t) for t in T.trees(seed, sizes)]
    words = words or max(1, -(-max(sizes) // 64))
    kv, table, kc, vc, ks, vs = R.pools(lens, page, Hkv, D, dtype, quant, g)
    cu = [0]
    for n in sizes:
        cu.append(cu[-1] + n)
    q = torch.randn((cu[-1] + extra, Hq, D), generator=g).to(dtype)
    s = scale if scale is not None else 1 / math.sqrt(D)
    parts = []
    for b, (k, v) in enumerate(kv):
        cut = [{i for i in row if i < 64 * words} for row in rows[b]]
        ok = T.visible(cut, lens[b], window, sinks)
        hidden = ~ok.any(0)
        pg = table[b, hidden.nonzero().squeeze(1) // page].long()
        at = hidden.nonzero().squeeze(1) % page
        if sizes[b]:
            for c in ([ks, vs] if quant else [kc, vc]):
                c[pg, at] = math.nan
        parts.append(R.attend(q[cu[b]:cu[b + 1]].double(), k, v, ok, s))
    none = torch.zeros((extra, Hq), dtype=torch.float64)
    parts.append([torch.zeros((extra, Hq, D), dtype=torch.float64), none - math.inf, torch.zeros((extra, Hq, D), dtype=torch.float64),
                  none, none])
    ref = [torch.cat(x) for x in zip(*parts)]
    ref[3] = ref[3].abs()  # the size of the scores, scale * max sum |q k|: its sign is the scale's
    mask = T.mask_words([r for rs in rows for r in rs] + [{0, 1}] * extra, words)
    kd, vd, ksd, vsd, td, qd, md = _dev(kc, vc, ks, vs, table, q, mask)
    if order == "nsd":
        kd, vd = (t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (kd, vd))
    elif order == "fused":
        both = torch.cat([kd, vd], dim=2)
        kd, vd = both[:, :, :Hkv], both[:, :, Hkv:]
        qd = torch.cat([qd, qd], dim=2).transpose(0, 1).contiguous().transpose(0, 1)[..., :D]
        md = torch.cat([md, md], dim=1)[:, :words]
    out, lse = ops.npu_tree_attention(qd, kd, vd, _ints(cu).to(DEV), td, _ints(lens).to(DEV), md, key_scale=ksd, value_scale=vsd,
                                      scale=scale, window=window, sinks=sinks)
    assert out.shape == q.shape and out.dtype == dtype and lse.dtype == torch.float32
    R.check(out, lse, ref, dtype, max(lens + [1]), extra_values=int(quant and dtype == F16))
    for i in range(times):
        if i % 2:  # what a pass leaves in its workspace and in LDS is another's
            ops.npu_tree_attention(-qd, kd, kd, _ints(cu).to(DEV), td, _ints(lens).to(DEV), md, key_scale=ksd, value_scale=ksd, scale=scale)
        again, lse2 = ops.npu_tree_attention(qd, kd, vd, _ints(cu).to(DEV), td, _ints(lens).to(DEV), md, key_scale=ksd, value_scale=vsd,
                                             scale=scale, window=window, sinks=sinks)
        assert torch.equal(out, again) and torch.equal(lse, lse2), "the same call twice"
    return out, lse


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("past,sizes", [([0], [1]), ([0, 5], [3, 0]), ([63], [2]), ([64, 1, 0], [1, 64, 7]), ([1000], [33]),
                                        ([0, 700, 30], [40, 1, 16])])
def test_sizes(ops, past, sizes, dtype, quant):
    _run(ops, past, sizes, dtype=dtype, quant=quant)


@pytest.mark.parametrize("past,sizes,words", [([100], [65], None), ([0], [128], None), ([37, 64], [129, 5], None), ([50], [70], 1),
                                              ([10, 200], [20, 190], 4)])
def test_words(ops, past, sizes, words):
    """Trees of more tokens than one word holds, and words of the mask that end before the tree, or behind it."""
    _run(ops, past, sizes, Hq=2, Hkv=1, words=words)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (7, 1), (4, 4), (16, 2), (48, 1), (40, 8)])
def test_heads(ops, Hq, Hkv, quant):
    _run(ops, [77, 300], [5, 18], Hq, Hkv, quant=quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("D", [8, 16, 40, 64, 80, 96, 112, 128, 192, 200, 256])
def test_widths(ops, D, quant):
    if quant and D % 16:
        pytest.skip("int8 rows are whole 16-byte pieces")
    _run(ops, [65, 530], [9, 30], 4, 2, D, dtype=F16, quant=quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("page", [1, 3, 7, 48, 100, 1024])
def test_pages(ops, page, quant):
    _run(ops, [1, 95, 301], [4, 20, 11], 4, 1, page=page, quant=quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (3, 2), (16, 0), (33, 4), (100, 40), (64, 1000), (1000, 4), (250, 63)])
def test_window(ops, window, sinks, quant):
    _run(ops, [0, 1, 40, 333, 600], [9, 20, 5, 30, 40], 4, 1, quant=quant, window=window, sinks=sinks)


@pytest.mark.parametrize("order", ["nsd", "fused"])
@pytest.mark.parametrize("quant", [False, True])
def test_orders(ops, order, quant):
    _run(ops, [200, 33], [10, 3], 8, 4, quant=quant, order=order)


@pytest.mark.parametrize("past,sizes", [([5000], [8]), ([4097, 1, 9000, 64, 0, 2500], [5, 30, 12, 0, 64, 1]), ([300] * 40, [4] * 40),
                                        ([200] * 130, [1, 2, 0] * 43 + [7])])
def test_long_and_many(ops, past, sizes):
    """Keys in many parts, alone and among short contexts, and more sequences than a wave has lanes."""
    _run(ops, past, sizes, 4, 1, dtype=F16)


def test_masks_of_no_tree(ops):
    """Rows that see later rows, not themselves, nothing of the tree, or bits past it."""
    rng = random.Random(4)
    rows = [[{k for k in range(30) if rng.random() < 0.4} for _ in range(20)], [set(), {2}, {0, 1, 2, 3, 60}], [set()]]
    _run(ops, [50, 0, 0], [20, 3, 1], rows=rows)
    _run(ops, [500, 3, 0], [20, 3, 1], rows=rows, window=7, sinks=2)


def test_rows_past_the_last_sequence(ops):
    _run(ops, [100, 20], [10, 4], extra=3)
    _run(ops, [3000], [40], 4, 1, extra=50)


def test_fewer_tokens_than_rows(ops):
    """A length below the tree's size: its first rows have no place in the cache, so nobody sees them."""
    _run(ops, [-3, -20, 4], [10, 20, 3])
    _run(ops, [-3, -70], [10, 90], 2, 1, window=4, sinks=1)


def test_large_scores(ops):
    _run(ops, [500, 64], [9, 9], scale=4.0)
    _run(ops, [500, 64], [9, 9], dtype=F16, scale=0.0)
    _run(ops, [500, 64], [9, 9], dtype=F16, scale=-1.0)


def test_hidden_values_that_are_not_finite(ops):
    """NaN and infinities in a drafted token that only its descendants see: all other rows stay as they are without them."""
    print("[case] hidden values", flush=True)
    g = torch.Generator().manual_seed(1)
    n, past, page, D = 12, 100, 16, 64
    tree = [-1, 0, 0, 1, 1, 2, 2, 3, 4, 5, 6, 7]
    seen = T.ancestors(tree)
    kv, table, kc, vc, _, _ = R.pools([past + n], page, 1, D, BF16, False, g, fill=0.0)
    q = torch.randn((n, 2, D), generator=g).to(BF16).to(DEV)
    mask, cu, lens = T.mask_words(seen, 1).to(DEV), _ints([0, n]).to(DEV), _ints([past + n]).to(DEV)
    want, want_lse = ops.npu_tree_attention(q, *_dev(kc, vc), cu, table.to(DEV), lens, mask)
    at = past + 4
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2 = kc.clone(), vc.clone()
        v2[table[0, at // page].long(), at % page, 0, ::3] = bad
        k2[table[0, at // page].long(), at % page] = math.nan
        out, lse = ops.npu_tree_attention(q, *_dev(k2, v2), cu, table.to(DEV), lens, mask)
        blind = torch.tensor([4 not in s for s in seen])
        assert torch.equal(out[blind.to(DEV)], want[blind.to(DEV)]) and torch.equal(lse[blind.to(DEV)], want_lse[blind.to(DEV)])
        assert torch.isnan(out[~blind.to(DEV)]).any()


def test_bad_tables(ops):
    """Page ids outside the pool hide their tokens; lengths past the table are cut, negative ones are empty."""
    print("[case] bad tables", flush=True)
    g = torch.Generator().manual_seed(3)
    page, D, n = 16, 64, 6
    kv, table, kc, vc, _, _ = R.pools([100], page, 1, D, BF16, False, g, fill=0.0)
    table[0, 1], table[0, 3] = -7, 1 << 30
    seen = T.ancestors(T.trees(1, [n])[0])
    ok = T.visible(seen, 100, 0, 0)
    ok[:, 16:32] = False
    ok[:, 48:64] = False
    q = torch.randn((n, 4, D), generator=g).to(BF16)
    ref = R.attend(q.double(), *kv[0], ok, 1 / 8)
    args = [q.to(DEV), *_dev(kc, vc), _ints([0, n]).to(DEV)]
    mask = T.mask_words(seen, 1).to(DEV)
    out, lse = ops.npu_tree_attention(*args, table.to(DEV), _ints([100]).to(DEV), mask)
    R.check(out, lse, ref, BF16, 100)
    out, lse = ops.npu_tree_attention(*args, table.to(DEV), _ints([-5]).to(DEV), mask)
    assert (out == 0).all() and torch.isneginf(lse).all()
    out, lse = ops.npu_tree_attention(*args, table[:, :5].contiguous().to(DEV), _ints([2 ** 31 - 1]).to(DEV), mask)
    seen80 = T.visible(seen, 80, 0, 0)
    seen80[:, 16:32] = False
    seen80[:, 48:64] = False
    ref = R.attend(q.double(), kv[0][0][:80], kv[0][1][:80], seen80, 1 / 8)
    R.check(out, lse, ref, BF16, 100)
    out, lse = ops.npu_tree_attention(*args, table[:, :0].to(DEV), _ints([100]).to(DEV), mask)
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_offsets_past_32_bits(ops):
    """A pool of more than 4 GB: the last pages hold the sequence."""
    print("[case] far pages", flush=True)
    page, Hkv, D, P, n = 64, 8, 128, 36000, 5
    kc = torch.empty((P, page, Hkv, D), dtype=BF16, device=DEV)
    vc = torch.empty_like(kc)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn((2 * page, Hkv, D), generator=g).to(BF16) for _ in range(2))
    for j, pg in enumerate((P - 1, P - 2)):
        kc[pg], vc[pg] = k[j * page:(j + 1) * page].to(DEV), v[j * page:(j + 1) * page].to(DEV)
    q = torch.randn((n, 16, D), generator=g).to(BF16)
    seen = T.ancestors(T.trees(2, [n])[0])
    ref = R.attend(q.double(), k[:100].double(), v[:100].double(), T.visible(seen, 100, 0, 0), 1 / math.sqrt(D))
    out, lse = ops.npu_tree_attention(q.to(DEV), kc, vc, _ints([0, n]).to(DEV), _ints([[P - 1, P - 2]]).to(DEV), _ints([100]).to(DEV),
                                      T.mask_words(seen, 1).to(DEV))
    R.check(out, lse, ref, BF16, 100)


def test_graph_replays_and_streams(ops):
    """Captured with a workspace of its own, replayed with other lengths and trees; and eager calls on two streams at once."""
    print("[case] graph", flush=True)
    g = torch.Generator().manual_seed(5)
    page, Hkv, D, Hq = 16, 2, 64, 8
    lens = [3000, 500]
    kv, table, kc, vc, _, _ = R.pools(lens, page, Hkv, D, BF16, False, g, fill=0.0)
    kd, vd, td = _dev(kc, vc, table)
    forms = []
    for seed, past, sizes in ((1, [2990, 480], [10, 20]), (2, [100, 200], [25, 5]), (3, [2970, 0], [30, 0])):
        rows = [T.ancestors(t) for t in T.trees(seed, sizes)]
        forms.append((_ints([0, sizes[0], 30][:3]).to(DEV), _ints([p + n for p, n in zip(past, sizes)]).to(DEV),
                      T.mask_words([r for rs in rows for r in rs], 1).to(DEV), torch.randn((30, Hq, D), generator=g).to(BF16).to(DEV)))
    cu, ln, mask, q = (t.clone() for t in forms[0])
    want = [ops.npu_tree_attention(f[3], kd, vd, f[0], td, f[1], f[2]) for f in forms]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.npu_tree_attention(q, kd, vd, cu, td, ln, mask)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = ops.npu_tree_attention(q, kd, vd, cu, td, ln, mask)
    for turn in range(2):
        for f, w in zip(forms, want):
            for to, new in zip((cu, ln, mask, q), f):
                to.copy_(new)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w[0]) and torch.equal(lse, w[1])
            again = ops.npu_tree_attention(f[3], kd, vd, f[0], td, f[1], f[2])
            assert torch.equal(again[0], w[0])
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(stream if i % 2 else torch.cuda.current_stream()):
            f = forms[i % 3]
            got.append((i % 3, ops.npu_tree_attention(f[3], kd, vd, f[0], td, f[1], f[2])))
    torch.cuda.synchronize()
    for i, (o, l) in got:
        assert torch.equal(o, want[i][0]) and torch.equal(l, want[i][1])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("sizes", [[16, 3, 15, 11, 5, 7, 1, 1, 3, 5, 5, 16, 2, 3, 3, 9, 3, 9, 13, 3, 11, 2, 9, 11], [40, 1, 64, 33, 20]])
def test_ragged_batches_again_and_again(ops, sizes, dtype):
    """Sequences in one part and in many side by side: each of many passes gives the same, another batch's pass between them."""
    rng = random.Random(len(sizes))
    past = [2000 if i % 6 == 0 else rng.choice([1, 6, 30, 150, 800]) for i in range(len(sizes))]
    first = _run(ops, past, sizes, Hq=32, Hkv=8, D=128, dtype=dtype, page=64, times=40)
    assert first[0].shape[0] == sum(sizes)


def test_no_rows(ops):
    k = torch.zeros((4, 16, 2, 64), dtype=BF16, device=DEV)
    out, lse = ops.npu_tree_attention(torch.zeros((0, 8, 64), dtype=BF16, device=DEV), k, k, _ints([0, 0]).to(DEV),
                                      _ints([[0, 1]]).to(DEV), _ints([5]).to(DEV), torch.zeros((0, 1), dtype=torch.int64, device=DEV))
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)
