"""npu_paged_attention and npu_prompt_attention against attention in 64 bits, where they can go wrong: lengths of zero and
one, pages that end inside a tile, windows and sinks, head counts and widths of every form, caches in other orders,
offsets past 32 bits, and NaN in every place that a row does not see."""
import math

import pytest
import torch

import attention_ref as R

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


def _decode_ref(q, rows, window, sinks, scale):
    parts = [R.attend(q[b:b + 1].double(), k, v, R.visible(1, len(k), window, sinks) if len(k) else
                      torch.zeros((1, 0), dtype=torch.bool), scale) for b, (k, v) in enumerate(rows)]
    return [torch.cat(x) for x in zip(*parts)]


def _hide(rows, table, caches, page, window, sinks, fill):
    """Puts `fill` where no row looks: the tokens that a window of the newest position hides."""
    for b, (k, _) in enumerate(rows):
        n = len(k)
        if n == 0:
            continue
        hidden = (~R.visible(1, n, window, sinks)[0]).nonzero().squeeze(1)
        pg = table[b, hidden // page].long()
        for c in caches:
            if c is not None:
                c[pg, hidden % page] = fill if c.is_floating_point() else 127


def _run_decode(ops, lens, Hq, Hkv, D, page, dtype=BF16, quant=False, window=0, sinks=0, scale=None, order="snd", seed=0):
    print(f"[case] decode lens={lens} Hq={Hq} Hkv={Hkv} D={D} page={page} {dtype} quant={quant} window={window} "
          f"sinks={sinks} {order}", flush=True)
    g = torch.Generator().manual_seed(seed)
    rows, table, kc, vc, ks, vs = R.pools(lens, page, Hkv, D, dtype, quant, g)
    _hide(rows, table, [ks, vs] if quant else [kc, vc], page, window, sinks, math.nan)
    q = torch.randn((len(lens), Hq, D), generator=g).to(dtype)
    ref = _decode_ref(q, rows, window, sinks, scale if scale is not None else 1 / math.sqrt(D))
    kd, vd, ksd, vsd, td, qd = _dev(kc, vc, ks, vs, table, q)
    if order == "nsd":  # heads before tokens inside a page
        kd, vd = (t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (kd, vd))
    elif order == "fused":  # keys and values of a token side by side
        both = torch.cat([kd, vd], dim=2)
        kd, vd = both[:, :, :Hkv], both[:, :, Hkv:]
    out, lse = ops.npu_paged_attention(qd, kd, vd, td, torch.tensor(lens, dtype=torch.int32, device=DEV), key_scale=ksd,
                                       value_scale=vsd, scale=scale, window=window, sinks=sinks)
    assert out.shape == q.shape and out.dtype == dtype and lse.dtype == torch.float32
    R.check(out, lse, ref, dtype, max(lens + [1]), extra_values=int(quant and dtype == F16))
    return out, lse


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens", [[1], [0, 1, 2], [31, 32, 33], [127, 128, 129, 5], [700], [0], [1000, 3, 0, 257]])
def test_decode_lengths(ops, lens, dtype, quant):
    _run_decode(ops, lens, 8, 2, 128, 16, dtype, quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (4, 4), (7, 1), (16, 2), (16, 1), (17, 1), (40, 2), (48, 1)])
def test_decode_heads(ops, Hq, Hkv, quant):
    _run_decode(ops, [77, 300], Hq, Hkv, 64, 16, BF16, quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("D", [8, 16, 32, 40, 64, 72, 80, 96, 112, 128, 160, 192, 200, 256])
def test_decode_widths(ops, D, quant):
    if quant and D % 16:
        pytest.skip("int8 rows are whole 16-byte pieces")
    _run_decode(ops, [65, 130], 6, 2, D, 16, F16, quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("page", [1, 2, 3, 7, 16, 48, 100, 128, 1024])
def test_decode_pages(ops, page, quant):
    _run_decode(ops, [1, 95, 301], 4, 1, 64, page, BF16, quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (33, 4), (100, 40), (64, 1000), (1000, 4), (250, 63)])
def test_decode_window(ops, window, sinks, quant):
    _run_decode(ops, [0, 1, 40, 333, 600], 8, 2, 64, 16, BF16, quant, window, sinks)


@pytest.mark.parametrize("order", ["nsd", "fused"])
@pytest.mark.parametrize("quant", [False, True])
def test_decode_orders(ops, order, quant):
    _run_decode(ops, [200, 33], 8, 4, 64, 16, BF16, quant, order=order)


@pytest.mark.parametrize("lens", [[5000], [4097, 1, 9000, 64, 0, 2500], [300] * 40])
def test_decode_long_and_many(ops, lens):
    """Sequences whose keys are split over workgroups, alone and among short ones."""
    _run_decode(ops, lens, 4, 1, 64, 16, F16)


def test_decode_scale_and_large_scores(ops):
    """Scores of some hundreds: all weight on few keys, the running maximum moves by many steps."""
    _run_decode(ops, [500, 64], 4, 2, 64, 16, BF16, scale=4.0)
    _run_decode(ops, [500, 64], 4, 2, 64, 16, F16, scale=0.0)


@pytest.mark.parametrize("quant", [False, True])
def test_decode_bad_tables(ops, quant):
    """Page ids outside the pool hide their tokens, lengths past the table are cut, negative lengths are empty."""
    print(f"[case] bad tables quant={quant}", flush=True)
    g = torch.Generator().manual_seed(3)
    page, Hkv, D, lens = 16, 2, 64, [100, 64, 40]
    rows, table, kc, vc, ks, vs = R.pools(lens, page, Hkv, D, BF16, quant, g, fill=0.0)
    q = torch.randn((3, 4, D), generator=g).to(BF16)
    table[0, 1], table[0, 3], table[1, :] = -7, 1 << 30, 10 ** 6
    ok = [R.visible(1, n, 0, 0) for n in lens]
    ok[0][:, 16:32] = False
    ok[0][:, 48:64] = False
    ok[1][:] = False
    parts = [R.attend(q[b:b + 1].double(), k, v, ok[b], 1 / 8) for b, (k, v) in enumerate(rows)]
    ref = [torch.cat(x) for x in zip(*parts)]
    kd, vd, ksd, vsd, td, qd = _dev(kc, vc, ks, vs, table, q)
    out, lse = ops.npu_paged_attention(qd, kd, vd, td, torch.tensor(lens, dtype=torch.int32, device=DEV), key_scale=ksd,
                                       value_scale=vsd)
    R.check(out, lse, ref, BF16, 100)
    # lengths: the table holds 3 pages at most here, sequence 2's third page is not full but all its slots are valid rows
    td3 = td[:, :3].contiguous()
    td3[0] = td3[2]
    td3[1] = td3[2]
    k2 = torch.cat([kc[p].double() * (ks[p].double()[..., None] if quant else 1) for p in td3[2].tolist()])
    v2 = torch.cat([vc[p].double() * (vs[p].double()[..., None] if quant else 1) for p in td3[2].tolist()])
    parts = [R.attend(q[0:1].double(), k2, v2, R.visible(1, 48, 0, 0), 1 / 8),
             R.attend(q[1:2].double(), k2, v2, torch.zeros((1, 48), dtype=torch.bool), 1 / 8),
             R.attend(q[2:3].double(), k2, v2, R.visible(1, 48, 0, 0), 1 / 8)]
    ref = [torch.cat(x) for x in zip(*parts)]
    out, lse = ops.npu_paged_attention(qd, kd, vd, td3, torch.tensor([2 ** 31 - 1, -5, 49], dtype=torch.int32, device=DEV),
                                       key_scale=ksd, value_scale=vsd)
    R.check(out, lse, ref, BF16, 48)


def test_decode_large_offsets(ops):
    """A cache whose last pages lie past 2^32 elements."""
    print("[case] large offsets", flush=True)
    P, page, Hkv, D = 66000, 32, 8, 256
    kc = torch.empty((P, page, Hkv, D), dtype=F16, device=DEV)
    vc = torch.empty_like(kc)
    assert kc.numel() > 2 ** 32
    pages = [P - 1, 3, P - 7, 32769, 65000]
    g = torch.Generator().manual_seed(1)
    k = torch.randn((150, Hkv, D), generator=g).to(F16)
    v = torch.randn((150, Hkv, D), generator=g).to(F16)
    for i, p in enumerate(pages):
        n = min(page, 150 - i * page)
        kc[p, :n], vc[p, :n] = k[i * page:i * page + n].to(DEV), v[i * page:i * page + n].to(DEV)
    q = torch.randn((1, 8, D), generator=g).to(F16)
    ref = R.attend(q.double(), k.double(), v.double(), R.visible(1, 150, 0, 0), 1 / 16)
    table = torch.tensor([pages], dtype=torch.int32, device=DEV)
    lens = torch.tensor([150], dtype=torch.int32, device=DEV)
    out, lse = ops.npu_paged_attention(q.to(DEV), kc, vc, table, lens)
    R.check(out, lse, ref, F16, 150)
    out, lse = ops.npu_prompt_attention(q.to(DEV), kc, vc, torch.tensor([0, 1], dtype=torch.int32, device=DEV),
                                        block_table=table, context_lens=lens)
    R.check(out, lse, ref, F16, 150)


def test_decode_nonfinite_seen(ops):
    """An infinity or NaN that a row does see reaches that row, and no other."""
    print("[case] non-finite values in sight", flush=True)
    g = torch.Generator().manual_seed(2)
    rows, table, kc, vc, _, _ = R.pools([50, 50], 16, 1, 64, BF16, False, g, fill=0.0)
    q = torch.randn((2, 2, 64), generator=g).to(BF16)
    vc[table[0, 1].long(), 3, 0, 5] = math.inf
    kc[table[1, 2].long(), 0, 0, 7] = math.nan
    kd, vd, td, qd = _dev(kc, vc, table, q)
    out, lse = ops.npu_paged_attention(qd, kd, vd, td, torch.tensor([50, 50], dtype=torch.int32, device=DEV))
    out = out.float().cpu()
    assert torch.isinf(out[0, :, 5]).all() and torch.isfinite(out[0, :, :5]).all() and torch.isfinite(out[0, :, 6:]).all()
    assert torch.isnan(out[1]).all()


def test_decode_repeats_and_graph(ops):
    """The same bits on every call, on another stream, and in a captured graph replayed among other work."""
    print("[case] graph", flush=True)
    g = torch.Generator().manual_seed(4)
    lens = [3000, 17, 900]
    _, table, kc, vc, _, _ = R.pools(lens, 16, 2, 128, BF16, False, g)
    q = torch.randn((3, 8, 128), generator=g).to(BF16)
    kd, vd, td, qd = _dev(kc, vc, table, q)
    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    first, first_lse = ops.npu_paged_attention(qd, kd, vd, td, ld)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again, _ = ops.npu_paged_attention(qd, kd, vd, td, ld)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_lse = ops.npu_paged_attention(qd, kd, vd, td, ld)
    for i in range(4):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, got) and torch.equal(first_lse, got_lse), f"replay {i}"
        assert torch.equal(ops.npu_paged_attention(qd, kd, vd, td, ld)[0], first)
    ld[0] = 2999  # the captured call reads the lengths where they are
    graph.replay()
    torch.cuda.synchronize()
    want, _ = ops.npu_paged_attention(qd, kd, vd, td, ld)
    assert torch.equal(want, got) and not torch.equal(first, got)


# ---------------------------------------------------------------- prompts


def _run_prompt(ops, q_lens, Hq, Hkv, D, past=None, page=0, dtype=BF16, quant=False, window=0, sinks=0, pad=0, k_lens=None,
                scale=None, seed=0):
    print(f"[case] prompt q={q_lens} past={past} Hq={Hq} Hkv={Hkv} D={D} page={page} {dtype} quant={quant} "
          f"window={window} sinks={sinks} pad={pad}", flush=True)
    g = torch.Generator().manual_seed(seed)
    kv = k_lens or [a + b for a, b in zip(q_lens, past or [0] * len(q_lens))]
    T = sum(q_lens) + pad
    q = torch.randn((T, Hq, D), generator=g).to(dtype)
    rows, table, kc, vc, ks, vs = R.pools(kv, page or 16, Hkv, D, dtype, quant, g)
    s = scale if scale is not None else 1 / math.sqrt(D)
    parts, at = [], 0
    for n, (k, v) in zip(q_lens, rows):
        ok = R.visible(n, len(k), window, sinks) if len(k) else torch.zeros((n, 0), dtype=torch.bool)
        parts.append(R.attend(q[at:at + n].double(), k, v, ok, s))
        at += n
    if pad:
        parts.append(R.attend(q[at:].double(), torch.zeros((0, Hkv, D), dtype=torch.float64),
                              torch.zeros((0, Hkv, D), dtype=torch.float64), torch.zeros((pad, 0), dtype=torch.bool), s))
    ref = [torch.cat(x) for x in zip(*parts)]
    cu = torch.tensor([0] + q_lens, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)
    if page:
        kd, vd, ksd, vsd, td = _dev(kc, vc, ks, vs, table)
        out, lse = ops.npu_prompt_attention(q.to(DEV), kd, vd, cu, block_table=td, scale=scale,
                                            context_lens=torch.tensor(kv, dtype=torch.int32, device=DEV), key_scale=ksd,
                                            value_scale=vsd, window=window, sinks=sinks)
    else:
        # the contiguous rows, taken out of a fused tensor: strides of their own
        both = torch.cat([torch.cat([k, v], dim=1) for k, v in rows]).to(dtype).to(DEV)
        cu_k = None
        if k_lens or past:
            cu_k = torch.tensor([0] + kv, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)
        out, lse = ops.npu_prompt_attention(q.to(DEV), both[:, :Hkv], both[:, Hkv:], cu, cu_seqlens_k=cu_k, scale=scale,
                                            window=window, sinks=sinks)
    R.check(out, lse, ref, dtype, max(kv + [1]), extra_values=int(quant and dtype == F16))
    return out, lse


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("q_lens", [[1], [2, 0, 1], [31, 32, 33], [63, 65], [127, 129], [300], [5, 200, 17, 64, 1]])
def test_prompt_lengths(ops, q_lens, dtype):
    _run_prompt(ops, q_lens, 4, 2, 128, dtype=dtype)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("page", [1, 3, 16, 48, 128])
def test_prompt_paged(ops, page, quant):
    _run_prompt(ops, [70, 1, 33], 4, 2, 64, past=[100, 257, 0], page=page, quant=quant)


@pytest.mark.parametrize("page,quant", [(0, False), (16, False), (16, True)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (33, 4), (100, 40), (64, 1000), (1000, 4), (130, 65)])
def test_prompt_window(ops, window, sinks, page, quant):
    _run_prompt(ops, [150, 40, 3], 4, 2, 64, past=[0, 300, 500] if page else None, page=page, quant=quant, window=window,
                sinks=sinks)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("D", [8, 16, 32, 40, 64, 72, 80, 96, 112, 128, 160, 192, 200, 256])
def test_prompt_widths(ops, D, quant):
    if quant and D % 16:
        pytest.skip("int8 rows are whole 16-byte pieces")
    _run_prompt(ops, [70, 9], 2, 1, D, past=[30, 0], page=16, dtype=F16, quant=quant)
    if not quant:
        _run_prompt(ops, [70, 9], 2, 1, D, dtype=F16)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 3), (7, 1), (12, 2), (17, 1), (48, 1)])
def test_prompt_heads(ops, Hq, Hkv):
    _run_prompt(ops, [40, 90], Hq, Hkv, 64)


def test_prompt_rows_that_see_nothing(ops):
    """More queries than keys (the first stand before the first key), sequences without keys, and rows past the last
    sequence: zeros and -inf."""
    _run_prompt(ops, [40, 10, 3], 2, 1, 64, k_lens=[10, 0, 3], pad=5)
    _run_prompt(ops, [140, 10, 3], 2, 1, 64, k_lens=[70, 0, 3], page=16, pad=150, window=8, sinks=2)
    _run_prompt(ops, [0, 0], 2, 1, 64, k_lens=[10, 0], page=16, pad=3)


def test_prompt_few_rows_long_past(ops):
    """A few new tokens (speculative or the tail of a prompt) over a long past."""
    _run_prompt(ops, [3, 1, 8], 4, 1, 64, past=[3000, 2000, 700], page=16)
    _run_prompt(ops, [5], 8, 1, 128, past=[4000], page=48, dtype=F16, quant=True, window=2000, sinks=4)


def test_prompt_scale_and_large_scores(ops):
    _run_prompt(ops, [200], 2, 1, 64, scale=4.0)
    _run_prompt(ops, [200], 2, 1, 64, scale=0.0, dtype=F16)


@pytest.mark.parametrize("page", [0, 16])
def test_prompt_nonfinite_later(ops, page):
    """NaN and infinities in keys and values that a row does not see (later tokens, tokens before its window) leave it
    alone; rows that see them get them."""
    print(f"[case] non-finite later page={page}", flush=True)
    g = torch.Generator().manual_seed(5)
    n, D, window = 200, 64, 50
    rows, table, kc, vc, _, _ = R.pools([n], 16, 1, D, BF16, False, g)
    q = torch.randn((n, 2, D), generator=g).to(BF16)
    k, v = rows[0]
    ref = R.attend(q.double(), k, v, R.visible(n, n, window, 0), 1 / 8)
    k16, v16 = k.to(BF16), v.to(BF16)
    at_k, at_v, at_i = 70, 100, 131
    for dst_k, dst_v, idx in ([(kc, vc, lambda j: (table[0, j // 16].long(), j % 16))] if page else [(k16, v16, lambda j: (j,))]):
        dst_k[idx(at_k)] = math.nan
        dst_v[idx(at_v)] = math.nan
        dst_v[idx(at_i)] = -math.inf
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    if page:
        out, lse = ops.npu_prompt_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), cu, block_table=table.to(DEV),
                                            context_lens=torch.tensor([n], dtype=torch.int32, device=DEV), window=window)
    else:
        out, lse = ops.npu_prompt_attention(q.to(DEV), k16.to(DEV), v16.to(DEV), cu, window=window)
    i = torch.arange(n)
    sees = lambda j: (i >= j) & (i < j + window)  # noqa: E731
    clean = ~(sees(at_k) | sees(at_v) | sees(at_i))
    R.check(out[clean], lse[clean], [x[clean] for x in ref], BF16, n)
    out = out.float().cpu()
    assert torch.isnan(out[sees(at_k) | sees(at_v)]).all()
    only = sees(at_i) & ~sees(at_k) & ~sees(at_v)
    assert only.any() and torch.isneginf(out[only]).all()


def test_prompt_equals_decode(ops):
    """One new token through either op: both within their bounds of the same reference (checked above); equal lse closely."""
    print("[case] prompt equals decode", flush=True)
    g = torch.Generator().manual_seed(6)
    lens = [90, 333]
    _, table, kc, vc, _, _ = R.pools(lens, 16, 2, 128, BF16, False, g)
    q = torch.randn((2, 8, 128), generator=g).to(BF16)
    kd, vd, td, qd = _dev(kc, vc, table, q)
    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    a, la = ops.npu_paged_attention(qd, kd, vd, td, ld)
    b, lb = ops.npu_prompt_attention(qd, kd, vd, torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), block_table=td,
                                     context_lens=ld)
    assert (la - lb).abs().max() < 1e-4 and (a.float() - b.float()).abs().max() < 0.05


def test_prompt_graph(ops):
    print("[case] prompt graph", flush=True)
    g = torch.Generator().manual_seed(7)
    n = 300
    q, k, v = (torch.randn((n, h, 128), generator=g).to(BF16).to(DEV) for h in (4, 2, 2))
    cu = torch.tensor([0, 130, 300], dtype=torch.int32, device=DEV)
    first, _ = ops.npu_prompt_attention(q, k, v, cu, window=64, sinks=2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = ops.npu_prompt_attention(q, k, v, cu, window=64, sinks=2)
    for i in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, got), f"replay {i}"
        assert torch.equal(ops.npu_prompt_attention(q, k, v, cu, window=64, sinks=2)[0], first)


def test_query_forms(ops):
    """Queries out of a fused projection, of odd strides and alignment, and empty batches."""
    print("[case] query forms", flush=True)
    g = torch.Generator().manual_seed(8)
    lens = [40, 7]
    _, table, kc, vc, _, _ = R.pools(lens, 16, 2, 64, BF16, False, g)
    kd, vd, td = _dev(kc, vc, table)
    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    wide = torch.randn((2, 4 * 64 + 3), generator=g).to(BF16).to(DEV)
    base = torch.randn((2, 8, 64), generator=g).to(BF16).to(DEV)
    for q in (base[:, :4], base[:, 1::2], wide[:, 3:].view(2, 4, 64), base[:, :4].transpose(1, 2).contiguous().transpose(1, 2)):
        want, want_lse = ops.npu_paged_attention(q.contiguous(), kd, vd, td, ld)
        got, got_lse = ops.npu_paged_attention(q, kd, vd, td, ld)
        assert torch.equal(want, got) and torch.equal(want_lse, got_lse)
    out, lse = ops.npu_paged_attention(base[:0, :4], kd, vd, td[:0], ld[:0])
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    out, _ = ops.npu_prompt_attention(base[:0, :4], base[:0, :2], base[:0, :2], torch.tensor([0, 0], dtype=torch.int32, device=DEV))
    assert out.shape == (0, 4, 64)
    out, lse = ops.npu_paged_attention(base[:, :4], kd, vd, td[:, :0], ld)  # a table without columns
    assert (out == 0).all() and torch.isneginf(lse).all()
