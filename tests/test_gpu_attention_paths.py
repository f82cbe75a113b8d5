"""The attention ops where their work is cut and joined, and where masks meet bad pages, values that are not finite, odd scales and
scales of an int8 cache far apart: against attention in 64 bits, with the bounds of attention_ref.check."""
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


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _decode(ops, lens, Hq, Hkv, D, page, dtype=BF16, quant=False, window=0, sinks=0, scale=None, spread=None, seed=0):
    print(f"[case] decode n={len(lens)} longest={max(lens)} Hq={Hq} Hkv={Hkv} D={D} page={page} {dtype} quant={quant} "
          f"window={window} scale={scale} spread={spread}", flush=True)
    g = torch.Generator().manual_seed(seed)
    rows, table, kc, vc, ks, vs = R.pools(lens, page, Hkv, D, dtype, quant, g, fill=0.0)
    if spread is not None:  # scales of the values from token to token far apart, some of them 0
        f = 10.0 ** (spread * (2 * torch.rand(vs.shape, generator=g) - 1))
        f[torch.rand(vs.shape, generator=g) < 0.1] = 0.0
        vs = (vs * f).float()
        rows = [(k, (vc[table[b, torch.arange(len(k)) // page].long(), torch.arange(len(k)) % page].double() *
                     vs[table[b, torch.arange(len(k)) // page].long(), torch.arange(len(k)) % page].double()[..., None]))
                for b, (k, _) in enumerate(rows)]
    q = torch.randn((len(lens), Hq, D), generator=g).to(dtype)
    s = scale if scale is not None else 1 / math.sqrt(D)
    parts = [R.attend(q[b:b + 1].double(), k, v, R.visible(1, len(k), window, sinks) if len(k) else
                      torch.zeros((1, 0), dtype=torch.bool), s) for b, (k, v) in enumerate(rows)]
    ref = [torch.cat(x) for x in zip(*parts)]
    if scale is not None and scale < 0:  # the size that roundings of the scores act on has no sign
        ref[3] = ref[3].abs()
    kd, vd, ksd, vsd, td, qd = _dev(kc, vc, ks, vs, table, q)
    call = lambda: ops.npu_paged_attention(qd, kd, vd, td, _ints(lens), key_scale=ksd, value_scale=vsd, scale=scale,  # noqa: E731
                                           window=window, sinks=sinks)
    out, lse = call()
    R.check(out, lse, ref, dtype, max(lens + [1]), extra_values=int(quant and dtype == F16))
    again, _ = call()
    assert torch.equal(out, again)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("lens,Hq,Hkv,D", [([20000], 4, 1, 64), ([9000, 40, 7000], 6, 2, 128), ([12000], 40, 1, 64),
                                           ([5000], 2, 1, 256)])
def test_decode_many_parts(ops, lens, Hq, Hkv, D, quant):
    """More parts of one sequence than are joined at a time, alone and beside short sequences."""
    _decode(ops, lens, Hq, Hkv, D, 16, F16 if quant else BF16, quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("n", [64, 65, 100, 300])
def test_decode_batches(ops, n, quant):
    """Around and past the batch that a wave scans by itself, empty and one-token sequences among them."""
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 90, (n,), generator=g).tolist()
    lens[0], lens[n // 2], lens[-1] = 0, 1500, 1
    _decode(ops, lens, 2, 1, 64, 16, BF16, quant, window=200 if n == 100 else 0, sinks=3)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("spread", [1, 3])
def test_decode_scales_far_apart(ops, dtype, spread):
    _decode(ops, [300, 64], 4, 2, 64, 16, dtype, True, spread=spread)


@pytest.mark.parametrize("quant", [False, True])
def test_decode_negative_scale(ops, quant):
    _decode(ops, [200, 33], 4, 2, 64, 16, BF16, quant, scale=-0.2)


def _prompt(ops, q_lens, past, Hq, Hkv, D, page, dtype=BF16, quant=False, window=0, sinks=0, scale=None, lose=(), spread=None,
            seed=0):
    print(f"[case] prompt q={q_lens} past={past} Hq={Hq} Hkv={Hkv} D={D} page={page} {dtype} quant={quant} window={window} "
          f"sinks={sinks} scale={scale} lose={lose} spread={spread}", flush=True)
    g = torch.Generator().manual_seed(seed)
    kv = [a + b for a, b in zip(q_lens, past)]
    rows, table, kc, vc, ks, vs = R.pools(kv, page, Hkv, D, dtype, quant, g, fill=0.0)
    at = lambda b: (table[b, torch.arange(kv[b]) // page].long(), torch.arange(kv[b]) % page)  # noqa: E731
    if spread is not None:
        f = 10.0 ** (spread * (2 * torch.rand(vs.shape, generator=g) - 1))
        f[torch.rand(vs.shape, generator=g) < 0.1] = 0.0
        vs = (vs * f).float()
        rows = [(k, vc[at(b)].double() * vs[at(b)].double()[..., None]) for b, (k, _) in enumerate(rows)]
    q = torch.randn((sum(q_lens), Hq, D), generator=g).to(dtype)
    s = scale if scale is not None else 1 / math.sqrt(D)
    parts, first = [], 0
    for b, (n, (k, v)) in enumerate(zip(q_lens, rows)):
        ok = R.visible(n, len(k), window, sinks)
        for p in lose:
            if p * page < len(k):
                ok[:, p * page:(p + 1) * page] = False
        parts.append(R.attend(q[first:first + n].double(), k, v, ok, s))
        first += n
    ref = [torch.cat(x) for x in zip(*parts)]
    if scale is not None and scale < 0:
        ref[3] = ref[3].abs()
    for i, p in enumerate(lose):
        table[:, min(p, table.shape[1] - 1)] = (-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1)[i % 4]
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    kd, vd, ksd, vsd, td, qd = _dev(kc, vc, ks, vs, table, q)
    call = lambda: ops.npu_prompt_attention(qd, kd, vd, _ints(cu), block_table=td, context_lens=_ints(kv), key_scale=ksd,  # noqa: E731
                                            value_scale=vsd, scale=scale, window=window, sinks=sinks)
    out, lse = call()
    R.check(out, lse, ref, dtype, max(kv), extra_values=int(quant and dtype == F16))
    again, _ = call()
    assert torch.equal(out, again)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("q_lens,past,Hq,Hkv,D", [([40], [3000], 4, 1, 64), ([3, 1], [2500, 700], 2, 1, 256),
                                                  ([2], [4000], 24, 1, 128), ([33, 0, 5], [1100, 10, 2000], 6, 2, 192),
                                                  ([5], [1500], 2, 2, 96)])
def test_prompt_parts(ops, q_lens, past, Hq, Hkv, D, quant):
    """Few rows over a long past: the keys are cut and joined."""
    _prompt(ops, q_lens, past, Hq, Hkv, D, 16, F16 if quant else BF16, quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("window,sinks", [(700, 0), (1500, 70), (64, 4)])
def test_prompt_parts_window(ops, window, sinks, quant):
    _prompt(ops, [30, 4], [2500, 900], 4, 2, 64, 48, BF16, quant, window, sinks)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("past", [0, 3000])
def test_prompt_bad_pages(ops, past, quant):
    """Page ids outside the pool, at the front, inside and at the end of a sequence, hide their tokens."""
    _prompt(ops, [70, 20], [past, 30], 4, 2, 64, 16, BF16, quant, lose=(0, 2, 3, 5))
    _prompt(ops, [40], [past], 2, 1, 64, 16, BF16, quant, window=33, sinks=20, lose=(1, (past + 39) // 16))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prompt_scales_far_apart(ops, dtype):
    _prompt(ops, [150, 9], [0, 400], 4, 2, 64, 16, dtype, True, spread=2)
    _prompt(ops, [9], [2000], 4, 2, 64, 16, dtype, True, window=900, sinks=4, spread=2)


@pytest.mark.parametrize("quant", [False, True])
def test_prompt_odd_factors(ops, quant):
    _prompt(ops, [90], [40], 4, 2, 64, 16, BF16, quant, scale=-0.2)
    _prompt(ops, [90], [40], 4, 2, 64, 16, F16, quant, scale=0.0)
    _prompt(ops, [9], [2000], 4, 2, 64, 16, F16, quant, scale=2.0)


@pytest.mark.parametrize("past", [0, 3000])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_prompt_values_not_finite(ops, D, dtype, past):
    """A NaN or an infinity in an element of V reaches the rows that see its token, in that element, and nothing else."""
    print(f"[case] not finite D={D} {dtype} past={past}", flush=True)
    g = torch.Generator().manual_seed(11)
    n, window = 90, 60
    total = n + past
    rows, table, kc, vc, _, _ = R.pools([total], 16, 1, D, dtype, False, g, fill=0.0)
    q = torch.randn((n, 3, D), generator=g).to(dtype)
    spots = [(past + 20, 3, math.nan), (past + 50, 7, math.inf), (past + 51, D - 1, -math.inf)]
    k, v = rows[0]
    ref = R.attend(q.double(), k, v, R.visible(n, total, window, 0), 1 / math.sqrt(D))
    for j, d, bad in spots:
        vc[table[0, j // 16].long(), j % 16, 0, d] = bad
    out, lse = ops.npu_prompt_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), _ints([0, n]), block_table=table.to(DEV),
                                        context_lens=_ints([total]), window=window)
    out = out.cpu()
    i = torch.arange(past, total)
    dirty = torch.zeros_like(out, dtype=torch.bool)
    for j, d, bad in spots:
        sees = (i >= j) & (i < j + window)
        assert sees.any() and not sees.all()
        dirty[sees, :, d] = True
        assert (torch.isnan(out[sees, :, d]) if bad != bad else out[sees, :, d] == bad).all(), (j, d, bad)
    clean = torch.where(dirty, ref[0].to(dtype), out)
    R.check(clean, lse, ref, dtype, total)


def test_prompt_parts_graph(ops):
    """Parts and their counters in a captured graph, replayed among eager calls of the same op."""
    print("[case] prompt parts graph", flush=True)
    g = torch.Generator().manual_seed(7)
    _, table, kc, vc, _, _ = R.pools([2600, 900], 16, 1, 128, BF16, False, g)
    q = torch.randn((7, 4, 128), generator=g).to(BF16)
    qd, kd, vd, td, cu, lens = *_dev(q, kc, vc, table), _ints([0, 4, 7]), _ints([2600, 900])
    call = lambda: ops.npu_prompt_attention(qd, kd, vd, cu, block_table=td, context_lens=lens)  # noqa: E731
    first, _ = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = call()
    for i in range(4):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, got), f"replay {i}"
        assert torch.equal(call()[0], first)


def test_sizes_refused(ops):
    """Sequences whose tokens the kernels could not count in 32 bits (refused before any launch)."""
    print("[case] sizes refused", flush=True)
    k = torch.empty((1, 1, 1, 16), dtype=BF16, device=DEV).expand(1, 2 ** 31 - 1, 1, 16)
    q = torch.empty((1, 1, 16), dtype=BF16, device=DEV)
    with pytest.raises(RuntimeError, match="31 bits"):
        ops.npu_paged_attention(q, k, k, _ints([[0]]), _ints([1]))
    with pytest.raises(RuntimeError, match="31 bits"):
        ops.npu_prompt_attention(q, k[0], k[0], _ints([0, 1]))
