"""npu_mrope and npu_mrope_scatter_kv: the rotation against 64 bits, its bits against 32-bit arithmetic in the stated order,
the cache write, the int8 cache against npu_dynamic_quant, and the places a bad index must not touch."""
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


def _inputs(T, Hq, Hkv, D, rot, axes, dtype, seed=0, far=5000):
    g = torch.Generator().manual_seed(seed)
    angle = torch.arange(far, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    table = torch.cat([angle.cos(), angle.sin()], 1).float()
    q, k, v = (torch.randn((T, h, D), generator=g).to(dtype) for h in (Hq, Hkv, Hkv))
    positions = torch.randint(0, far, (axes, T), generator=g, dtype=torch.int32)
    half = rot // 2
    cut = sorted(torch.randint(0, half + 1, (axes - 1,), generator=g).tolist())
    sections = [b - a for a, b in zip([0] + cut, cut + [half])]
    return q, k, v, table, positions, sections


def _same_bits(x, positions, table, sections, mode):
    """The rotation in 32 bits, each product and sum rounded, then one rounding to x's type."""
    half = table.shape[1] // 2
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)])
    at = positions.long()[axis].t()
    i = torch.arange(half)
    c, s = table[at, i].float()[:, None], table[at, half + i].float()[:, None]
    y = x.clone()
    e0, e1 = (i, i + half) if mode == "half" else (2 * i, 2 * i + 1)
    x0, x1 = x[..., e0].float(), x[..., e1].float()
    y[..., e0], y[..., e1] = (x0 * c - x1 * s).to(x.dtype), (x1 * c + x0 * s).to(x.dtype)
    return y


FORMS = [  # T, Hq, Hkv, D, rotary, axes, mode
    (1, 32, 8, 128, 128, 1, "half"), (7, 4, 2, 128, 128, 3, "half"), (33, 5, 1, 64, 32, 3, "half"),
    (9, 3, 3, 80, 80, 2, "half"), (6, 2, 1, 96, 48, 4, "half"), (5, 2, 2, 256, 256, 3, "half"), (4, 2, 1, 72, 40, 3, "half"),
    (3, 3, 1, 8, 2, 1, "half"), (700, 4, 2, 128, 128, 3, "half"), (11, 2, 2, 256, 2, 1, "half"),
    (7, 4, 2, 128, 128, 3, "interleave"), (5, 3, 1, 64, 16, 1, "interleave"), (4, 2, 1, 40, 20, 2, "interleave"),
    (5, 2, 2, 256, 256, 3, "interleave"), (600, 48, 1, 128, 64, 3, "interleave"), (130, 70, 3, 64, 64, 1, "half"),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("form", FORMS)
def test_mrope(ops, form, dtype):
    T, Hq, Hkv, D, rot, axes, mode = form
    print(f"[case] mrope {form} {dtype}", flush=True)
    q, k, _, table, positions, sections = _inputs(T, Hq, Hkv, D, rot, axes, dtype)
    if axes == 1:
        pos, sec = positions[0], None
    else:
        pos, sec = positions, sections
    oq, ok = ops.npu_mrope(pos.to(DEV), q.to(DEV), k.to(DEV), table.to(DEV), mrope_section=sec, rotary_mode=mode)
    for x, y in ((q, oq), (k, ok)):
        y = y.cpu()
        assert torch.equal(y, _same_bits(x, positions, table, sections, mode))
        # one rounding to 16 bits of two rounded products and a rounded sum
        ref = R.rotate(x, positions, table, sections, mode)
        tol = R.half_step(dtype) * ref.abs() + 4 * 2.0 ** -24 * 2 * x.double().abs().amax() + 2.0 ** -25
        assert ((y.double() - ref).abs() <= tol).all()
    t16 = table.to(dtype)  # a table of the tensors' type
    oq, _ = ops.npu_mrope(pos.to(DEV), q.to(DEV), k.to(DEV), t16.to(DEV), mrope_section=sec, rotary_mode=mode)
    assert torch.equal(oq.cpu(), _same_bits(q, positions, t16, sections, mode))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("form", FORMS)
def test_scatter(ops, form, dtype, quant):
    T, Hq, Hkv, D, rot, axes, mode = form
    if quant and D % 16:
        pytest.skip("int8 rows are whole 16-byte pieces")
    print(f"[case] scatter {form} {dtype} quant={quant}", flush=True)
    q, k, v, table, positions, sections = _inputs(T, Hq, Hkv, D, rot, axes, dtype, seed=1)
    page = 48 if T > 100 else 3
    P = -(-T // page) + 2
    g = torch.Generator().manual_seed(9)
    slots = torch.randperm(P * page, generator=g)[:T].to(torch.int32)
    if T > 2:
        slots[0], slots[T // 2], slots[T - 1] = -1, P * page, 2 ** 31 - 1  # padding tokens
    fused = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1).to(DEV)  # the projection's output; views of it below
    qd, kd, vd = (t.view(T, -1, D) for t in fused.split([Hq * D, Hkv * D, Hkv * D], 1))
    kind = torch.int8 if quant else dtype
    kc, vc = (torch.full((P, page, Hkv, D), 7, dtype=kind, device=DEV) for _ in range(2))
    ks, vs = (torch.full((P, page, Hkv), -1.0, device=DEV) for _ in range(2)) if quant else (None, None)
    pos, sec = (positions[0], None) if axes == 1 else (positions, sections)
    oq = ops.npu_mrope_scatter_kv(pos.to(DEV), qd, kd, vd, table.to(DEV), kc, vc, slots.to(DEV), key_scale=ks,
                                  value_scale=vs, mrope_section=sec, rotary_mode=mode)
    want_q, want_k = (_same_bits(x, positions, table, sections, mode) for x in (q, k))
    assert torch.equal(oq.cpu(), want_q)
    put = (slots >= 0) & (slots < P * page)
    for cache, scales, rows in ((kc, ks, want_k), (vc, vs, v)):
        want = torch.full((P * page, Hkv, D), 7, dtype=kind)
        if quant:
            y, s = ops.npu_dynamic_quant(rows.to(DEV))
            want[slots[put].long()] = y.cpu()[put]
            want_s = torch.full((P * page, Hkv), -1.0)
            want_s[slots[put].long()] = s.cpu()[put]
            assert torch.equal(scales.cpu().flatten(0, 1), want_s)
        else:
            want[slots[put].long()] = rows[put]
        assert torch.equal(cache.cpu().flatten(0, 1), want)


def test_scatter_orders(ops):
    """Caches whose pages hold heads before tokens, and keys and values side by side in one tensor."""
    print("[case] scatter orders", flush=True)
    q, k, v, table, positions, _ = _inputs(20, 4, 2, 64, 64, 1, BF16, seed=2)
    slots = torch.arange(5, 25, dtype=torch.int32)
    want = _same_bits(k, positions, table, [32], "half")
    both = torch.zeros((4, 2, 2, 16, 64), dtype=BF16, device=DEV)  # [pages, key or value, heads, tokens, D]
    kc, vc = (both[:, i].permute(0, 2, 1, 3) for i in range(2))
    ops.npu_mrope_scatter_kv(positions[0].to(DEV), q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), kc, vc, slots.to(DEV))
    got_k, got_v = (t.reshape(64, 2, 64).cpu() for t in (kc, vc))
    assert torch.equal(got_k[5:25], want) and torch.equal(got_v[5:25], v)
    assert (got_k[:5] == 0).all() and (got_k[25:] == 0).all() and (got_v[25:] == 0).all()


def test_bad_positions(ops):
    """A position outside the table gives NaN pairs in its own section and nothing else."""
    print("[case] bad positions", flush=True)
    q, k, _, table, positions, _ = _inputs(6, 2, 1, 64, 32, 3, F16, seed=3)
    sections = [4, 6, 6]
    positions[0, 1], positions[1, 3], positions[2, 3] = -1, table.shape[0], 2 ** 31 - 1
    oq, ok = ops.npu_mrope(positions.to(DEV), q.to(DEV), k.to(DEV), table.to(DEV), mrope_section=sections)
    safe = positions.clamp(0, table.shape[0] - 1)
    for x, y in ((q, oq), (k, ok)):
        want = _same_bits(x, safe, table, sections, "half")
        for t, lo, hi in ((1, 0, 4), (3, 4, 16)):
            want[t, :, lo:hi] = math.nan
            want[t, :, 16 + lo:16 + hi] = math.nan
        y = y.cpu()
        assert torch.equal(torch.isnan(y), torch.isnan(want))
        assert torch.equal(y.nan_to_num(), want.nan_to_num())


def test_unaligned_and_strided(ops):
    """Inputs at odd offsets and strides: the same bits."""
    print("[case] unaligned", flush=True)
    q, k, v, table, positions, _ = _inputs(9, 4, 2, 64, 64, 1, BF16, seed=4)
    want_q, want_k = (_same_bits(x, positions, table, [32], "half") for x in (q, k))
    wide = torch.zeros((9, 4 * 64 + 5), dtype=BF16, device=DEV)
    wide[:, 5:] = q.flatten(1).to(DEV)
    kt = k.to(DEV).permute(2, 0, 1).contiguous().permute(1, 2, 0)  # last dimension not dense
    oq, ok = ops.npu_mrope(positions[0].to(DEV), wide[:, 5:].view(9, 4, 64), kt, table.to(DEV))
    assert torch.equal(oq.cpu(), want_q) and torch.equal(ok.cpu(), want_k)


def test_scatter_graph(ops):
    print("[case] scatter graph", flush=True)
    q, k, v, table, positions, _ = _inputs(12, 4, 2, 64, 64, 1, BF16, seed=5)
    kc, vc = (torch.zeros((2, 16, 2, 64), dtype=BF16, device=DEV) for _ in range(2))
    args = [t.to(DEV) for t in (positions[0], q, k, v, table)]
    slots = torch.arange(12, dtype=torch.int32, device=DEV)
    ops.npu_mrope_scatter_kv(*args, kc, vc, slots)
    first = kc.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.npu_mrope_scatter_kv(*args, kc, vc, slots)
    for i in range(3):
        kc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kc, first), f"replay {i}"
