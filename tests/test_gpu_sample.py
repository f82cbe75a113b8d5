"""npu_sample against the definition in 64 bits, row by row: every filter alone and together, ties at every border, masked logits
of every kind, settings at their ends, rows of every length and alignment."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TYPES = [F16, BF16, F32]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import op_plugin_amd
    return op_plugin_amd


def _row(x, u, t, k, p, m):
    """(tokens that may be drawn, logprob of each) of one row, x float64.

    The kernel's weights are whole multiples of 2^-F of the largest, half a unit off each, so a sum of n of them is off by
    n * 2^-(F + 1) at most, and the exponentials by some roundings of 64 bits: 2^-50 of the sum.  A token whose border lies that near
    the drawn number may be the one before or behind."""
    n = len(x)
    x = np.where(np.isnan(x), -np.inf, x)
    if np.isneginf(x).all():
        return {-1: -math.inf}
    order = np.argsort(-x, kind="stable")
    if not t > 0:
        return {int(order[0]): 0.0}
    top = x.max()
    with np.errstate(invalid="ignore"):
        away = np.where(x == top, 0.0, np.where(np.isneginf(x), np.inf, (top - x) / t if np.isfinite(t) else 0.0))
        if np.isinf(top):
            away = np.where(x == top, 0.0, np.inf)
    w = np.exp(-away)[order]
    keep = np.arange(n) < (k if k > 0 else n)
    if p < 1:
        total = math.fsum(w[keep])
        before = np.cumsum(w) - w
        keep &= (before < p * total) | (np.arange(n) == 0)
    if m > 0:
        keep &= (away[order] <= -math.log(min(m, 1.0)))
    kept = np.zeros(n, bool)
    kept[order[keep]] = True
    w = np.exp(-away) * kept
    total = math.fsum(w)
    sums = np.cumsum(w)
    F = min(50, 62 - math.ceil(math.log2(n)) if n > 1 else 50)
    slack = n * 2.0 ** -(F + 1) + 2.0 ** -50 * total
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    found = {}
    for i in np.nonzero(kept & (w > 0) & (sums + slack > u * total) & (sums - w - slack <= u * total))[0]:
        found[int(i)] = math.log(w[i] / total)
    return found


def _check(ops, x, u, t=None, k=None, p=None, m=None):
    R, V = x.shape
    print(f"[case] sample {R} x {V} {x.dtype} t={t is not None} k={k is not None} p={p is not None} m={m is not None}", flush=True)
    dev = lambda v, dt: None if v is None else torch.as_tensor(v, dtype=dt).expand(R).contiguous().to(DEV)  # noqa: E731
    u, t, p, m, k = dev(u, F32), dev(t, F32), dev(p, F32), dev(m, F32), dev(k, torch.int32)
    tokens, logprobs = ops.npu_sample(x.to(DEV), u, temperature=t, top_k=k, top_p=p, min_p=m)
    assert tokens.dtype == torch.int32 and logprobs.dtype == F32 and tokens.shape == logprobs.shape == (R,)
    at = lambda v, r, d: d if v is None else float(v[r])  # noqa: E731
    rows = x.double().cpu().numpy()
    for r in range(R):
        found = _row(rows[r], float(u[r]), at(t, r, 1.0), int(at(k, r, 0)), at(p, r, 1.0), at(m, r, 0.0))
        got, lp = int(tokens[r]), float(logprobs[r])
        assert got in found, (r, got, found)
        want = found[got]
        if math.isinf(want):
            assert lp == want
        else:
            # rounded once to 32 bits; before that, what the weights' sum is off by
            tol = abs(want) * 2.0 ** -24 + V * 2.0 ** -40 + 2.0 ** -149
            assert abs(lp - want) <= tol, (r, lp, want)
    return tokens, logprobs


def _logits(g, R, V, dtype, scale=2.5, peaks=6):
    x = scale * torch.randn((R, V), generator=g)
    if peaks:
        x.scatter_(1, torch.randint(0, V, (R, peaks), generator=g), 5 + 6 * torch.rand((R, peaks), generator=g))
    return x.to(dtype)


def _settings(g, R, V):
    pick = lambda vs: torch.tensor(vs)[torch.randint(0, len(vs), (R,), generator=g)]  # noqa: E731
    return dict(t=pick([0.0, 0.5, 0.8, 1.0, 1.5]), k=pick([0, 1, 3, 20, 50, V, 5 * V]), p=pick([1.0, 0.5, 0.9, 0.95, 0.999]),
                m=pick([0.0, 0.01, 0.1, 0.5]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 3, 7, 63, 64, 65, 1000, 1023, 1024, 1025, 4097, 32001, 70000])
def test_lengths(ops, V, dtype):
    g = torch.Generator().manual_seed(V)
    _check(ops, _logits(g, 9, V, dtype), torch.rand(9, generator=g), **_settings(g, 9, V))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("filters", ["", "t", "k", "p", "m", "kp", "tpm", "tkpm"])
def test_filters(ops, filters, dtype):
    g = torch.Generator().manual_seed(5)
    R, V = 40, 5003
    s = _settings(g, R, V)
    _check(ops, _logits(g, R, V, dtype), torch.rand(R, generator=g), **{f: s[f] for f in filters})


@pytest.mark.parametrize("R", [1, 2, 3, 16, 64, 65, 130, 300, 600])
def test_rows(ops, R):
    """Few rows, whose work is split, to more rows than the card has places."""
    g = torch.Generator().manual_seed(R)
    _check(ops, _logits(g, R, 9001, BF16), torch.rand(R, generator=g), **_settings(g, R, 9001))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("values", [1, 2, 5, 40])
def test_ties(ops, values, dtype):
    """Logits of few values: borders inside a run of equal ones, which stay by their index."""
    g = torch.Generator().manual_seed(values)
    for V in (50, 3001, 40000):
        x = torch.randint(0, values, (24, V), generator=g).to(dtype)
        x[::5, ::3] = -0.0 if values == 1 else 0.0
        s = _settings(g, 24, V)
        s["k"][::3] = V // 3
        s["t"] = s["t"].clamp(min=0.5)
        _check(ops, x, torch.rand(24, generator=g), **s)
        _check(ops, x, torch.rand(24, generator=g), k=s["k"])
        _check(ops, x, torch.rand(24, generator=g), p=torch.full((24,), 0.37))


def test_equal_weights_are_drawn_evenly(ops):
    """All logits equal: token floor(u V); of the first half, floor(u V / 2)."""
    V = 4096
    u = (torch.arange(V) + 0.5) / V
    x = torch.full((V, V), 1.25, dtype=BF16, device=DEV)
    tokens, lp = ops.npu_sample(x, u.to(DEV))
    assert torch.equal(tokens.cpu(), torch.arange(V, dtype=torch.int32))
    assert (lp.cpu() - -math.log(V)).abs().max() < 2.0 ** -20
    half = torch.full((V,), 0.5, device=DEV)
    tokens, _ = ops.npu_sample(x, u.to(DEV), top_p=half)
    assert torch.equal(tokens.cpu(), (torch.arange(V) // 2).to(torch.int32))
    tokens, _ = ops.npu_sample(x, u.to(DEV), top_k=torch.full((V,), V // 2, dtype=torch.int32, device=DEV))
    assert torch.equal(tokens.cpu(), (torch.arange(V) // 2).to(torch.int32))


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_logits(ops, dtype):
    g = torch.Generator().manual_seed(2)
    R, V = 20, 3000
    low = torch.finfo(dtype).min
    for fill in (-math.inf, math.nan, low):
        x = _logits(g, R, V, dtype)
        x[:, torch.rand(V, generator=g) < 0.7] = fill
        x[3] = fill
        x[4, 1:] = fill
        x[5, :-1] = fill
        x[6, 7] = low
        s = _settings(g, R, V)
        _check(ops, x, torch.rand(R, generator=g), **s)
        _check(ops, x, torch.rand(R, generator=g))
        _check(ops, x, torch.rand(R, generator=g), k=torch.full((R,), 2500), p=torch.full((R,), 0.99))


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_logits(ops, dtype):
    """All weight on the infinite ones, in equal parts."""
    g = torch.Generator().manual_seed(3)
    x = _logits(g, 12, 500, dtype)
    x[:, 17] = math.inf
    x[4:, 400] = math.inf
    x[8:, 401:450] = math.inf
    x[:, 30] = -math.inf
    x[:, 31] = math.nan
    s = _settings(g, 12, 500)
    _check(ops, x, torch.rand(12, generator=g), **s)
    _check(ops, x, torch.rand(12, generator=g))
    _check(ops, x, torch.rand(12, generator=g), t=torch.full((12,), math.inf), k=torch.full((12,), 20))


def test_ends_of_settings(ops):
    g = torch.Generator().manual_seed(4)
    R, V = 30, 2000
    x = _logits(g, R, V, F32)
    u = torch.rand(R, generator=g)
    u[:6] = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan])
    for t in (0.0, -1.0, math.nan, 1e-45, 1e-30, 1e-3, 1e4, 1e30, math.inf):
        _check(ops, x, u, t=torch.full((R,), t))
        _check(ops, x, u, t=torch.full((R,), t), k=torch.full((R,), 40), p=torch.full((R,), 0.7))
    for k in (-1, 0, 1, V - 1, V, V + 1, 2 ** 31 - 1):
        _check(ops, x, u, k=torch.full((R,), k))
    for p in (-1.0, 0.0, 1e-30, 1e-3, 1 - 2.0 ** -24, 1.0, 7.0, math.nan):
        _check(ops, x, u, p=torch.full((R,), p))
        _check(ops, x, u, p=torch.full((R,), p), k=torch.full((R,), 9))
    for m in (-1.0, 0.0, 1e-40, 1e-6, 1.0, 3.0, math.nan):
        _check(ops, x, u, m=torch.full((R,), m))
        _check(ops, x, u, m=torch.full((R,), m), p=torch.full((R,), 0.9))


def test_far_logits(ops):
    """Differences that pass the range of 32 bits, values of the smallest size, and one peak above a flat rest."""
    g = torch.Generator().manual_seed(6)
    x = torch.zeros((8, 3000))
    x[0] = torch.linspace(-3e38, 3e38, 3000)
    x[1] = 1e-44 * torch.randint(0, 5, (3000,), generator=g)
    x[2] = 1000.0 + torch.randint(0, 3, (3000,), generator=g) * 2.0 ** -14
    x[3, 777] = 50.0
    x[4, 777] = 9.0
    x[5] = -1e5 - torch.rand(3000, generator=g)
    x[6] = torch.randn(3000, generator=g) * 1e-6
    u = torch.rand(8, generator=g)
    _check(ops, x, u)
    for p in (0.3, 0.9, 0.9999):
        _check(ops, x, u, p=torch.full((8,), p))
        _check(ops, x, u, t=torch.full((8,), 1e-3), p=torch.full((8,), p), k=torch.full((8,), 1500))
    _check(ops, x, u, t=torch.full((8,), 1e38), m=torch.full((8,), 0.5))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_lie_anywhere(ops, dtype):
    """Rows at odd elements, apart, the same row for all, and columns that are not dense."""
    g = torch.Generator().manual_seed(7)
    big = _logits(g, 12, 6007, dtype).to(DEV)
    s = _settings(g, 12, 5001)
    u = torch.rand(12, generator=g)
    for view in (big[:, 1:5002], big[:, 3:5004], big[:, 7:5008], big[3:4, 5:5006].expand(12, 5001), big[:, ::2],
                 big.t().contiguous().t()[:, :999]):
        _check(ops, view, u, **s)


def test_same_call_twice_and_streams(ops):
    g = torch.Generator().manual_seed(8)
    x = _logits(g, 33, 50000, BF16).to(DEV)
    s = {k: v.to(DEV) for k, v in _settings(g, 33, 50000).items()}
    u = torch.rand(33, generator=g).to(DEV)
    kw = dict(temperature=s["t"], top_k=s["k"].to(torch.int32), top_p=s["p"], min_p=s["m"])
    want = ops.npu_sample(x, u, **kw)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i in range(9):
        with torch.cuda.stream(streams[i % 3]):
            got.append(ops.npu_sample(x, u, **kw))
    torch.cuda.synchronize()
    for a in got:
        assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1])


@pytest.mark.parametrize("R", [1, 20, 400])
def test_graph_replays(ops, R):
    g = torch.Generator().manual_seed(9)
    V = 20011
    x, u = torch.empty((R, V), dtype=F16, device=DEV), torch.empty(R, device=DEV)
    s = {k: v.to(DEV) for k, v in _settings(g, R, V).items()}
    kw = dict(temperature=s["t"], top_k=s["k"].to(torch.int32), top_p=s["p"], min_p=s["m"])
    x.zero_(), u.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.npu_sample(x, u, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, lp = ops.npu_sample(x, u, **kw)
    for i in range(4):
        x.copy_(_logits(g, R, V, F16) if i % 2 else torch.randint(0, 3, (R, V), generator=g).to(F16))
        u.copy_(torch.rand(R, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = ops.npu_sample(x, u, **kw)
        assert torch.equal(tokens, want[0]) and torch.equal(lp, want[1])


def test_no_rows(ops):
    tokens, lp = ops.npu_sample(torch.zeros((0, 100), device=DEV), torch.zeros(0, device=DEV))
    assert tokens.shape == lp.shape == (0,)
