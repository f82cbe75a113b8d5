"""npu_sample where rows leave the usual paths: borders among thousands of near tokens, vocabularies past what a split row holds, as
many rows as a launch takes."""
import pytest
import torch

from test_gpu_sample import BF16, DEV, F16, F32, _check, _logits, _settings, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R", [6, 200])
@pytest.mark.parametrize("scale", [0.03, 0.1, 0.2, 0.4])
def test_borders_among_near_tokens(ops, scale, R):  # noqa: F811
    """From some hundreds to more tokens in the border's bins than are listed."""
    g = torch.Generator().manual_seed(int(100 * scale) + R)
    V = 40000
    for dtype in (F32, F16):
        x = _logits(g, R, V, dtype, scale=scale, peaks=0)
        u = torch.rand(R, generator=g)
        _check(ops, x, u, k=torch.randint(1, V, (R,), generator=g))
        _check(ops, x, u, p=0.05 + 0.9 * torch.rand(R, generator=g))
        _check(ops, x, u, k=torch.randint(V // 4, V, (R,), generator=g), p=0.3 + 0.7 * torch.rand(R, generator=g))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [(1 << 20) - 8, (1 << 20) - 7, (1 << 20) + 5, 1300001])
def test_large_vocabularies(ops, V, dtype):  # noqa: F811
    g = torch.Generator().manual_seed(V)
    x, u = _logits(g, 4, V, dtype), torch.rand(4, generator=g)
    _check(ops, x, u)
    _check(ops, x, u, t=torch.tensor([0.0, 0.5, 1.0, 2.0]), k=torch.tensor([0, 5, 700, 0]), p=torch.tensor([1.0, 0.9, 0.999, 0.95]),
           m=torch.tensor([0.0, 0.0, 0.01, 0.1]))


def test_as_many_rows_as_a_launch_takes(ops):  # noqa: F811
    """Two equal logits: the second from a half on."""
    R = (1 << 22) - 1
    print(f"[case] sample {R} x 2", flush=True)
    u = torch.rand(R, generator=torch.Generator().manual_seed(1)).to(DEV)
    tokens, _ = ops.npu_sample(torch.zeros((R, 2), dtype=BF16, device=DEV), u)
    assert torch.equal(tokens, (u >= 0.5).to(torch.int32))


@pytest.mark.parametrize("filters", ["", "t", "tm", "kp", "tkpm"])
@pytest.mark.parametrize("R,V,dtype", [(1, 20000, BF16), (2, 16384, F32), (40, 30001, F16), (9, 49152, F32), (90, 40000, BF16), (100, 100001, F16),
                                       (3, 131072, BF16), (128, 20001, F32), (5, 300007, F16)])
def test_rows_in_parts(ops, R, V, dtype, filters):  # noqa: F811
    """Sizes around those at which rows are split in the one way or the other, rows of every kind among them: an infinite logit,
    nothing to draw, NaN and -inf at the ends, runs of equal logits, one logit above all others."""
    g = torch.Generator().manual_seed(R + V)
    x, s = _logits(g, R, V, dtype), _settings(g, R, V)
    for r in range(0, R, 7):
        kind = r // 7 % 6
        if kind == 0:
            x[r, :V // 3], x[r, V - 5:] = float("nan"), float("-inf")
        elif kind == 1:
            x[r, [V // 2, V - 1]] = float("inf")
        elif kind == 2:
            x[r] = float("-inf")
        elif kind == 3:
            x[r] = 0.5
        elif kind == 4:
            x[r, V - 1] = 60.0
        else:
            s["t"][r] = 0.0
    _check(ops, x, torch.rand(R, generator=g), **{f: s[f] for f in filters})


@pytest.mark.parametrize("R,V", [(2, 30000), (100, 17000), (100, 100001)])
@pytest.mark.parametrize("filtered", [False, True])
def test_graph_replays_of_rows_in_parts(ops, R, V, filtered):  # noqa: F811
    print(f"[case] sample graph {R} x {V} {filtered}", flush=True)
    g = torch.Generator().manual_seed(V)
    x, u = torch.empty((R, V), dtype=BF16, device=DEV), torch.empty(R, device=DEV)
    s = dict(temperature=torch.full((R,), 0.9, device=DEV))
    if filtered:
        s.update(top_p=torch.full((R,), 0.9, device=DEV), top_k=torch.full((R,), 600, dtype=torch.int32, device=DEV))

    def fill():
        x.copy_(_logits(g, R, V, BF16))
        u.copy_(torch.rand(R, generator=g))

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.npu_sample(x, u, **s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, logprobs = ops.npu_sample(x, u, **s)
    for _ in range(4):
        fill()
        want = ops.npu_sample(x, u, **s)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens, want[0]) and torch.equal(logprobs, want[1])
