"""npu_kv_accept against the walk in plain Python and the moves on a copy of the pool: whole numbers and bytes, all equal."""
import random

import pytest
import torch

import tree_ref as T

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import op_plugin_amd
    return op_plugin_amd


def _ints(v, dev=DEV):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _walk(tokens, parents, sampled):
    way, at = [], 0
    while True:
        way.append(at)
        nxt = [c for c in range(at + 1, len(tokens)) if parents[c] == at and tokens[c] >= 0 and tokens[c] == sampled[at]]
        if not nxt:
            return way, sampled[at]
        at = nxt[0]


def _tree(rng, n, right=0.8):
    """tokens, parents, sampled of a tree whose drafts are right now and then; siblings share tokens now and then."""
    parents = T.random_tree(rng, n)
    tokens = [rng.randrange(12) for _ in range(n)]
    sampled = [rng.randrange(100, 200) for _ in range(n)]
    for i in range(n):
        below = [c for c in range(n) if parents[c] == i]
        if below and rng.random() < right:
            sampled[i] = tokens[rng.choice(below)]
    return tokens, parents, sampled


def _state(g, lens, page, spare=2, max_seqs=None, width=None):
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    order = torch.randperm(P, generator=g)
    table = torch.full((max_seqs or len(lens), width or max(need + [0]) + 1), -1, dtype=torch.int32)
    count = torch.zeros(P, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k].to(torch.int32)
        count[order[at:at + k]] = 1
        at += k
    all_lens = torch.zeros(table.shape[0], dtype=torch.int32)
    all_lens[:len(lens)] = torch.tensor(lens, dtype=torch.int32)
    return table, all_lens, count, P


def _expect(caches, table, lens, count, page, seqs, cu, tokens, parents, sampled):
    """In place on CPU tensors; returns path, accepted, next."""
    path = [-1] * len(tokens)
    accepted, drawn = [], []
    for i, seq in enumerate(seqs):
        a, b = cu[i], cu[i + 1]
        n = b - a
        if not 0 <= seq < table.shape[0] or n == 0 or int(lens[seq]) < n:
            accepted.append(0)
            drawn.append(-1)
            continue
        past = int(lens[seq]) - n
        way, nxt = _walk(tokens[a:b], parents[a:b], sampled[a:b])
        for j, r in enumerate(way):
            path[a + j] = a + r
            src, dst = past + r, past + j
            p0, p1 = int(table[seq, src // page]), int(table[seq, dst // page])
            if src != dst and 0 <= p0 < count.numel() and 0 <= p1 < count.numel():
                for c in caches:
                    c[p1, dst % page] = c[p0, src % page]
        now = past + len(way)
        for j in range(-(-now // page), -(-(past + n) // page)):
            if 0 <= int(table[seq, j]) < count.numel():
                count[int(table[seq, j])] -= 1
            table[seq, j] = -1
        lens[seq] = now
        accepted.append(len(way))
        drawn.append(nxt)
    return path, accepted, drawn


def _run(ops, past, sizes, page=16, shapes=((2, 64),), dtypes=(torch.bfloat16,), layers=2, seqs=None, max_seqs=None, seed=0, right=0.8,
         make=None, extra=0):
    print(f"[case] accept past={past} sizes={sizes} page={page} shapes={shapes} layers={layers} seqs={seqs}", flush=True)
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    lens = [p + n for p, n in zip(past, sizes)]
    table, all_lens, count, P = _state(g, lens, page, max_seqs=max_seqs)
    caches = []
    for _ in range(layers):
        for shape, dtype in zip(shapes, dtypes):
            c = torch.randint(-100, 100, (P, page, *shape), generator=g).to(dtype)
            caches.append(c)
    trees = [make(rng, n) if make else _tree(rng, n, right) for n in sizes]
    tokens, parents, sampled = ([v for t in trees for v in t[i]] + [0] * extra for i in range(3))
    cu = [0]
    for n in sizes:
        cu.append(cu[-1] + n)
    seqs = list(range(len(sizes))) if seqs is None else seqs
    dev = [c.to(DEV) for c in caches]
    td, ld, cd = table.to(DEV), all_lens.to(DEV), count.to(DEV)
    want = _expect(caches, table, all_lens, count, page, seqs, cu, tokens, parents, sampled)
    path, accepted, nxt = ops.npu_kv_accept(dev, td, ld, cd, _ints(seqs), _ints(cu), _ints(tokens), _ints(parents), _ints(sampled), page)
    assert path.tolist() == want[0] and accepted.tolist() == want[1] and nxt.tolist() == want[2]
    assert torch.equal(td.cpu(), table) and torch.equal(ld.cpu(), all_lens) and torch.equal(cd.cpu(), count)
    for a, b in zip(dev, caches):
        assert torch.equal(a.cpu(), b)
    return want


@pytest.mark.parametrize("page", [1, 2, 7, 16, 48])
@pytest.mark.parametrize("past,sizes", [([0], [1]), ([5], [1]), ([0, 3], [9, 20]), ([100, 31, 0, 64], [7, 1, 40, 16]), ([1000], [64]),
                                        ([20] * 70, [5, 0, 12, 1, 3, 8, 2] * 10)])
def test_sizes(ops, past, sizes, page):
    _run(ops, past, sizes, page)


@pytest.mark.parametrize("shapes,dtypes", [(((2, 64), (2,)), (torch.int8, torch.float32)), (((1, 8),), (torch.float16,)),
                                           (((5, 80), (5,)), (torch.bfloat16, torch.float32)), (((3,),), (torch.int8,)),
                                           (((),), (torch.float32,)), (((8, 256),), (torch.bfloat16,)), (((2, 3, 4),), (torch.bfloat16,))])
def test_tensors(ops, shapes, dtypes):
    """Rows of every size: whole 16-byte pieces, single bytes, scales, wider than a workgroup."""
    _run(ops, [30, 7], [20, 33], shapes=shapes, dtypes=dtypes, layers=3)


def test_many_tensors(ops):
    _run(ops, [30, 7], [20, 33], shapes=((2, 16),), layers=150)
    _run(ops, [30, 7], [20, 33], layers=0)


def test_passed_over(ops):
    """Numbers outside the table, and lengths below the tree's."""
    _run(ops, [30, 7, 12, 40], [20, 9, 5, 6], seqs=[0, -1, 99, 3], max_seqs=6, extra=5)
    print("[case] accept: a tree larger than its sequence", flush=True)
    c = torch.arange(4 * 16, dtype=torch.float32, device=DEV).view(4, 16, 1)
    table, lens, count = _ints([[0, 1]]), _ints([5]), _ints([1, 1, 0, 0])
    before = c.clone()
    path, accepted, nxt = ops.npu_kv_accept([c], table, lens, count, _ints([0]), _ints([0, 6]), _ints([1] * 6), _ints([-1, 0, 0, 1, 1, 2]),
                                            _ints([1] * 6), 16)
    assert path.tolist() == [-1] * 6 and accepted.tolist() == [0] and nxt.tolist() == [-1]
    assert torch.equal(c, before) and lens.tolist() == [5] and count.tolist() == [1, 1, 0, 0]
    path, accepted, nxt = ops.npu_kv_accept([c], table, lens, count, _ints([]), _ints([0]), _ints([1] * 3), _ints([0] * 3), _ints([1] * 3), 16)
    assert path.tolist() == [-1] * 3 and accepted.shape == nxt.shape == (0,)


def test_long_way(ops):
    """All drafts right along one branch that skips rows: every row moves, over many pages."""
    def make(rng, n):
        parents = [-1] + [max(0, i - 2) for i in range(1, n)]
        tokens = list(range(n))
        sampled = [tokens[min(i + 2, n - 1)] for i in range(n)]
        return tokens, parents, sampled
    assert _run(ops, [50], [200], page=7, make=make)[1][0] > 90
    assert _run(ops, [50, 3], [1000, 1024], page=16, make=make, layers=1)[1][0] > 400


@pytest.mark.parametrize("n", [1024, 1025, 3000])
def test_large_trees(ops, n):
    _run(ops, [5, 40], [n, 9], page=16, right=0.97, layers=2)


def test_odd_trees(ops):
    """Parents that are none, tokens below 0, equal siblings (the lowest is taken), a row that names itself."""
    def make(rng, n):
        tokens = [rng.choice([-1, 1, 2]) for _ in range(n)]
        parents = [rng.choice([-5, i, i + 1, 99, max(0, i - 1), max(0, i - 2), max(0, i - 3), 0]) for i in range(n)]
        sampled = [rng.choice([-1, 1, 2]) for _ in range(n)]
        return tokens, parents, sampled
    for seed in range(12):
        _run(ops, [20] * 9, [1, 3, 8, 15, 30, 30, 60, 64, 65], make=make, seed=seed, layers=1)


@pytest.mark.parametrize("form", ["heads first", "keys beside values", "odd"])
def test_strided_tensors(ops, form):
    print(f"[case] accept strided {form}", flush=True)
    rng, g = random.Random(1), torch.Generator().manual_seed(1)
    page, H, D, sizes, past = 16, 3, 16, [20, 30], [40, 5]
    table, lens, count, P = _state(g, [a + b for a, b in zip(sizes, past)], page)
    if form == "heads first":
        whole = torch.randn((P, H, page, D), generator=g)
        view = lambda t: [t.permute(0, 2, 1, 3)]  # noqa: E731
    elif form == "keys beside values":
        whole = torch.randn((P, page, 2 * H, D), generator=g).to(torch.bfloat16)
        view = lambda t: [t[:, :, :H], t[:, :, H:]]  # noqa: E731
    else:
        whole = torch.randn((P + 1, page, H, D + 3), generator=g).to(torch.bfloat16)
        view = lambda t: [t[1:, :, :, 1:D + 2]]  # noqa: E731
    trees = [_tree(rng, n) for n in sizes]
    tokens, parents, sampled = ([v for t in trees for v in t[i]] for i in range(3))
    dev = whole.to(DEV)
    td, ld, cd = table.to(DEV), lens.to(DEV), count.to(DEV)
    want = _expect(view(whole), table, lens, count, page, [0, 1], [0, 20, 50], tokens, parents, sampled)
    path, accepted, nxt = ops.npu_kv_accept(view(dev), td, ld, cd, _ints([0, 1]), _ints([0, 20, 50]), _ints(tokens), _ints(parents),
                                            _ints(sampled), page)
    assert path.tolist() == want[0] and accepted.tolist() == want[1] and nxt.tolist() == want[2]
    assert torch.equal(dev.cpu(), whole) and torch.equal(td.cpu(), table) and torch.equal(ld.cpu(), lens)


@pytest.mark.parametrize("layers", [3, 70])
def test_tensors_that_are_there_twice(ops, layers):
    """Layers that share a cache: a row moves once."""
    print(f"[case] accept twice {layers}", flush=True)
    rng, g = random.Random(2), torch.Generator().manual_seed(2)
    page, sizes, past = 16, [40, 30], [9, 40]
    table, lens, count, P = _state(g, [a + b for a, b in zip(sizes, past)], page)
    caches = [torch.randn((P, page, 2, 64), generator=g) for _ in range(2)]
    trees = [_tree(rng, n, right=1.0) for n in sizes]
    tokens, parents, sampled = ([v for t in trees for v in t[i]] for i in range(3))
    dev = [c.to(DEV) for c in caches]
    td, ld, cd = table.to(DEV), lens.to(DEV), count.to(DEV)
    want = _expect(caches, table, lens, count, page, [0, 1], [0, 40, 70], tokens, parents, sampled)
    path, accepted, nxt = ops.npu_kv_accept(dev * layers, td, ld, cd, _ints([0, 1]), _ints([0, 40, 70]), _ints(tokens), _ints(parents),
                                            _ints(sampled), page)
    assert path.tolist() == want[0] and accepted.tolist() == want[1] and nxt.tolist() == want[2] and min(want[1]) >= 3
    for a, b in zip(dev, caches):
        assert torch.equal(a.cpu(), b)
    with pytest.raises(RuntimeError, match="begin at one place"):
        ops.npu_kv_accept([dev[0], dev[0][:, :, :1]], td, ld, cd, _ints([0, 1]), _ints([0, 40, 70]), _ints(tokens), _ints(parents),
                          _ints(sampled), page)


def test_bad_pages(ops):
    """A page id outside the pool is not followed: its rows stay, the others move, and it is not counted."""
    print("[case] accept bad pages", flush=True)
    g = torch.Generator().manual_seed(2)
    page = 4
    table, lens, count, P = _state(g, [40], page)
    table[0, 5], table[0, 7] = 10 ** 6, -3
    c = torch.randn((P, page, 2), generator=g)
    tokens, parents = list(range(24)), [-1] + [max(0, i - 2) for i in range(1, 24)]
    sampled = [min(i + 2, 23) for i in range(24)]
    args = [t.clone() for t in (c, table, lens, count)]
    td, ld, cd, dev = table.to(DEV), lens.to(DEV), count.to(DEV), c.to(DEV)
    want = _expect([args[0]], args[1], args[2], args[3], page, [0], [0, 24], tokens, parents, sampled)
    got = ops.npu_kv_accept([dev], td, ld, cd, _ints([0]), _ints([0, 24]), _ints(tokens), _ints(parents), _ints(sampled), page)
    assert [t.tolist() for t in got] == list(want)
    assert torch.equal(dev.cpu(), args[0]) and torch.equal(td.cpu(), args[1]) and torch.equal(cd.cpu(), args[3])


def test_graph_replays(ops):
    print("[case] accept graph", flush=True)
    rng, g = random.Random(3), torch.Generator().manual_seed(3)
    page, sizes, past = 16, [20, 30, 8], [40, 5, 100]
    table, lens, count, P = _state(g, [a + b for a, b in zip(sizes, past)], page)
    c = torch.randn((P, page, 2, 16), generator=g)
    start = [t.to(DEV) for t in (c, table, lens, count)]
    now = [t.clone() for t in start]
    cu, seqs = _ints([0, 20, 50, 58]), _ints([0, 1, 2])
    tokens, parents, sampled = (torch.zeros(58, dtype=torch.int32, device=DEV) for _ in range(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.npu_kv_accept([now[0]], *now[1:], seqs, cu, tokens, parents, sampled, page)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        path, accepted, nxt = ops.npu_kv_accept([now[0]], *now[1:], seqs, cu, tokens, parents, sampled, page)
    for _ in range(4):
        trees = [_tree(rng, n) for n in sizes]
        flat = [[v for t in trees for v in t[i]] for i in range(3)]
        for to, new in zip((tokens, parents, sampled), flat):
            to.copy_(_ints(new))
        for to, new in zip(now, start):
            to.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        host = [t.cpu().clone() for t in start]
        want = _expect([host[0]], *host[1:], page, [0, 1, 2], [0, 20, 50, 58], *flat)
        assert [t.tolist() for t in (path, accepted, nxt)] == list(want)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(now, host))
