"""The pages' ops against bookkeeping in plain Python, bit for bit, with the pool's contents."""
import random

import pytest
import torch

import attention_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import op_plugin_amd
    return op_plugin_amd


def _state(rng, P, S, W, page, fill=0.6):
    """A pool whose sequences hold random pages; some slots are empty."""
    order = list(range(P))
    rng.shuffle(order)
    table = torch.full((S, W), -1, dtype=torch.int32)
    lens = torch.zeros(S, dtype=torch.int32)
    count = torch.zeros(P, dtype=torch.int32)
    used = 0
    for s in range(S):
        n = rng.randrange(0, W * page // 2 + 1) if rng.random() < 0.7 else 0
        pages = -(-n // page)
        if used + pages > fill * P:
            continue
        for j in range(pages):
            table[s, j] = order[used]
            count[order[used]] = 1
            used += 1
        lens[s] = n
    return table, lens, count


def _same(dev, pool):
    table, lens, count = dev
    assert table.cpu().tolist() == pool.table
    assert lens.cpu().tolist() == pool.lens
    assert count.cpu().tolist() == pool.count


@pytest.mark.parametrize("P,S,W,page,seed", [(8, 3, 4, 4, 0), (50, 9, 10, 16, 1), (5000, 200, 30, 16, 2), (777, 40, 25, 3, 3),
                                             (9000, 1100, 12, 1, 4)])
def test_life_of_a_pool(ops, P, S, W, page, seed):
    """Random forks, growth, releases and compactions, the state and every page's contents checked after each."""
    print(f"[case] pool P={P} S={S} W={W} page={page}", flush=True)
    rng = random.Random(seed)
    table, lens, count = _state(rng, P, S, W, page)
    pool = R.Pool(table, lens, count, page)
    dev = [t.to(DEV) for t in (table, lens, count)]
    caches = [torch.randint(-128, 128, (P, page, 2, 24), dtype=torch.int8), torch.randn((P, page, 3)),
              torch.randn((P, 5)).to(torch.bfloat16)]
    cd = [c.to(DEV) for c in caches]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    for step in range(12):
        kind = ["extend", "fork", "free", "compact", "extend"][step % 5]
        held = [s for s in range(S) if pool.lens[s] > 0]
        empty = [s for s in range(S) if pool.lens[s] == 0]
        if kind == "free":
            seqs = rng.sample(range(S), max(1, S // 3)) + [-1, S]
            ops.npu_kv_free(*dev, ints(seqs), page)
            pool.free(seqs)
        elif kind == "extend":
            seqs = rng.sample(range(S), max(1, S // 2)) + [S + 3]
            tokens = [rng.randrange(0, 2 * page + 2) for _ in seqs]
            cu = [0]
            for t in tokens:
                cu.append(cu[-1] + t)
            slots, positions, missing = ops.npu_kv_extend(*dev, ints(seqs), ints(cu), cu[-1], page)
            want = pool.extend(seqs, tokens)
            assert (slots.cpu().tolist(), positions.cpu().tolist(), int(missing)) == want
        elif kind == "fork":
            n = min(len(held), len(empty))
            parents = [rng.choice(held) for _ in range(n)] + [-2, 0]
            children = rng.sample(empty, n) + [0, S]
            missing = ops.npu_kv_fork(cd, *dev, ints(parents), ints(children), page)
            pairs, lack = pool.fork(parents, children)
            assert int(missing) == lack
            for a, b in pairs or []:
                for c in caches:
                    c[b] = c[a]
        else:
            new_table, new_count, moved = ops.npu_kv_compact(cd, dev[0], dev[2])
            want_table, want_count, pairs = pool.compact()
            assert int(moved) == len(pairs)
            assert new_table.cpu().tolist() == want_table and new_count.cpu().tolist() == want_count
            _same(dev, pool)  # the old state stands
            for a, b in pairs:
                for c in caches:
                    c[b] = c[a]
            dev[0], dev[2] = new_table, new_count
            pool.table, pool.count = want_table, want_count
        _same(dev, pool)
        for c, d in zip(caches, cd):
            assert torch.equal(c.view(torch.uint8) if c.dtype != torch.int8 else c, d.cpu().view(torch.uint8) if c.dtype != torch.int8 else d.cpu()), (step, kind)


def test_missing_pages(ops):
    """Too few pages or columns: the number that is missing, and nothing else written."""
    print("[case] missing pages", flush=True)
    table = torch.full((4, 3), -1, dtype=torch.int32, device=DEV)
    lens = torch.zeros(4, dtype=torch.int32, device=DEV)
    count = torch.tensor([1, 0, 2, 0, 1, 1], dtype=torch.int32, device=DEV)
    state = [t.clone() for t in (table, lens, count)]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    slots, positions, missing = ops.npu_kv_extend(table, lens, count, ints([0, 1]), ints([0, 8, 13]), 13, 4)
    assert int(missing) == 2 and (slots == -1).all() and (positions == -1).all()
    assert all(torch.equal(a, b) for a, b in zip(state, (table, lens, count)))
    _, _, missing = ops.npu_kv_extend(table, lens, count, ints([2]), ints([0, 17]), 17, 4)  # 5 pages of 3 columns
    assert int(missing) == 2 and all(torch.equal(a, b) for a, b in zip(state, (table, lens, count)))
    slots, positions, missing = ops.npu_kv_extend(table, lens, count, ints([3, 1]), ints([0, 2, 5]), 5, 4)
    assert int(missing) == 0 and slots.tolist() == [4, 5, 12, 13, 14] and positions.tolist() == [0, 1, 0, 1, 2]
    cache = torch.zeros((6, 4), device=DEV)
    state = [t.clone() for t in (table, lens, count)]
    missing = ops.npu_kv_fork([cache], table, lens, count, ints([3, 1]), ints([0, 2]), 4)
    assert int(missing) == 2 and all(torch.equal(a, b) for a, b in zip(state, (table, lens, count)))


def test_free_twice(ops):
    """A sequence named twice is freed once; a page shared by two sequences stays with the other."""
    print("[case] free twice", flush=True)
    table = torch.tensor([[0, 2, -1], [0, 1, -1]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([7, 8], dtype=torch.int32, device=DEV)
    count = torch.tensor([2, 1, 1], dtype=torch.int32, device=DEV)
    ops.npu_kv_free(table, lens, count, torch.tensor([0] * 50, dtype=torch.int32, device=DEV), 4)
    assert count.tolist() == [1, 1, 0] and lens.tolist() == [0, 8] and table.tolist() == [[-1] * 3, [0, 1, -1]]


@pytest.mark.parametrize("shape,dtype", [((9, 16, 8, 128), torch.bfloat16), ((9, 3, 1, 5), torch.int8), ((9, 1, 3), torch.float32),
                                         ((9, 40000), torch.float16)])
def test_copy_pages(ops, shape, dtype):
    print(f"[case] copy {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(0)
    caches = [torch.randint(-100, 100, shape, generator=g).to(dtype) for _ in range(130)]  # past one launch's list
    cd = [c.to(DEV) for c in caches]
    src, dst = [1, -1, 8, 3, 2, 9], [0, 5, 7, -4, 6, 4]
    ops.npu_kv_copy_pages(cd, torch.tensor(src, dtype=torch.int32, device=DEV), torch.tensor(dst, dtype=torch.int32, device=DEV))
    for c, d in zip(caches, cd):
        for a, b in zip(src, dst):
            if 0 <= a < 9 and 0 <= b < 9:
                c[b] = c[a]
        assert torch.equal(c, d.cpu())
    pool = torch.randn((2, 9, 4, 6), generator=g)  # pages apart from each other: a slice, and heads before tokens
    pd = pool.to(DEV)
    ops.npu_kv_copy_pages([pd[0, :, :3], pd[1].transpose(1, 2)], torch.tensor([4], dtype=torch.int32, device=DEV),
                          torch.tensor([1], dtype=torch.int32, device=DEV))
    pool[0, 1, :3], pool[1, 1] = pool[0, 4, :3], pool[1, 4]
    assert torch.equal(pool, pd.cpu())


def test_empty_calls(ops):
    print("[case] empty", flush=True)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    table = torch.full((2, 2), -1, dtype=torch.int32, device=DEV)
    lens, count = torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(5, dtype=torch.int32, device=DEV)
    ops.npu_kv_free(table, lens, count, none, 4)
    assert int(ops.npu_kv_fork([], table, lens, count, none, none, 4)) == 0
    slots, _, missing = ops.npu_kv_extend(table, lens, count, none, torch.zeros(1, dtype=torch.int32, device=DEV), 0, 4)
    assert slots.numel() == 0 and int(missing) == 0
    ops.npu_kv_copy_pages([], none, none)
    new_table, new_count, moved = ops.npu_kv_compact([], table, count)
    assert torch.equal(new_table, table) and torch.equal(new_count, count) and int(moved) == 0
