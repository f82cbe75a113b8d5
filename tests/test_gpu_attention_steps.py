"""quant_attention and the paged cache in a server's steps: padded batches."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, HQ, HKV, D, LAYERS = 256, 8, 2, 64, 2


@pytest.fixture(scope="module")
def mods():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from op_plugin_amd import attention, kv_cache
    return attention, kv_cache


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Model:
    """The weights of one attention block, and its steps over a cache."""

    def __init__(self, mods, kind=torch.bfloat16, seed=0):
        self.att, kvc = mods
        self.g = torch.Generator().manual_seed(seed)
        self.cache = kvc.PagedKVCache(LAYERS, 40, 16, HKV, D, max_seqs=6, max_len=200, dtype=kind, device=DEV)
        int8 = lambda *shape: torch.randint(-127, 128, shape, generator=self.g, dtype=torch.int8).to(DEV)  # noqa: E731
        self.w_qkv, self.w_o = int8(H, (HQ + 2 * HKV) * D), int8(HQ * D, H)
        self.s_qkv, self.s_o = torch.full((self.w_qkv.shape[1],), 1e-3, device=DEV), torch.full((H,), 1e-3, device=DEV)
        self.gamma = torch.ones(H, dtype=torch.bfloat16, device=DEV)
        angle = torch.arange(256, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float().to(DEV)

    def input(self, tokens):
        return torch.randn((tokens, H), generator=self.g).to(torch.bfloat16).to(DEV)

    def step(self, x, seqs, cu, one_each=False, **kw):
        """x through the block in every layer, each layer's own cache; the layers' outputs."""
        slots, positions, missing = self.cache.extend(seqs, cu, x.shape[0])
        return [self.att.quant_attention(x, self.gamma, self.w_qkv, self.s_qkv, self.w_o, self.s_o, self.cache, layer, seqs,
                                         None if one_each else cu, slots, positions, self.cos_sin, HQ, **kw)
                for layer in range(LAYERS)], missing


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.int8])
def test_padded_batches(mods, kind):
    """Sequence numbers outside the table are padding: their rows are 0, and the others what they are without."""
    print(f"[case] padded batches {kind}", flush=True)
    a, b = Model(mods, kind), Model(mods, kind)
    x = a.input(37 + 5)
    plain, _ = a.step(x, _ints([0, 5]), _ints([0, 37, 42]))
    wide = torch.cat([a.input(3), x[:37], a.input(2), x[37:]])
    padded, missing = b.step(wide, _ints([-1, 0, 6, 5]), _ints([0, 3, 40, 42, 47]))
    assert int(missing) == 0
    for p, w in zip(plain, padded):
        assert torch.equal(p, torch.cat([w[3:40], w[42:]])) and (w[:3] == 0).all() and (w[40:42] == 0).all()
    x = a.input(2)
    plain, _ = a.step(x, _ints([5, 0]), _ints([0, 1, 2]), one_each=True)
    wide = torch.cat([x[:1], a.input(2), x[1:], a.input(1)])
    padded, missing = b.step(wide, _ints([5, -1, 2 ** 31 - 1, 0, 6]), _ints([0, 1, 2, 3, 4, 5]), one_each=True)
    assert int(missing) == 0
    for p, w in zip(plain, padded):
        assert torch.equal(p, w[[0, 3]]) and (w[[1, 2, 4]] == 0).all()
    assert torch.equal(a.cache.block_table, b.cache.block_table) and torch.equal(a.cache.context_lens, b.cache.context_lens)


@pytest.mark.parametrize("one_each", [False, True])
def test_rows_taken_once(mods, one_each, monkeypatch):
    """The table's rows taken once for all layers give the bits of rows taken in each layer."""
    print(f"[case] rows taken once one_each={one_each}", flush=True)
    a, b = Model(mods), Model(mods)
    seqs, cu = _ints([3, -1, 0]), _ints([0, 1, 2, 3] if one_each else [0, 20, 21, 60])
    x = a.input(3 if one_each else 60)
    want, _ = a.step(x, seqs, cu, one_each)
    slots, positions, _ = b.cache.extend(seqs, cu, x.shape[0])
    rows = b.cache.rows(seqs)
    monkeypatch.setattr(b.cache, "rows", None)  # no layer takes them again
    for layer in range(LAYERS):
        got = b.att.quant_attention(x, b.gamma, b.w_qkv, b.s_qkv, b.w_o, b.s_o, b.cache, layer, seqs, None if one_each else cu,
                                    slots, positions, b.cos_sin, HQ, rows=rows)
        assert torch.equal(got, want[layer])


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.int8])
def test_graph_of_a_step_across_compact(mods, kind):
    """A decode step captured before a compaction works on the compacted cache: the same bits as eager steps, every time."""
    print(f"[case] graph across compact {kind}", flush=True)
    a, b = Model(mods, kind), Model(mods, kind)  # a: eager; b: the captured step
    seqs, cu, x = _ints([0, 3, 5]), _ints([0, 1, 2, 3]), a.input(3)
    first = a.input(90)
    for m in (a, b):
        m.step(first, _ints([0, 1, 3, 5]), _ints([0, 20, 57, 60, 90]))
        m.step(x, seqs, cu, one_each=True)  # the libraries' and the allocator's first use, outside the capture
    held = [t.data_ptr() for t in (b.cache.block_table, b.cache.context_lens, b.cache.ref_count)]
    graph, given = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        got, missing = b.step(given, seqs, cu, one_each=True)
    torch.cuda.synchronize()

    def same(what):
        xs = a.input(3)
        given.copy_(xs)
        graph.replay()
        torch.cuda.synchronize()
        want, _ = a.step(xs, seqs, cu, one_each=True)
        assert int(missing) == 0 and all(torch.equal(w, g) for w, g in zip(want, got)), what
        for s, t in ((a.cache.block_table, b.cache.block_table), (a.cache.context_lens, b.cache.context_lens),
                     (a.cache.ref_count, b.cache.ref_count)):
            assert torch.equal(s, t), what

    same("before")
    for m in (a, b):
        m.cache.free(_ints([1]))
        assert int(m.cache.compact()) > 0
    assert held == [t.data_ptr() for t in (b.cache.block_table, b.cache.context_lens, b.cache.ref_count)]
    used = int((b.cache.ref_count > 0).sum())
    assert (b.cache.ref_count[:used] > 0).all() and int(b.cache.block_table.max()) < used
    for i in range(20):  # past the pages' ends: new ones are taken from behind those that moved
        same(f"after, step {i}")
        garbage = [torch.full_like(b.cache.block_table, 10 ** 6) for _ in range(4)]  # what an old table's memory may become
        del garbage
