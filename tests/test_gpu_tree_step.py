"""Decoding with drafts as a server runs it: prompts, then steps of trees through every layer, drawn tokens, accepted ways, a fork
between them, eagerly and as one replayed graph."""
import math
import random

import pytest
import torch

import attention_ref as R
import tree_ref as T
from test_gpu_kv_accept import _walk
from test_gpu_sample import _row

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
H, HQ, HKV, D, PAGE, V, LAYERS = 256, 8, 2, 64, 16, 16, 2


@pytest.fixture(scope="module")
def q():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import op_plugin_amd
    return op_plugin_amd


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Decoder:
    """Two attention blocks between an embedding of 16 tokens and their logits."""

    def __init__(self, q, kind, window=0, sinks=0):
        from op_plugin_amd import attention, kv_cache
        g = torch.Generator().manual_seed(5)
        self.q, self.att, self.window, self.sinks = q, attention, window, sinks
        self.cache = kv_cache.PagedKVCache(LAYERS, 60, PAGE, HKV, D, max_seqs=6, max_len=300, dtype=kind, device=DEV)
        ints = lambda *shape: torch.randint(-127, 128, shape, generator=g, dtype=torch.int8).to(DEV)  # noqa: E731
        self.embedding = torch.randn((V, H), generator=g).to(BF16).to(DEV)
        self.w_qkv = [ints(H, (HQ + 2 * HKV) * D) for _ in range(LAYERS)]
        self.w_o = [ints(HQ * D, H) for _ in range(LAYERS)]
        self.w_out = ints(H, V)
        self.s_qkv = torch.full(((HQ + 2 * HKV) * D,), 1e-3, device=DEV)
        self.s_o = torch.full((H,), 1e-3, device=DEV)
        self.s_out = torch.full((V,), 2e-3, device=DEV)
        self.gamma = torch.ones(H, dtype=BF16, device=DEV)
        angle = torch.arange(512, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float().to(DEV)

    def block(self, x, layer, seqs, cu, slots, positions, rows, mask=None):
        return self.att.quant_attention(x, self.gamma, self.w_qkv[layer], self.s_qkv, self.w_o[layer], self.s_o, self.cache, layer, seqs,
                                        cu, slots, positions, self.cos_sin, HQ, rows=rows, window=self.window, sinks=self.sinks,
                                        tree_mask=mask)

    def logits(self, x):
        y, s = self.q.npu_dynamic_quant(x)
        return self.q.npu_quant_matmul(y, self.w_out, self.s_out, pertoken_scale=s, output_dtype=BF16)

    def turned(self, x, layer, positions):
        y, s, _ = self.q.npu_rms_norm_dynamic_quant(x, self.gamma, 1e-6)
        qkv = self.q.npu_quant_matmul(y, self.w_qkv[layer], self.s_qkv, pertoken_scale=s, output_dtype=BF16)
        qq, kk, vv = qkv.view(-1, HQ + 2 * HKV, D).split([HQ, HKV, HKV], dim=1)
        return *self.q.npu_mrope(positions, qq, kk, self.cos_sin), vv

    def prompt(self, seqs, texts):
        cu = [0]
        for t in texts:
            cu.append(cu[-1] + len(t))
        slots, positions, missing = self.cache.extend(_ints(seqs), _ints(cu), cu[-1])
        assert int(missing) == 0
        x = self.embedding[_ints([t for text in texts for t in text]).long()]
        for layer in range(LAYERS):
            x = x + self.block(x, layer, _ints(seqs), _ints(cu), slots, positions, None)

    def step(self, seqs, cu, tokens, parents, uniform, settings, words, see=None):
        """One step on the device; see(layer, x, out, positions): after each layer's block."""
        from op_plugin_amd.tree import tree_mask, tree_positions
        slots, positions, missing = self.cache.extend(seqs, cu, tokens.numel())
        mask, depth = tree_mask(parents, cu, words)
        positions = tree_positions(positions, cu, depth)
        rows = self.cache.rows(seqs)
        x = self.embedding[tokens.long()]
        for layer in range(LAYERS):
            out = self.block(x, layer, seqs, cu, slots, positions, rows, mask)
            if see:
                see(layer, x, out, positions)
            x = x + out
        logits = self.logits(x)
        sampled, logprobs = self.q.npu_sample(logits, uniform, **settings)
        return logits, sampled, logprobs, missing, *self.cache.accept(seqs, cu, tokens, parents, sampled)

    def rows(self, pool, scales, seq, n, layer):
        table = self.cache.block_table[seq].cpu()
        j = torch.arange(n)
        out = pool[layer].cpu()[table[j // PAGE].long(), j % PAGE].double()
        return out if scales[layer] is None else out * scales[layer].cpu()[table[j // PAGE].long(), j % PAGE].double()[..., None]

    def held(self, seq, n):
        """Everything that the cache holds of a sequence, as it lies there."""
        c, j = self.cache, torch.arange(n, device=DEV)
        page = c.block_table[seq][j // PAGE].long()
        return [pool[page, j % PAGE] for pool in c._pools()]


def _tree(rng, n):
    """Every token below the root (one of them is drawn), then drafts at random."""
    parents = ([-1] + [0] * V + [rng.randrange(1, i) for i in range(V + 1, n)])[:n]
    tokens = ([0] + rng.sample(range(V), V) + [rng.randrange(V) for _ in range(V + 1, n)])[:n]
    return parents, tokens


@pytest.mark.parametrize("kind,window,sinks", [(BF16, 0, 0), (torch.int8, 0, 0), (BF16, 20, 3)])
def test_steps(q, kind, window, sinks):
    """Each block's output against attention in 64 bits over the rows of the cache that the row's ancestors and their context are,
    with the block test's bounds; each drawn token against its row's logits; each accepted way against a walk along the drawn
    tokens.  What the cache holds behind a step is what it held at the way's rows, and its first layer (which hangs on tokens
    and positions alone) is, bit for bit, what the accepted text gives at positions one after another."""
    print(f"[case] steps {kind} window={window} sinks={sinks}", flush=True)
    m = Decoder(q, kind, window, sinks)
    rng, g = random.Random(1), torch.Generator().manual_seed(2)
    text = {0: [rng.randrange(V) for _ in range(37)], 3: [rng.randrange(V) for _ in range(5)]}
    m.prompt([0, 3], [text[0], text[3]])
    root = {0: 7, 3: 2}
    for turn, sizes in enumerate([{0: 60, 3: 17, -1: 5}, {3: 1, 0: 33}, {0: 100, 4: 20, 9: 3, 3: 64}, {4: 17, 0: 1, 3: 40}]):
        if turn == 2:
            assert int(m.cache.fork(_ints([0]), _ints([4]))) == 0
            text[4], root[4] = list(text[0]), root[0]
        seqs, live = list(sizes), [s for s in sizes if s in root]
        trees = [_tree(rng, n) for n in sizes.values()]
        for s, (_, tokens) in zip(seqs, trees):
            tokens[0] = root.get(s, 0)
        cu = [0]
        for n in sizes.values():
            cu.append(cu[-1] + n)
        words = max(1, -(-max(sizes.values()) // 64))
        parents, tokens = ([v for t in trees for v in t[i]] for i in range(2))
        T_all = cu[-1]
        settings = dict(temperature=torch.tensor([0.0, 0.7, 1.3])[torch.randint(0, 3, (T_all,), generator=g)].to(DEV),
                        top_k=_ints([rng.choice([0, 3]) for _ in range(T_all)]),
                        top_p=torch.tensor([1.0, 0.9])[torch.randint(0, 2, (T_all,), generator=g)].to(DEV))
        uniform = torch.rand(T_all, generator=g).to(DEV)
        before = {}

        def see(layer, x, out, positions):
            turned, _, _ = m.turned(x, layer, positions)
            if layer == LAYERS - 1:
                before.update({s: m.held(s, len(text[s]) + sizes[s]) for s in live})
            for i, s in enumerate(seqs):
                a, b = cu[i], cu[i + 1]
                if s not in live:
                    assert (out[a:b] == 0).all()
                    continue
                n = len(text[s]) + sizes[s]
                ok = T.visible(T.ancestors(trees[i][0]), n, window, sinks)
                k, v = (m.rows(p, sc, s, n, layer) for p, sc in ((m.cache.keys, m.cache.key_scales),
                                                                 (m.cache.values, m.cache.value_scales)))
                o, _, away, size, _ = R.attend(turned[a:b].double().cpu(), k, v, ok, 1 / math.sqrt(D))
                o, away = o.flatten(1), away.flatten(1)
                u = 2.0 ** -8
                delta = (size.amax() * (D + 8) + n + 64) * 2.0 ** -24
                slack = away * (u + 2 * delta) + o.abs() * u + o.abs().amax(1, keepdim=True) * (0.5 + 2 * u) / 127
                w = m.w_o[layer].double().cpu()
                want = (o @ w) * 1e-3
                tol = (slack @ w.abs()) * 1e-3 + want.abs() * u
                got = out[a:b].double().cpu()
                assert ((got - want).abs() <= tol).all(), (s, layer, float(((got - want).abs() / tol).max()))

        logits, sampled, logprobs, missing, path, accepted, nxt = m.step(_ints(seqs), _ints(cu), _ints(tokens), _ints(parents), uniform,
                                                                         settings, words, see)
        assert int(missing) == 0
        drawn, x = sampled.tolist(), logits.double().cpu().numpy()
        for r in range(T_all):
            found = _row(x[r], float(uniform[r]), float(settings["temperature"][r]), int(settings["top_k"][r]),
                         float(settings["top_p"][r]), 0.0)
            assert drawn[r] in found, r
            assert abs(float(logprobs[r]) - found[drawn[r]]) <= abs(found[drawn[r]]) * 2.0 ** -24 + V * 2.0 ** -40
        for i, s in enumerate(seqs):
            a, b = cu[i], cu[i + 1]
            if s not in live:
                assert int(accepted[i]) == 0 and int(nxt[i]) == -1 and (path[a:b] == -1).all()
                continue
            way, then = _walk(tokens[a:b], parents[a:b], drawn[a:b])
            assert path[a:b].tolist() == [a + r for r in way] + [-1] * (b - a - len(way))
            assert int(accepted[i]) == len(way) and int(nxt[i]) == then and (len(way) > 1 or b - a <= V)
            past = len(text[s])
            keep = torch.tensor(list(range(past)) + [past + r for r in way], device=DEV)
            text[s] += [tokens[a + r] for r in way]
            root[s] = then
            assert int(m.cache.context_lens[s]) == len(text[s])
            now = m.held(s, len(text[s]))
            for old, new in zip(before[s], now):
                assert torch.equal(old[keep], new)
            _, k, v = m.turned(m.embedding[_ints(text[s]).long()], 0, torch.arange(len(text[s]), device=DEV, dtype=torch.int32))
            if kind == BF16:
                assert torch.equal(now[0], k) and torch.equal(now[LAYERS], v)
            else:
                for at, rows in ((0, k), (LAYERS, v)):
                    y, sc = q.npu_dynamic_quant(rows.reshape(-1, D))
                    assert torch.equal(now[at].reshape(-1, D), y) and torch.equal(now[at + 2 * LAYERS].reshape(-1), sc)
    used = sum(-(-len(t) // PAGE) for t in text.values())
    assert int(m.cache.ref_count.sum()) == used


@pytest.mark.parametrize("kind", [BF16, torch.int8])
def test_step_as_a_graph(q, kind):
    """A whole step, from extend to accept, in one graph: replays, with eager steps between them, give what the eager step gives and
    leave the cache as it does."""
    print(f"[case] step as a graph {kind}", flush=True)
    m = Decoder(q, kind)
    rng, g = random.Random(4), torch.Generator().manual_seed(6)
    m.prompt([1, 2], [[rng.randrange(V) for _ in range(45)], [rng.randrange(V) for _ in range(16)]])
    sizes = [40, 20]
    seqs, cu = _ints([1, 2]), _ints([0, 40, 60])
    tokens, parents, uniform = _ints([0] * 60), _ints([-1] * 60), torch.zeros(60, device=DEV)
    settings = dict(temperature=torch.full((60,), 0.8, device=DEV), top_p=torch.full((60,), 0.95, device=DEV))
    state = [m.cache.block_table, m.cache.context_lens, m.cache.ref_count, *m.cache._pools()]

    def draft(roots):
        trees = [_tree(rng, n) for n in sizes]
        for t, r in zip(trees, roots):
            t[1][0] = r
        parents.copy_(_ints([v for t in trees for v in t[0]]))
        tokens.copy_(_ints([v for t in trees for v in t[1]]))
        uniform.copy_(torch.rand(60, generator=g))

    step = lambda: m.step(seqs, cu, tokens, parents, uniform, settings, 1)  # noqa: E731
    draft([3, 4])
    start = [t.clone() for t in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for a, b in zip(state, start):
        a.copy_(b)
    roots = [3, 4]
    for turn in range(4):
        draft(roots)
        start = [t.clone() for t in state]
        want = [t.clone() for t in step()]
        after = [t.clone() for t in state]
        assert int(want[3]) == 0 and (want[5] > 1).all()
        for a, b in zip(state, start):
            a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), turn
        for a, b in zip(state[:3], after[:3]):
            assert torch.equal(a, b), turn
        held = m.cache.ref_count > 0
        for a, b in zip(state[3:], after[3:]):
            assert torch.equal(a[held].view(torch.uint8), b[held].view(torch.uint8)), turn
        roots = want[6].tolist()


def test_step_without_room(q):
    """A step that finds no pages leaves everything as it was where its sequences are passed over for it."""
    print("[case] step without room", flush=True)
    from op_plugin_amd.tree import tree_mask, tree_positions
    m = Decoder(q, BF16)
    m.prompt([0], [[1] * 50])
    c = m.cache
    c.ref_count[c.ref_count == 0] = 1  # every other page is somebody's
    start = [t.clone() for t in (c.block_table, c.context_lens, c.ref_count)]
    held = m.held(0, 50)
    parents, tokens = (_ints(v) for v in _tree(random.Random(3), 30))
    seqs, cu = _ints([0]), _ints([0, 30])
    slots, positions, missing = c.extend(seqs, cu, 30)
    assert int(missing) > 0 and (slots == -1).all()
    seqs = torch.where(missing == 0, seqs, -1)
    mask, depth = tree_mask(parents, cu)
    out = m.block(m.embedding[tokens.long()], 0, seqs, cu, slots, tree_positions(positions, cu, depth), c.rows(seqs), mask)
    assert (out == 0).all()
    path, accepted, nxt = c.accept(seqs, cu, tokens, parents, tokens)
    assert (path == -1).all() and accepted.tolist() == [0] and nxt.tolist() == [-1]
    for a, b in zip((c.block_table, c.context_lens, c.ref_count), start):
        assert torch.equal(a, b)
    for a, b in zip(m.held(0, 50), held):
        assert torch.equal(a, b)
