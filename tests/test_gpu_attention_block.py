"""The attention block over a paged cache as a server runs it: prompts in chunks, tokens one by one, forks, releases and a
compaction between them, against the same block over each sequence's whole text."""
import math

import pytest
import torch

import attention_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def mods():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import op_plugin_amd
    from op_plugin_amd import attention, kv_cache
    return op_plugin_amd, attention, kv_cache


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("kind,window,sinks", [(torch.bfloat16, 0, 0), (torch.int8, 0, 0), (torch.bfloat16, 20, 3)])
def test_serving_steps(mods, kind, window, sinks):
    """Each step's block output is W_o of attention over the sequence's keys and values so far: the rows in the cache are read
    back, attention is done on them in 64 bits, and the block's own steps before and after it (whose bits other tests pin) are
    the ops themselves.  Between the two lie the rounding of the attention's output to 16 bits, its weights' (one half step
    each, as in the attention tests) and so at most one step of the int8 rows that W_o reads."""
    q, att, kvc = mods
    print(f"[case] block {kind} window={window} sinks={sinks}", flush=True)
    g = torch.Generator().manual_seed(3)
    H, Hq, Hkv, D, page, dt = 256, 8, 2, 64, 16, torch.bfloat16
    cache = kvc.PagedKVCache(2, 40, page, Hkv, D, max_seqs=6, max_len=200, dtype=kind, device=DEV)
    w_qkv = torch.randint(-127, 128, (H, (Hq + 2 * Hkv) * D), generator=g, dtype=torch.int8).to(DEV)
    w_o = torch.randint(-127, 128, (Hq * D, H), generator=g, dtype=torch.int8).to(DEV)
    s_qkv = torch.full((w_qkv.shape[1],), 1e-3, device=DEV)
    s_o = torch.full((H,), 1e-3, device=DEV)
    gamma = torch.ones(H, dtype=dt, device=DEV)
    angle = torch.arange(256, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float().to(DEV)

    def rows(which, scales, seq, n, layer):
        table = cache.block_table[seq].cpu()
        pool, sc = which[layer].cpu(), scales[layer]
        j = torch.arange(n)
        out = pool[table[j // page].long(), j % page].double()
        return out if sc is None else out * sc.cpu()[table[j // page].long(), j % page].double()[..., None]

    def step(seqs, tokens, one_each):
        cu = [0]
        for n in tokens:
            cu.append(cu[-1] + n)
        slots, positions, missing = cache.extend(_ints(seqs), _ints(cu), cu[-1])
        assert int(missing) == 0
        for layer in range(2):
            x = torch.randn((cu[-1], H), generator=g).to(dt).to(DEV)
            out = att.quant_attention(x, gamma, w_qkv, s_qkv, w_o, s_o, cache, layer, _ints(seqs), None if one_each else _ints(cu),
                                      slots, positions, cos_sin, Hq, window=window, sinks=sinks)
            y, s, _ = q.npu_rms_norm_dynamic_quant(x, gamma, 1e-6)
            qkv = q.npu_quant_matmul(y, w_qkv, s_qkv, pertoken_scale=s, output_dtype=dt)
            qq, kk, _ = qkv.view(-1, Hq + 2 * Hkv, D).split([Hq, Hkv, Hkv], dim=1)
            turned, _ = q.npu_mrope(positions, qq, kk, cos_sin)
            for i, seq in enumerate(seqs):
                n = int(cache.context_lens[seq])
                k, v = rows(cache.keys, cache.key_scales, seq, n, layer), rows(cache.values, cache.value_scales, seq, n, layer)
                ok = R.visible(tokens[i], n, window, sinks)
                o, _, away, size, _ = R.attend(turned[cu[i]:cu[i + 1]].double().cpu(), k, v, ok, 1 / math.sqrt(D))
                o, away = o.flatten(1), away.flatten(1)
                # int8 rows: scale absmax / 127, a step of them where 16-bit roundings differ; W_o sums Hq * D products
                u = 2.0 ** -8
                delta = (size.amax() * (D + 8) + n + 64) * 2.0 ** -24
                slack = away * (u + 2 * delta) + o.abs() * u + o.abs().amax(1, keepdim=True) * (0.5 + 2 * u) / 127
                want = (o @ w_o.double().cpu()) * 1e-3
                tol = (slack @ w_o.double().cpu().abs()) * 1e-3 + want.abs() * u
                got = out[cu[i]:cu[i + 1]].double().cpu()
                assert ((got - want).abs() <= tol).all(), (seq, layer, float(((got - want).abs() / tol).max()))

    step([0, 3], [37, 5], False)      # two prompts
    step([0, 3], [1, 1], True)        # a token each
    step([0, 1], [20, 33], False)     # a chunk of the first, a new sequence
    assert int(cache.fork(_ints([0, 0]), _ints([2, 4]))) == 0
    step([2, 0, 4, 3], [1, 1, 1, 1], True)
    cache.free(_ints([0, 1]))
    moved = int(cache.compact())
    used = int((cache.ref_count > 0).sum())
    assert moved > 0 and (cache.ref_count[:used] > 0).all() and int(cache.block_table.max()) < used
    step([4, 2, 3], [1, 1, 1], True)
    step([0, 5], [18, 1], False)


def test_refusals(mods):
    _, _, kvc = mods
    with pytest.raises(ValueError, match="dtype"):
        kvc.PagedKVCache(1, 4, 16, 2, 64, 2, 64, dtype=torch.float32, device=DEV)
    cache = kvc.PagedKVCache(1, 2, 4, 1, 16, max_seqs=2, max_len=8, device=DEV)
    slots, _, missing = cache.extend(_ints([0, 1]), _ints([0, 5, 10]), 10)  # four pages of two
    assert int(missing) == 2 and (slots == -1).all() and int(cache.context_lens.sum()) == 0
