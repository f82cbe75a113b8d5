"""The attention side of a decoder layer in serving, as cases that can be timed and checked.

Four kinds of call, on the inputs a server has in hand:

* ``decode``  attention of one new token per sequence over a paged key-value cache (``npu_paged_attention``);
* ``prompt``  causal attention of ragged prompts or prompt chunks, with a sliding window and first tokens that stay
              visible (``npu_prompt_attention``), keys contiguous or in the paged cache;
* ``rope``    rotary positions of one or several axes and the write of the new keys and values into the cache
              (``npu_mrope_scatter_kv``);
* ``pages``   the cache's own work: a beam step (free the losers, fork the winners), admission of new prompts (free,
              extend) and compaction of the pool.

``run`` computes each in its plain form (elementary torch operations in 32 bits, rounded once at the end), or, where
``own`` is true, through ``op_plugin_amd``.  Lengths belong to a case; the seed makes the values and the order of the
pages.  A page table's order is a random permutation of the pool: after some hours of serving it is.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
_q = None


def _ops():
    """The package, imported at the first call that needs it."""
    global _q
    if _q is None:
        path = os.path.join(os.getcwd(), "ascend-python_amd")
        if path not in sys.path:
            sys.path.insert(1, path)
        import op_plugin_amd
        _q = op_plugin_amd
    return _q


# ---------------------------------------------------------------- cases


def listed():
    return [
        # One user's chat, a thousand tokens in: the smallest attention call, launch latency and one split.
        dict(name="decode_single", kind="decode", B=1, Hq=32, Hkv=8, D=128, L=997, lens=0, page=16, cache="fp",
             window=0, sinks=0, dtype="bf16"),
        # A decode batch of unequal sequences, a few long ones among many short.
        dict(name="decode_batch_ragged", kind="decode", B=48, Hq=32, Hkv=8, D=128, L=8191, lens=11, page=64,
             cache="fp", window=0, sinks=0, dtype="fp16"),
        # Few sequences with very long contexts: the work is along the cache, a pure stream of 2.1 GB.
        dict(name="decode_long", kind="decode", B=4, Hq=64, Hkv=8, D=128, L=131072, lens=0, page=128, cache="fp",
             window=0, sinks=0, dtype="bf16"),
        # A large batch on an int8 cache with a sliding window and four sink tokens.
        dict(name="decode_int8_window", kind="decode", B=96, Hq=32, Hkv=8, D=128, L=12000, lens=5, page=16,
             cache="int8", window=4096, sinks=4, dtype="bf16"),
        # A short question, nothing cached: 77 tokens.
        dict(name="prompt_short", kind="prompt", B=1, Hq=32, Hkv=8, D=128, T=77, past=0, lens=0, page=0, cache="fp",
             window=0, sinks=0, dtype="bf16"),
        # One prompt of 8192 tokens, full causal attention: compute-bound.
        dict(name="prompt_long", kind="prompt", B=1, Hq=32, Hkv=8, D=128, T=8192, past=0, lens=0, page=0, cache="fp",
             window=0, sinks=0, dtype="bf16"),
        # Chunks of several prompts whose earlier tokens lie in the cache, sliding window and sinks.
        dict(name="prompt_chunk_window", kind="prompt", B=6, Hq=32, Hkv=8, D=128, T=1023, past=12000, lens=3, page=16,
             cache="fp", window=2048, sinks=4, dtype="fp16"),
        # The new tokens of a decode batch, text positions on one axis.
        dict(name="rope_decode", kind="rope", T=64, Hq=32, Hkv=8, D=128, R=128, axes=1, mode="half", page=16,
             dtype="bf16"),
        # A prompt with images: time, height and width positions.
        dict(name="rope_prompt_axes", kind="rope", T=4099, Hq=32, Hkv=8, D=128, R=128, axes=3, mode="half", page=16,
             dtype="bf16"),
        # One step of a beam search (or parallel sampling): half of the hypotheses are dropped, the others forked.
        dict(name="pages_beam", kind="pages", op="beam", layers=16, Hkv=8, D=128, pool=1024, page=16, seqs=32, L=500,
             lens=7, dtype="bf16"),
        # A server replaces 64 finished sequences by new prompts: pages and slots of every new token.
        dict(name="pages_admit", kind="pages", op="admit", layers=0, Hkv=8, D=128, pool=16384, page=16, seqs=256,
             L=1500, lens=9, dtype="bf16"),
        # A pool with holes, after many sequences have gone, is packed to its front.
        dict(name="pages_compact", kind="pages", op="compact", layers=16, Hkv=8, D=128, pool=1024, page=16, seqs=64,
             L=250, lens=13, dtype="bf16"),
    ]


# query heads, key-value heads, width of a head: grouped, multi-head and single-head forms, odd group sizes among them
_HEADS = [(32, 8, 128), (32, 8, 128), (64, 8, 128), (32, 32, 128), (40, 40, 128), (12, 2, 128), (14, 2, 64), (16, 16, 64),
          (20, 4, 80), (24, 8, 96), (8, 1, 256), (48, 1, 128)]


def _spread(rng, lo, hi):
    """A whole number spread over its logarithm; every other one is odd."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        n |= 1
    return max(lo, min(n, hi))


def draw(rng):
    kind = rng.choice(["decode", "decode", "prompt", "prompt", "rope", "pages"])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "pages":
        op = rng.choice(["beam", "admit", "compact"])
        layers, page, L, seqs = rng.choice([4, 7, 16]), rng.choice([16, 32, 48]), _spread(rng, 20, 500), _spread(rng, 4, 48)
        pool = seqs * (-(-L // page) + 1) + rng.randrange(5, 200)
        if op == "admit":
            layers, L, seqs, pool = 0, _spread(rng, 20, 1500), _spread(rng, 8, 256), 16384
        Hkv, D = rng.choice([(8, 128), (4, 128), (2, 64), (5, 80)])
        return dict(kind=kind, op=op, layers=layers, Hkv=Hkv, D=D, pool=pool, page=page, seqs=seqs, L=L,
                    lens=rng.randrange(1, 1000), dtype=dtype)
    Hq, Hkv, D = rng.choice(_HEADS)
    if kind == "rope":
        axes = rng.choice([1, 3])
        R = D if rng.random() < 0.7 else D // 2
        most = 4099 * 48 // (Hq + 2 * Hkv)
        return dict(kind=kind, T=_spread(rng, 1, most), Hq=Hq, Hkv=Hkv, D=D, R=R, axes=axes,
                    mode=rng.choice(["half", "half", "interleave"]), page=rng.choice([16, 48, 128]), dtype=dtype)
    window = rng.choice([0, 0, 128, 1000, 4096])
    sinks = rng.choice([0, 1, 4]) if window else 0
    cache = rng.choice(["fp", "fp", "int8"])
    page = rng.choice([16, 16, 48, 64, 128])
    lens = rng.choice([0, rng.randrange(1, 1000)])
    if kind == "decode":
        B = _spread(rng, 1, 128)
        L = _spread(rng, 1, max(1, min(131072, (1 << 28) // (B * Hkv * D))))
        return dict(kind=kind, B=B, Hq=Hq, Hkv=Hkv, D=D, L=L, lens=lens, page=page, cache=cache, window=window,
                    sinks=sinks, dtype=dtype)
    B, T = _spread(rng, 1, 8), _spread(rng, 1, 4096)
    past = rng.choice([0, _spread(rng, 1, 12000)])
    while B * Hq * T * (T + past) > 1 << 30:
        T, past = max(1, T * 2 // 3), past * 2 // 3
    if past == 0 and rng.random() < 0.7:
        page, cache = 0, "fp"
    return dict(kind=kind, B=B, Hq=Hq, Hkv=Hkv, D=D, T=T, past=past, lens=lens, page=page, cache=cache, window=window,
                sinks=sinks, dtype=dtype)


def _lengths(case, most, salt):
    """The lengths of a case's sequences: all `most`, or spread over their logarithm with `most` first."""
    n = case.get("B") or case["seqs"]
    if not case["lens"]:
        return [most] * n
    rng = random.Random(case["lens"] * 7919 + salt)
    return [most] + [_spread(rng, 1, most) if most else 0 for _ in range(n - 1)]


def _prompt_lengths(case):
    q = _lengths(case, case["T"], 1)
    past = _lengths(case, case["past"], 2)
    return q, [a + b for a, b in zip(q, past)]


# ---------------------------------------------------------------- inputs


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _paged(g, case, lens):
    """A cache pool, and the table of sequences of the given lengths over a random order of its pages."""
    S, Hkv, D, dtype = case["page"], case["Hkv"], case["D"], _DT[case["dtype"]]
    need = [-(-n // S) for n in lens]
    width, pool = max(need) + 1, sum(need) + 3
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([0] + need, device="cuda").cumsum(0)
    j = torch.arange(width, device="cuda")
    at = first[:-1, None] + j
    table = torch.where(at < first[1:, None], order[at.clamp(max=pool - 1)], -1).to(torch.int32).contiguous()
    state = dict(table=table, lens=_ints(lens))
    for name in ("k", "v"):
        if case["cache"] == "int8":
            state[name] = torch.randint(-127, 128, (pool, S, Hkv, D), generator=g, device="cuda", dtype=torch.int8)
            state[name + "_scale"] = 0.01 + 0.02 * torch.rand((pool, S, Hkv), generator=g, device="cuda")
        else:
            state[name] = _normal(g, (pool, S, Hkv, D), dtype)
            state[name + "_scale"] = None
    return state


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, dtype, D = case["kind"], _DT[case["dtype"]], case["D"]
    if kind == "decode":
        lens = _lengths(case, case["L"], 0)
        return dict(_paged(g, case, lens), case=case, q=_normal(g, (case["B"], case["Hq"], D), dtype))
    if kind == "prompt":
        q_lens, kv_lens = _prompt_lengths(case)
        cu = [0]
        cu += [cu[-1] + sum(q_lens[:i + 1]) for i in range(len(q_lens))]
        state = dict(case=case, q=_normal(g, (cu[-1], case["Hq"], D), dtype), cu=_ints(cu), longest=max(kv_lens))
        if case["page"]:
            state.update(_paged(g, case, kv_lens))
        else:
            state.update(k=_normal(g, (cu[-1], case["Hkv"], D), dtype), v=_normal(g, (cu[-1], case["Hkv"], D), dtype),
                         k_scale=None, v_scale=None)
        return state
    if kind == "rope":
        T, Hq, Hkv, R, S = case["T"], case["Hq"], case["Hkv"], case["R"], case["page"]
        far = 32768  # positions of the table
        angle = torch.arange(far, dtype=torch.float64, device="cuda")[:, None] * \
            10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
        table = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        pool = -(-T // S) + 8
        qkv = _normal(g, (T, (Hq + 2 * Hkv) * D), dtype)  # the fused projection's output; q, k and v are views of it
        q, k, v = qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1)
        shape = (T,) if case["axes"] == 1 else (case["axes"], T)
        return dict(case=case, q=q.view(T, Hq, D), k=k.view(T, Hkv, D), v=v.view(T, Hkv, D), cos_sin=table,
                    positions=torch.randint(0, far, shape, generator=g, device="cuda", dtype=torch.int32),
                    slots=torch.randperm(pool * S, generator=g, device="cuda")[:T].to(torch.int32),
                    sections=None if case["axes"] == 1 else [R // 2 - 2 * (3 * R // 16), 3 * R // 16, 3 * R // 16],
                    k_cache=_normal(g, (pool, S, Hkv, D), dtype), v_cache=_normal(g, (pool, S, Hkv, D), dtype))
    S, pool, seqs = case["page"], case["pool"], case["seqs"]
    lens = _lengths(case, case["L"], 3)
    need = [-(-n // S) for n in lens]
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([0] + need, device="cuda").cumsum(0)
    at = first[:-1, None] + torch.arange(max(need) + 1, device="cuda")
    used = at < first[1:, None]
    lens_t = _ints(lens)
    if case["op"] == "beam":  # the second half of the slots are the losers, empty at first
        used[seqs // 2:] = False
        lens_t[seqs // 2:] = 0
    table = torch.where(used, order[at.clamp(max=pool - 1)], -1).to(torch.int32).contiguous()
    count = torch.zeros(pool, dtype=torch.int32, device="cuda")
    count[table[used].long()] = 1
    state = dict(case=case, table=table, lens=lens_t, count=count)
    if case["layers"]:
        state["pool"] = _normal(g, (case["layers"], 2, pool, S, case["Hkv"], D), dtype)
        state["caches"] = list(state["pool"].flatten(0, 1).unbind(0))
    half = seqs // 2
    if case["op"] == "beam":
        state["parents"] = torch.randint(0, half, (seqs - half,), generator=g, device="cuda", dtype=torch.int32)
        state["children"] = torch.arange(half, seqs, device="cuda", dtype=torch.int32)
    elif case["op"] == "admit":
        going = torch.randperm(seqs, generator=g, device="cuda")[:max(1, seqs // 4)].to(torch.int32)
        new = _lengths(dict(case, seqs=int(going.numel())), case["L"], 4)
        state.update(going=going, cu=torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32), total=sum(new),
                     longest=max(new))
    return state


# ---------------------------------------------------------------- plain forms


def _rows(cache, scale, table, n):
    """The first n tokens of every sequence out of the pages, [B, n, Hkv, D] in 32 bits."""
    j = torch.arange(n, device=table.device)
    page = table[:, j // cache.shape[1]].clamp(min=0).long()
    rows = cache[page, j % cache.shape[1]].float()
    return rows if scale is None else rows * scale[page, j % cache.shape[1]][..., None]


def _attend(q, k, v, position, visible):
    """q [B, Q, Hq, D], k, v [B, N, Hkv, D], all in 32 bits, visible [B, Q, N] -> out [B, Q, Hq, D], lse [B, Q, Hq]."""
    B, Q, Hq, D = q.shape
    N, Hkv = k.shape[1:3]
    qh = q.view(B, Q, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    s = (qh @ k.permute(0, 2, 3, 1).contiguous()).view(B, Hkv, Hq // Hkv, Q, N)
    s.mul_(1.0 / math.sqrt(D)).masked_fill_(~visible[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(m.clamp(min=torch.finfo(torch.float32).min)).exp_()
    total = p.sum(-1, keepdim=True)
    out = p.view(B, Hkv, -1, N) @ v.permute(0, 2, 1, 3).contiguous()
    out = out.view(B, Hkv, -1, Q, D) / total.clamp(min=torch.finfo(torch.float32).tiny)
    lse = (m + total.log()).squeeze(-1)
    return out.permute(0, 3, 1, 2, 4).reshape(B, Q, Hq, D), lse.permute(0, 3, 1, 2).reshape(B, Q, Hq)


def _seen(case, position, n):
    """Which of n keys a query at `position` sees."""
    j = torch.arange(n, device=position.device)
    p = position[..., None]
    near = (p - j < case["window"]) | (j < case["sinks"]) if case["window"] else torch.ones_like(p - j, dtype=torch.bool)
    return (j <= p) & near


def _plain_decode(s):
    case = s["case"]
    n = case["L"]
    k, v = _rows(s["k"], s["k_scale"], s["table"], n), _rows(s["v"], s["v_scale"], s["table"], n)
    position = (s["lens"] - 1)[:, None]
    out, lse = _attend(s["q"].float()[:, None], k, v, position, _seen(case, position, n))
    return out[:, 0].to(s["q"].dtype), lse[:, 0]


def _plain_prompt(s):
    case, cu, q = s["case"], s["cu"].long(), s["q"]
    T = case["T"]
    q_lens = cu[1:] - cu[:-1]
    i = torch.arange(T, device=q.device)
    padded = q[(cu[:-1, None] + i).clamp(max=q.shape[0] - 1)].float()  # [B, T, Hq, D]
    n = s["longest"]
    if case["page"]:
        k, v, kv_lens = _rows(s["k"], s["k_scale"], s["table"], n), _rows(s["v"], s["v_scale"], s["table"], n), s["lens"]
    else:
        at = (cu[:-1, None] + torch.arange(n, device=q.device)).clamp(max=q.shape[0] - 1)
        k, v, kv_lens = s["k"][at].float(), s["v"][at].float(), q_lens
    position = (kv_lens - q_lens)[:, None] + i
    out, lse = _attend(padded, k, v, position, _seen(case, position, n))
    t = torch.arange(q.shape[0], device=q.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return out[b, t - cu[b]].to(q.dtype), lse[b, t - cu[b]]


def _rotated(x, cos, sin, mode):
    """x [T, H, D] with its first dimensions rotated, cos and sin [T, R / 2]; in 32 bits, rounded to x's type."""
    R = 2 * cos.shape[1]
    c, s = cos[:, None], sin[:, None]
    turn, rest = x[..., :R].float(), x[..., R:]
    if mode == "half":
        a, b = turn[..., :R // 2], turn[..., R // 2:]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    else:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    return torch.cat([turned.to(x.dtype), rest], dim=-1)


def _plain_rope(s):
    half = s["case"]["R"] // 2
    i = torch.arange(half, device=s["q"].device)
    at = s["positions"].long()
    if s["sections"] is None:
        at = at[:, None].expand(-1, half)
    else:
        first, second = s["sections"][0], s["sections"][0] + s["sections"][1]
        at = at[(i >= first).long() + (i >= second).long()].t()
    cos, sin = s["cos_sin"][at, i], s["cos_sin"][at, half + i]
    q, k = _rotated(s["q"], cos, sin, s["case"]["mode"]), _rotated(s["k"], cos, sin, s["case"]["mode"])
    s["k_cache"].flatten(0, 1)[s["slots"].long()] = k
    s["v_cache"].flatten(0, 1)[s["slots"].long()] = s["v"]
    return q, s["k_cache"], s["v_cache"]


def _plain_free(s, seqs):
    S, rows = s["case"]["page"], s["table"][seqs.long()]
    j = torch.arange(rows.shape[1], device=rows.device)
    held = j < ((s["lens"][seqs.long()] + S - 1) // S)[:, None]
    s["count"].index_add_(0, rows.clamp(min=0).flatten().long(), -held.flatten().to(torch.int32))
    s["table"][seqs.long()] = -1
    s["lens"][seqs.long()] = 0


def _plain_beam(s):
    S, children, parents = s["case"]["page"], s["children"].long(), s["parents"].long()
    _plain_free(s, children)
    lens, rows = s["lens"][parents], s["table"][parents]
    j = torch.arange(rows.shape[1], device=rows.device)
    s["count"].index_add_(0, rows.clamp(min=0).flatten().long(), (j < (lens // S)[:, None]).flatten().to(torch.int32))
    started = (lens % S != 0).nonzero().squeeze(1)
    new = (s["count"] == 0).nonzero().squeeze(1)[:started.numel()]
    last = (lens // S).long()[started]
    s["pool"][:, :, new] = s["pool"][:, :, rows[started, last].long()]
    rows[started, last] = new.to(torch.int32)
    s["count"][new] = 1
    s["table"][children] = rows
    s["lens"][children] = lens
    return s["pool"], s["table"], s["lens"], s["count"]


def _plain_admit(s):
    S, going, cu = s["case"]["page"], s["going"].long(), s["cu"]
    _plain_free(s, going)
    tokens = cu[1:] - cu[:-1]
    pages = (tokens + S - 1) // S
    first = pages.cumsum(0) - pages
    new = (s["count"] == 0).nonzero().squeeze(1)
    j = torch.arange(s["table"].shape[1], device=cu.device)
    held = j < pages[:, None]
    rows = torch.where(held, new[(first[:, None] + j).clamp(max=new.numel() - 1)].to(torch.int32), -1)
    s["count"][rows[held].long()] = 1
    s["table"][going] = rows.to(torch.int32)
    s["lens"][going] = tokens
    t = torch.arange(s["total"], device=cu.device, dtype=torch.int32)
    b = torch.searchsorted(cu, t, right=True) - 1
    i = t - cu[b]
    return rows[b, (i // S).long()] * S + i % S, i, s["table"], s["lens"], s["count"]


def _plain_compact(s):
    count, table = s["count"], s["table"]
    live = count > 0
    ids = torch.arange(count.numel(), device=count.device)
    front = ids < live.sum()
    src, dst = (live & ~front).nonzero().squeeze(1), (~live & front).nonzero().squeeze(1)
    s["pool"][:, :, dst] = s["pool"][:, :, src]
    place = ids.to(torch.int32)
    place[src] = dst.to(torch.int32)
    moved = count.clone()
    moved[dst], moved[src] = count[src], 0
    return s["pool"], torch.where(table >= 0, place[table.clamp(min=0).long()], table), moved


# ---------------------------------------------------------------- one pass


def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if not own:
        if kind == "pages":
            return {"beam": _plain_beam, "admit": _plain_admit, "compact": _plain_compact}[case["op"]](s)
        return {"decode": _plain_decode, "prompt": _plain_prompt, "rope": _plain_rope}[kind](s)
    q = _ops()
    if kind == "decode":
        return q.npu_paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], key_scale=s["k_scale"],
                                     value_scale=s["v_scale"], window=case["window"], sinks=case["sinks"])
    if kind == "prompt":
        paged = dict(block_table=s["table"], context_lens=s["lens"]) if case["page"] else {}
        return q.npu_prompt_attention(s["q"], s["k"], s["v"], s["cu"], key_scale=s["k_scale"], value_scale=s["v_scale"],
                                      window=case["window"], sinks=case["sinks"], **paged)
    if kind == "rope":
        out = q.npu_mrope_scatter_kv(s["positions"], s["q"], s["k"], s["v"], s["cos_sin"], s["k_cache"], s["v_cache"],
                                     s["slots"], mrope_section=s["sections"], rotary_mode=case["mode"])
        return out, s["k_cache"], s["v_cache"]
    S = case["page"]
    if case["op"] == "beam":
        q.npu_kv_free(s["table"], s["lens"], s["count"], s["children"], S)
        q.npu_kv_fork(s["caches"], s["table"], s["lens"], s["count"], s["parents"], s["children"], S)
        return s["pool"], s["table"], s["lens"], s["count"]
    if case["op"] == "admit":
        q.npu_kv_free(s["table"], s["lens"], s["count"], s["going"], S)
        slots, positions, _ = q.npu_kv_extend(s["table"], s["lens"], s["count"], s["going"], s["cu"], s["total"], S)
        return slots, positions, s["table"], s["lens"], s["count"]
    table, count, _ = q.npu_kv_compact(s["caches"], s["table"], s["count"])
    return s["pool"], table, count


# ---------------------------------------------------------------- what a pass cannot do without


def _pairs(case, q_len, kv_len):
    """Visible (query, key) pairs of one sequence, and the keys that any of its queries sees."""
    pairs = 0
    for i in range(q_len):
        p = kv_len - q_len + i
        n = p + 1
        if case["window"] and n > case["window"]:
            n = case["window"] + min(case["sinks"], n - case["window"])
        pairs += n
    low = max(0, kv_len - q_len + 1 - case["window"]) if case["window"] else 0
    return pairs, kv_len - low + min(case["sinks"], low)


def work(case):
    kind, D = case["kind"], case["D"]
    if kind in ("decode", "prompt"):
        if kind == "decode":
            q_lens, kv_lens = [1] * case["B"], _lengths(case, case["L"], 0)
        else:
            q_lens, kv_lens = _prompt_lengths(case)
        seen = [_pairs(case, a, b) for a, b in zip(q_lens, kv_lens)]
        token = case["Hkv"] * (2 * D + 8 if case["cache"] == "int8" else 4 * D)
        return dict(bytes=sum(keys for _, keys in seen) * token + sum(q_lens) * case["Hq"] * (4 * D + 4),
                    flops=4 * D * case["Hq"] * sum(pairs for pairs, _ in seen))
    if kind == "rope":
        return dict(bytes=case["T"] * (4 * D * (case["Hq"] + 2 * case["Hkv"]) + 4 * case["R"] + 4 * case["axes"] + 4),
                    flops=0)
    S, lens = case["page"], _lengths(case, case["L"], 3)
    page = case["layers"] * 2 * S * case["Hkv"] * D * 2
    pages = [-(-n // S) for n in lens]
    if case["op"] == "beam":
        half = case["seqs"] // 2
        share = (case["seqs"] - half) / half
        return dict(bytes=int(share * sum(2 * page * (n % S != 0) + 24 * k for n, k in zip(lens[:half], pages[:half]))),
                    flops=0)
    if case["op"] == "admit":
        new = _lengths(dict(case, seqs=max(1, case["seqs"] // 4)), case["L"], 4)
        return dict(bytes=8 * sum(new) + 24 * sum(-(-n // S) for n in new), flops=0)
    live = sum(pages)
    moved = live * (case["pool"] - live) // case["pool"]  # live pages in a random order that lie past the front
    return dict(bytes=2 * page * moved + 8 * case["pool"] + 8 * case["seqs"] * (max(pages) + 1), flops=0)


# ---------------------------------------------------------------- the definition in 64 bits


def _sequence(s, name, b, n):
    """The n keys or values of sequence b, [n, Hkv, D] in 64 bits."""
    cache, scale = s[name], s[name + "_scale"]
    if "table" not in s:
        start = int(s["cu"][b])
        return cache[start:start + n].double()
    S = cache.shape[1]
    pages = s["table"][b, :-(-n // S)].long()
    rows = cache[pages].flatten(0, 1)[:n].double()
    return rows if scale is None else rows * scale[pages].flatten(0, 1)[:n].double().unsqueeze(-1)


def exact(case, seed):
    kind = case["kind"]
    s = prepare(case, seed)
    if kind == "pages":
        return None  # whole numbers and copies: no value is computed
    if kind == "rope":
        half = case["R"] // 2
        axis = [0] * half
        if s["sections"]:
            axis = [a for a, n in enumerate(s["sections"]) for _ in range(n)]
        at = torch.stack([(s["positions"] if s["positions"].dim() == 1 else s["positions"][a]).long() for a in axis])
        pair = torch.arange(half, device="cuda")[:, None]
        turn = torch.complex(s["cos_sin"].double()[at, pair], s["cos_sin"].double()[at, half + pair]).t()[:, None]

        def turned(x):
            y = x.double().clone()
            if case["mode"] == "half":
                z = torch.complex(y[..., :half], y[..., half:2 * half]) * turn
                y[..., :half], y[..., half:2 * half] = z.real, z.imag
            else:
                y[..., :2 * half] = torch.view_as_real(torch.view_as_complex(y[..., :2 * half].unflatten(-1, (half, 2))
                                                                             .contiguous()) * turn).flatten(-2)
            return y

        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        k_cache.flatten(0, 1)[s["slots"].long()] = turned(s["k"])
        v_cache.flatten(0, 1)[s["slots"].long()] = s["v"].double()
        return turned(s["q"]), k_cache, v_cache
    if kind == "decode":
        q_lens, kv_lens = [1] * case["B"], _lengths(case, case["L"], 0)
    else:
        q_lens, kv_lens = _prompt_lengths(case)
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    outs, lses, start = [], [], 0
    for b, (n_q, n) in enumerate(zip(q_lens, kv_lens)):
        q = s["q"][start:start + n_q].double()
        start += n_q
        k, v = _sequence(s, "k", b, n), _sequence(s, "v", b, n)
        out, lse = torch.empty_like(q), torch.empty((n_q, Hq), dtype=torch.float64, device="cuda")
        back = torch.arange(n - n_q, n, device="cuda")[:, None] - torch.arange(n, device="cuda")  # how far back a key is
        hidden = back < 0
        if case["window"]:
            hidden |= (back >= case["window"]) & (torch.arange(n, device="cuda") >= case["sinks"])
        for h in range(Hq):
            g = h * Hkv // Hq
            score = torch.mv(k[:, g], q[0, h])[None] if n_q == 1 else q[:, h] @ k[:, g].t()
            score = (score / math.sqrt(D)).masked_fill(hidden, -math.inf)
            lse[:, h] = torch.logsumexp(score, -1)
            out[:, h] = torch.softmax(score, -1) @ v[:, g]
        outs.append(out)
        lses.append(lse)
    return torch.cat(outs), torch.cat(lses)
