"""Attention, rotary positions and page bookkeeping in plain 64-bit / integer form, and the bounds that the kernels are held to.

Every function works on CPU tensors and Python loops over sequences; nothing here is shared with the package.
"""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def visible(n_q, n_k, window, sinks):
    """[n_q, n_k]: which keys the last n_q positions of n_k see."""
    p = torch.arange(n_k - n_q, n_k)[:, None]
    j = torch.arange(n_k)[None, :]
    ok = j <= p
    if window:
        ok &= (p - j < window) | (j < sinks)
    return ok


def attend(q, k, v, ok, scale):
    """q [Q, Hq, D], k, v [N, Hkv, D] float64, ok [Q, N] -> out, lse and the bounds' ingredients.

    away: attention of |v|, the size that roundings of the weights and values act on; size: the largest
    scale * sum |q k| a row sees, which roundings of the scores act on; edge: what weights below float16's normal range
    lose (half a step of 2^-24 each, over the sum of the weights, the largest of which is 1)."""
    Q, Hq, D = q.shape
    N, Hkv = k.shape[:2]
    out, away = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((Q, Hq), -math.inf, dtype=torch.float64)
    size = torch.zeros((Q, Hq), dtype=torch.float64)
    edge = torch.zeros((Q, Hq), dtype=torch.float64)
    for h in range(Hq):
        g = h // (Hq // Hkv)
        for i in range(Q):
            seen = ok[i].nonzero().squeeze(1)
            if not seen.numel():
                continue
            kk, vv = k[seen, g], v[seen, g]
            s = (kk @ q[i, h]) * scale
            m = s.max()
            w = torch.exp(s - m)
            lse[i, h] = m + torch.log(w.sum())
            edge[i, h] = len(seen) * 2.0 ** -25 * vv.abs().max() / w.sum()
            w = w / w.sum()
            out[i, h] = w @ vv
            away[i, h] = w @ vv.abs()
            size[i, h] = (kk.abs() @ q[i, h].abs()).max() * scale
    return out, lse, away, size, edge


def check(got, got_lse, ref, dtype, keys, extra_values=0):
    """Holds out and lse to bounds counted in roundings.

    A weight is rounded once to 16 bits (half a step u), an int8 value in a float16 result once more (extra_values), and
    the result once.  In 32 bits: a score is a sum of D products (relative to the sum of their sizes D * 2^-24), its
    exponential some 64 half steps over the whole range of arguments, and a sum over `keys` weights keys * 2^-24."""
    out, lse, away, size, edge = ref
    u, f = half_step(dtype), 2.0 ** -24
    D = out.shape[-1]
    delta = size * (D + 8) * f + (keys + 64) * f
    tol = away * ((1 + extra_values) * u + 2 * delta[..., None]) * (1 + 2 * u) + out.abs() * u
    if dtype == torch.float16:
        tol = tol + edge[..., None] + 2.0 ** -25
    got, got_lse = got.double().cpu(), got_lse.double().cpu()
    assert torch.isfinite(got).all(), "non-finite output"
    bad = (got - out).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} outputs off, worst {float(((got - out).abs() / tol.clamp(min=1e-30)).max()):.2f} of the bound"
    none = torch.isinf(lse)
    assert torch.equal(none, torch.isinf(got_lse)) and (got_lse[none] < 0).all()
    lse_tol = delta + 4 * f * lse.abs()
    assert ((got_lse - lse).abs() <= lse_tol)[~none].all(), "lse off"
    assert (got[none] == 0).all(), "a row that sees nothing must be zero"


def pools(lens, page, Hkv, D, dtype, quant, g, spare=2, fill=math.nan):
    """Keys and values of sequences of the given lengths: per-sequence float64 rows, and a cache pool whose unused slots
    and pages hold `fill` (int8: 127 with a NaN scale), with its table in a random order."""
    need = [-(-max(n, 0) // page) for n in lens]
    P = sum(need) + spare
    order = torch.randperm(P, generator=g)
    table = torch.full((len(lens), max(need + [0]) + 1), -1, dtype=torch.int32)
    if quant:
        kc = torch.full((P, page, Hkv, D), 127, dtype=torch.int8)
        vc = kc.clone()
        ks, vs = torch.full((P, page, Hkv), fill), torch.full((P, page, Hkv), fill)
    else:
        kc = torch.full((P, page, Hkv, D), fill, dtype=dtype)
        vc = kc.clone()
        ks = vs = None
    rows, at = [], 0
    for b, n in enumerate(lens):
        pages = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = pages.to(torch.int32)
        j = torch.arange(max(n, 0))
        pg, sl = pages[j // page] if n > 0 else j, j % page
        if quant:
            k = torch.randint(-127, 128, (len(j), Hkv, D), generator=g).to(torch.int8)
            v = torch.randint(-127, 128, (len(j), Hkv, D), generator=g).to(torch.int8)
            sk, sv = 0.002 + 0.02 * torch.rand((len(j), Hkv), generator=g), 0.002 + 0.02 * torch.rand((len(j), Hkv), generator=g)
            kc[pg, sl], vc[pg, sl], ks[pg, sl], vs[pg, sl] = k, v, sk, sv
            rows.append((k.double() * sk.double()[..., None], v.double() * sv.double()[..., None]))
        else:
            k = torch.randn((len(j), Hkv, D), generator=g).to(dtype)
            v = torch.randn((len(j), Hkv, D), generator=g).to(dtype)
            kc[pg, sl], vc[pg, sl] = k, v
            rows.append((k.double(), v.double()))
    return rows, table, kc, vc, ks, vs


def rotate(x, positions, table, sections, mode):
    """x [T, H, D] -> float64, rotated; positions [axes, T], table [P, R]."""
    half = table.shape[1] // 2
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    y = x.double().clone()
    for i, a in enumerate(axis):
        c, s = table[positions[a].long(), i].double()[:, None], table[positions[a].long(), half + i].double()[:, None]
        e0, e1 = (i, i + half) if mode == "half" else (2 * i, 2 * i + 1)
        x0, x1 = x[..., e0].double(), x[..., e1].double()
        y[..., e0], y[..., e1] = x0 * c - x1 * s, x1 * c + x0 * s
    return y


class Pool:
    """The pages' bookkeeping in plain Python."""

    def __init__(self, table, lens, count, page):
        self.table, self.lens, self.count, self.page = table.tolist(), lens.tolist(), count.tolist(), page

    def free_pages(self):
        return [i for i, c in enumerate(self.count) if c <= 0]

    def free(self, seqs):
        for s in seqs:
            if not 0 <= s < len(self.lens):
                continue
            for j in range(-(-self.lens[s] // self.page)):
                self.count[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.lens[s] = 0

    def fork(self, parents, children):
        """Pairs (src, dst) of pages to copy; None if pages are missing (then nothing has changed), with how many."""
        pairs = []
        todo = [(p, c) for p, c in zip(parents, children) if 0 <= p < len(self.lens) and 0 <= c < len(self.lens)]
        new = self.free_pages()
        need = sum(self.lens[p] % self.page != 0 for p, _ in todo)
        if need > len(new):
            return None, need - len(new)
        for p, c in todo:
            row, n = list(self.table[p]), self.lens[p]
            for j in range(n // self.page):
                self.count[row[j]] += 1
            if n % self.page:
                page = new.pop(0)
                pairs.append((row[n // self.page], page))
                row[n // self.page] = page
                self.count[page] = 1
            self.table[c], self.lens[c] = row, n
        return pairs, 0

    def extend(self, seqs, tokens):
        new = self.free_pages()
        need = over = 0
        for s, t in zip(seqs, tokens):
            if 0 <= s < len(self.lens):
                now = -(-(self.lens[s] + t) // self.page)
                if now > len(self.table[s]):
                    over += now - len(self.table[s])
                else:
                    need += now - -(-self.lens[s] // self.page)
        if over or need > len(new):
            return [-1] * sum(tokens), [-1] * sum(tokens), over or need - len(new)
        slots, positions = [], []
        for s, t in zip(seqs, tokens):
            for _ in range(t):
                if not 0 <= s < len(self.lens):
                    slots.append(-1)
                    positions.append(-1)
                    continue
                n = self.lens[s]
                if n % self.page == 0:
                    page = new.pop(0)
                    self.table[s][n // self.page] = page
                    self.count[page] = 1
                slots.append(self.table[s][n // self.page] * self.page + n % self.page)
                positions.append(n)
                self.lens[s] = n + 1
        return slots, positions, 0

    def compact(self):
        live = sum(c > 0 for c in self.count)
        src = [i for i, c in enumerate(self.count) if c > 0 and i >= live]
        dst = [i for i, c in enumerate(self.count) if c <= 0 and i < live]
        place = dict(zip(src, dst))
        table = [[place.get(p, p) for p in row] for row in self.table]
        count = [max(c, 0) for c in self.count]
        for s, d in place.items():
            count[d], count[s] = count[s], 0
        return table, count, list(zip(src, dst))
