"""Trees of drafted tokens in plain Python: random trees, their masks, and what a row of one sees."""
import random

import torch


def random_tree(rng, n):
    """Parents of n rows, -1 for the root."""
    return [-1] + [max(0, i - rng.choice([1, 1, 2, 3, 7])) for i in range(1, n)] if n else []


def ancestors(tree):
    """Sets: each row with its ancestors."""
    seen = []
    for i, p in enumerate(tree):
        seen.append((seen[p] if p >= 0 else set()) | {i})
    return seen


def mask_words(rows, words):
    """Rows as sets of whole numbers -> int64 [len(rows), words]."""
    out = torch.zeros((len(rows), words), dtype=torch.int64)
    for t, row in enumerate(rows):
        for w in range(words):
            bits = sum(1 << (k - 64 * w) for k in row if 64 * w <= k < 64 * w + 64)
            out[t, w] = bits - (1 << 64) if bits >> 63 else bits
    return out


def visible(rows, n_keys, window, sinks):
    """[len(rows), n_keys] bool for the n rows (sets of bits below 64 * words) of a sequence of n_keys tokens."""
    n = len(rows)
    past = n_keys - n
    ok = torch.zeros((n, n_keys), dtype=torch.bool)
    for i, row in enumerate(rows):
        p = past - 1 + sum(k < n for k in row)
        for j in range(max(past, 0)):
            ok[i, j] = not window or p - j < window or j < sinks
        for k in row:
            if k < n and past + k >= 0:
                ok[i, past + k] = True
    return ok


def trees(seed, sizes):
    rng = random.Random(seed)
    return [random_tree(rng, n) for n in sizes]
