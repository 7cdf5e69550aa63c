"""Attention that reads a part of its cache, restated in 64 bits: page bounds, the selection of pages, attention over listed pages.

Everything is written for one sequence at a time over its keys and values in order of position ([tokens, kv_heads, d])."""
import math

import torch

PAGE = 64


def bounds_of(keys):
    """[full pages, kv_heads, 2, d]: lowest, then highest values of the pages that are full."""
    n = keys.shape[0] // PAGE
    k = keys[:n * PAGE].reshape(n, PAGE, keys.shape[1], keys.shape[2])
    return torch.stack((k.amin(1), k.amax(1)), 2)


def scores(q, bounds):
    """q [heads, d], bounds [pages, kv_heads, 2, d] -> [kv_heads, pages]: per head and channel the larger of q lo and q hi, which is
    q hi for q > 0, q lo for q < 0 and nothing for q = 0; a score that is NaN counts as -inf."""
    kvh = bounds.shape[1]
    q = q.double().reshape(kvh, -1, 1, q.shape[-1])
    b = bounds.double()
    low, high = b[:, :, 0].permute(1, 0, 2).unsqueeze(1), b[:, :, 1].permute(1, 0, 2).unsqueeze(1)
    terms = torch.where(q > 0, q * high, torch.where(q < 0, q * low, q * 0.0))
    s = terms.sum((1, 3))
    return torch.where(s.isnan(), -math.inf, s)


def choose(score, own, top, first, last):
    """The chosen pages of one kv head, ascending: score [>= own + 1]."""
    n = own + 1
    if n <= top:
        return list(range(n))
    rest = list(range(first, n - last))
    s = [float(score[j]) for j in rest]
    order = sorted(range(len(rest)), key=lambda i: (-s[i], rest[i]))
    return sorted(list(range(first)) + list(range(n - last, n)) + [rest[i] for i in order[:top - first - last]])


def attend(q, keys, values, listed, pos, scale):
    """One row: q [heads, d]; keys, values [tokens, kv_heads, d]; listed: one list of pages a kv head.  Returns the row [heads, d]
    and the weighted sum of the values' sizes, which bounds what rounding the weights can do."""
    kvh, d = keys.shape[1], keys.shape[2]
    G = q.shape[0] // kvh
    out = torch.zeros((q.shape[0], d), dtype=torch.float64)
    size = torch.zeros_like(out)
    for g in range(kvh):
        at = [t for j in listed[g] if j >= 0 for t in range(j * PAGE, (j + 1) * PAGE) if t <= pos]
        if not at:
            continue
        k, v = keys[at, g].double(), values[at, g].double()
        for h in range(g * G, (g + 1) * G):
            p = torch.softmax(k @ q[h].double() * scale, 0)
            out[h] = p @ v
            size[h] = p @ v.abs()
    return out, size
