"""Paged key-value cache and draft verification -- test infrastructure only.

Restated in float64 numpy from the definitions in include/soupsuck_amd.h (the reference
trains only and has no counterpart).  Caches are [pages, kv heads, page size, D], block
tables lists of page numbers, a page outside the cache holds nothing.

Pins (tests/test_oracle_cache.py): attention of a whole prompt over a cache equals
oracle.attention.forward; a window over all rows, and all rows as sinks, change nothing;
append equals oracle.rope's rotation up to its roundings; eviction against sorting by hand;
verification against the distribution that its tokens must have.
"""

import math

import numpy as np


def held(length, table, page_size, pages):
    """Rows j < length with their (page, row of the page); rows on no page left out."""
    for j in range(max(0, min(int(length), len(table) * page_size))):
        page = int(table[j // page_size])
        if 0 <= page < pages:
            yield j, page, j % page_size


def rotate(x, cos, sin):
    """x [..., D] turned by cos / sin [..., D] (halves c and c + D / 2)."""
    x, cos, sin = (np.asarray(t, np.float64) for t in (x, cos, sin))
    half = x.shape[-1] // 2
    return x * cos + np.concatenate((-x[..., half:], x[..., :half]), -1) * sin


def append(k_cache, v_cache, k, v, table, lengths, cu, cos=None, sin=None):
    """The caches (float64 copies) after the packed tokens' k / v [T, heads, D]."""
    kc, vc = np.array(k_cache, np.float64), np.array(v_cache, np.float64)
    pages, _, size, _ = kc.shape
    k = np.asarray(k, np.float64)
    if cos is not None:
        k = rotate(k, np.asarray(cos)[:, None], np.asarray(sin)[:, None])
    for b, length in enumerate(lengths):
        for t in range(int(cu[b]), int(cu[b + 1])):
            row = int(length) - int(cu[b + 1]) + t
            if row < 0 or row >= len(table[b]) * size:
                continue
            page = int(table[b][row // size])
            if 0 <= page < pages:
                kc[page, :, row % size] = k[t]
                vc[page, :, row % size] = np.asarray(v[t], np.float64)
    return kc, vc


def attention(q, k_cache, v_cache, table, lengths, cu, scale, window=None, sinks=0):
    """o [T, Hq, D], the sums of |p v| (for tolerances), the greatest sum of |q k| scale of a
    row, and per sequence the weights [heads, rows of the table * page size]."""
    q = np.asarray(q, np.float64)
    kc, vc = np.asarray(k_cache, np.float64), np.asarray(v_cache, np.float64)
    pages, heads, size, dim = kc.shape
    group = q.shape[1] // heads
    out, spread, reach = np.zeros_like(q), np.zeros_like(q), 0.0
    weights = np.zeros((len(lengths), heads, len(table[0]) * size))
    for b, length in enumerate(lengths):
        rows = list(held(length, table[b], size, pages))
        for t in range(int(cu[b]), min(int(cu[b + 1]), q.shape[0])):
            at = int(length) - int(cu[b + 1]) + t
            seen = [r for r in rows if r[0] <= at
                    and (not window or r[0] > at - window or r[0] < sinks)]
            if not seen:
                continue
            index, page, row = (np.array(c) for c in zip(*seen))
            for h in range(heads):
                keys, values = kc[page, h, row], vc[page, h, row]
                qs = q[t, h * group:(h + 1) * group]
                s = qs @ keys.T * scale
                p = np.exp(s - s.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                out[t, h * group:(h + 1) * group] = p @ values
                spread[t, h * group:(h + 1) * group] = p @ np.abs(values)
                reach = max(reach, float((np.abs(qs) @ np.abs(keys).T).max()) * abs(scale))
                weights[b, h, index] += p.sum(0)
    return out, spread, reach, weights


def evict(k_cache, v_cache, table, lengths, weights, out_table, budget, sinks, recent):
    """(new lengths, new weights, caches) after the kept rows moved to out_table's pages."""
    kc, vc = np.array(k_cache), np.array(v_cache)
    pages, heads, size, _ = kc.shape
    new_weights = np.zeros((len(lengths), heads, len(out_table[0]) * size), np.float32)
    new_lengths = []
    for b, length in enumerate(lengths):
        length = max(0, min(int(length), len(table[b]) * size))
        keep = min(length, budget)
        new_lengths.append(keep)
        for h in range(heads):
            kept = list(range(length))
            if length > budget:
                middle = range(sinks, length - recent)

                def order(j):
                    w = float(weights[b, h, j])
                    return (0, 0.0, j) if math.isnan(w) else (1, -w, j)

                heavy = sorted(middle, key=order)[:budget - sinks - recent]
                kept = sorted([*range(sinks), *heavy, *range(length - recent, length)])
            for i, j in enumerate(kept):
                new_weights[b, h, i] = weights[b, h, j]
                to, source = int(out_table[b][i // size]), int(table[b][j // size])
                if not 0 <= to < pages:
                    continue
                good = 0 <= source < pages
                kc[to, h, i % size] = k_cache[source, h, j % size] if good else 0
                vc[to, h, i % size] = v_cache[source, h, j % size] if good else 0
    return np.array(new_lengths, np.int32), new_weights, kc, vc


def probabilities(logits, temperature):
    """softmax(logits / T): NaN as -inf, +inf logits share the whole, none without any."""
    x = np.array(logits, np.float64)
    x[np.isnan(x)] = -np.inf
    top = x.max()
    if top == -np.inf:
        return np.zeros_like(x)
    if top == np.inf:
        return (x == np.inf) / np.count_nonzero(x == np.inf)
    e = np.exp((x - top) / temperature)
    return e / e.sum()


def draw(mass, u):
    """The first place at which the running sum exceeds u times the whole; -1 without mass."""
    total = np.cumsum(mass)
    if not total[-1] > 0:
        return -1
    over = np.nonzero((total > u * total[-1]) & (mass > 0))[0]
    return int(over[0]) if len(over) else int(np.nonzero(mass > 0)[0][-1])


def verify(target, tokens, uniform, draft=None, counts=None, temperature=1.0):
    """(accepted, tokens) of one sequence: target [G + 1, V], tokens [G], uniform [G + 1]."""
    drafts = len(tokens)
    vocab = target.shape[1]
    count = drafts if counts is None else max(0, min(int(counts), drafts))
    out = []
    last = None
    for i in range(count):
        x = int(tokens[i])
        if temperature == 0:
            p = np.array(target[i], np.float64)
            p[np.isnan(p)] = -np.inf
            best = int(p.argmax()) if p.max() > -np.inf else -1
            if best >= 0 and best == x:
                out.append(x)
                continue
            last = best
            break
        p = probabilities(target[i], temperature)
        q = np.zeros(vocab) if draft is None else probabilities(draft[i], temperature)
        if draft is None and 0 <= x < vocab:
            q[x] = 1.0
        if 0 <= x < vocab and float(uniform[i]) * q[x] < p[x]:
            out.append(x)
            continue
        rest = np.maximum(p - q, 0)
        last = draw(rest if rest.sum() > 0 else p, float(uniform[drafts]))
        break
    if last is None:
        if temperature == 0:
            p = np.array(target[count], np.float64)
            p[np.isnan(p)] = -np.inf
            last = int(p.argmax()) if p.max() > -np.inf else -1
        else:
            last = draw(probabilities(target[count], temperature), float(uniform[drafts]))
    return len(out), out + [last] + [-1] * (drafts - len(out))
