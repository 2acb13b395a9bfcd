"""Plain float64 restatement of the KV-cache operators (test infrastructure):
loops over sequences, heads, tokens and rows, straight from the definitions.

Caches are [B, C, Hkv, D] arrays, ``past`` a list of rows per sequence
(negative: no sequence), ``parents`` None (a chain) or a list of lists."""

import numpy as np


def seen_rows(past, parents, n, capacity):
    """For each token the list of rows it sees, None where it is not there."""
    seen = []
    past = min(past, capacity)
    for i in range(n):
        chain, at = [], i
        while True:
            chain.append(at)
            up = at - 1 if parents is None else parents[at]
            if up == -1 or not 0 <= up < at:
                break
            at = up
        there = past >= 0 and up == -1 and past + i < capacity
        seen.append(list(range(past)) + [past + a for a in sorted(chain)] if there else None)
    return seen


def tree_attention(q, k, v, past, parents=None):
    """(out [B,N,Hq,D], m, l [B,Hq,N])."""
    b, n, hq, d = q.shape
    c, hkv = k.shape[1:3]
    out = np.zeros(q.shape)
    m = np.full((b, hq, n), -np.inf)
    l = np.zeros((b, hq, n))
    for x in range(b):
        for i, rows in enumerate(seen_rows(past[x], parents and parents[x], n, c)):
            if rows is None:
                continue
            for h in range(hq):
                g = h // (hq // hkv)
                s = k[x, rows, g].astype(np.float64) @ q[x, i, h].astype(np.float64) / np.sqrt(d)
                m[x, h, i] = s.max()
                p = np.exp(s - s.max())
                l[x, h, i] = p.sum()
                out[x, i, h] = p @ v[x, rows, g].astype(np.float64) / p.sum()
    return out, m, l


def key_weights(q, k, past, m, l, weights, out, parents=None):
    """The new contents of ``out`` [B,Hkv,C] (weights: [B,Hkv,C] or None)."""
    b, n, hq, d = q.shape
    c, hkv = k.shape[1:3]
    w = np.zeros((b, hkv, c))
    for x in range(b):
        for i, rows in enumerate(seen_rows(past[x], parents and parents[x], n, c)):
            if rows is None:
                continue
            for h in range(hq):
                if not l[x, h, i] > 0 or m[x, h, i] == -np.inf:
                    continue
                g = h // (hq // hkv)
                s = k[x, rows, g].astype(np.float64) @ q[x, i, h].astype(np.float64) / np.sqrt(d)
                w[x, g, rows] += np.exp(s - m[x, h, i]) / l[x, h, i]
    res = np.array(out, dtype=np.float64)
    for x in range(b):
        if past[x] < 0:
            continue
        p = min(past[x], c)
        e = min(p + n, c)
        res[x, :, :e] = w[x, :, :e]
        if weights is not None:
            res[x, :, :p] += weights[x, :, :p]
    return res


def evict(k, v, weights, lens, budget, sinks=0, recent=0, positions=None, kept=None, ends=None):
    """Copies of (k, v, weights, positions, lens) after the eviction; positions
    rows at and past the new lengths are what they were (0 without positions)."""
    k, v, weights = k.copy(), v.copy(), weights.copy()
    b, c, hkv, _ = k.shape
    pos_out = np.zeros((b, hkv, c), np.int32) if positions is None else positions.copy()
    lens_out = []
    for x in range(b):
        n = max(0, min(lens[x], c))
        end = n if ends is None else ends[x]
        old = 0 if kept is None else max(0, min(kept[x], n))
        for h in range(hkv):
            pos = [int(positions[x, h, j]) if j < old else end - n + j for j in range(n)]

            def rank(j):
                if pos[j] < sinks or pos[j] >= end - recent:
                    return (0, 0.0, j)
                w = weights[x, h, j]
                return (2, 0.0, j) if np.isnan(w) else (1, -float(w), j)

            keep = sorted(sorted(range(n), key=rank)[:budget])
            held = set(keep)
            holes = [j for j in range(min(budget, n)) if j not in held]
            movers = [j for j in keep if j >= budget]
            assert len(holes) == len(movers)
            for j in keep:
                if j < budget:
                    pos_out[x, h, j] = pos[j]
            for dst, src in zip(holes, movers):
                k[x, dst, h], v[x, dst, h] = k[x, src, h], v[x, src, h]
                weights[x, h, dst], pos_out[x, h, dst] = weights[x, h, src], pos[src]
        lens_out.append(min(n, budget))
    return k, v, weights, pos_out, lens_out


def commit(k, v, past, path):
    """Copies of one layer's (k, v) and the new lengths."""
    k, v = k.copy(), v.copy()
    lens = []
    for x in range(k.shape[0]):
        if past[x] < 0:
            lens.append(past[x])
            continue
        last, n = -1, 0
        for p in path[x]:
            if p <= last or past[x] + p >= k.shape[1]:
                break
            k[x, past[x] + n], v[x, past[x] + n] = k[x, past[x] + p], v[x, past[x] + p]
            last = p
            n += 1
        lens.append(past[x] + n)
    return k, v, lens
