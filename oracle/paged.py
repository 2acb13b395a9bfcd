"""Plain float64 restatement of rotary positions and of the paged 8-bit cache
(test infrastructure): loops over sequences, heads, pages and tokens, straight
from the definitions.

A pool is a dict of k [P, Hkv, rows, D] and v [P, Hkv, D, rows] as the values of
their e4m3 codes, and k_scale, v_scale [P, Hkv]."""

import math

import numpy as np


def e4m3(x):
    """The e4m3 value nearest to x (ties to the even code), for |x| <= 448; NaN
    for what is not finite."""
    x = np.asarray(x, np.float64)
    ok = np.isfinite(x)
    y = np.where(ok, x, 0.0)
    _, e = np.frexp(y)
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.where(ok, np.round(y / step) * step, np.nan)


def block_scale(amax):
    """The smallest power of two s >= 2^-126 with amax <= 448 s."""
    s = 2.0 ** -126
    if amax > 0:
        s = max(s, 2.0 ** math.floor(math.log2(amax / 448.0) - 2))
        while amax > 448.0 * s:
            s *= 2
    return s


def rotate(x, positions, inv_freq, factor=1.0, interleaved=False, backward=False):
    """x [tokens, heads, D] turned to positions [tokens]."""
    x = np.asarray(x, np.float64)
    y = x.copy()
    half = len(inv_freq)
    for t, pos in enumerate(positions):
        for i, f in enumerate(inv_freq):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            angle = math.fmod(float(pos) * f, 2 * math.pi) * (-1 if backward else 1)
            c, s = factor * math.cos(angle), factor * math.sin(angle)
            y[t, :, a] = x[t, :, a] * c - x[t, :, b] * s
            y[t, :, b] = x[t, :, b] * c + x[t, :, a] * s
    return y


def page_of(table, pages, at):
    return int(table[at]) if 0 <= at < len(table) and 0 <= table[at] < pages else None


def append(pool, table, past, counts, k, v):
    """Writes k (turned already) and v [B, N, Hkv, D] into the pool."""
    rows = pool["k"].shape[2]
    for b, n in enumerate(counts):
        if past[b] < 0:
            continue
        for p in range(past[b] // rows, (past[b] + n - 1) // rows + 1 if n > 0 else 0):
            page = page_of(table[b], len(pool["k"]), p)
            if page is None:
                continue
            lo, hi = max(past[b] - p * rows, 0), min(past[b] + n - p * rows, rows)
            for h in range(pool["k"].shape[1]):
                for name, x in (("k", k), ("v", v)):
                    codes = pool[name][page, h] if name == "k" else pool[name][page, h].T
                    new = np.asarray(x[b, p * rows + lo - past[b]:p * rows + hi - past[b], h], np.float64)
                    scale = block_scale(np.abs(new[np.isfinite(new)]).max(initial=0.0))
                    if lo > 0:
                        was = pool[name + "_scale"][page, h]
                        scale = max(scale, was)
                        codes[:lo] = e4m3(codes[:lo] * (was / scale))
                    codes[lo:hi] = e4m3(new / scale)
                    pool[name + "_scale"][page, h] = scale


def attention(q, pool, table, past, counts):
    """(out [B,N,Hq,D], m, l [B,Hq,N])."""
    b_, n_, hq, d = q.shape
    hkv, rows = pool["k"].shape[1:3]
    out = np.zeros(q.shape)
    m = np.full((b_, hq, n_), -np.inf)
    l = np.zeros((b_, hq, n_))
    for b in range(b_):
        if past[b] < 0:
            continue
        for i in range(counts[b]):
            where = []
            for r in range(past[b] + i + 1):
                page = page_of(table[b], len(pool["k"]), r // rows)
                if page is not None:
                    where.append((page, r % rows))
            if not where:
                continue
            pg, rw = np.array(where).T
            for h in range(hq):
                g = h // (hq // hkv)
                k = pool["k"][pg, g, rw] * pool["k_scale"][pg, g][:, None]
                v = pool["v"][pg, g, :, rw] * pool["v_scale"][pg, g][:, None]
                s = k.astype(np.float64) @ q[b, i, h].astype(np.float64) / np.sqrt(d)
                m[b, h, i] = s.max()
                p = np.exp(s - s.max())
                l[b, h, i] = p.sum()
                out[b, i, h] = p @ v / p.sum()
    return out, m, l
