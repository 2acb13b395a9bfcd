"""Attention over the paged 8-bit cache (longctx100m_amd/paged.py), each row by what it
sees: errors of the size that its roundings add up to, where tests/test_gpu_paged.py
allows their worst case.  Without a GPU: the comparison refuses a result with a key
left out, values of other rows, or probabilities or queries of fewer bits.

Roundings to nearest of a relative bound r are independent, of r / sqrt(3) rms at most.
With u = 2^-24, a row's probabilities p, its keys' scores s and values v, its output o:
  score    T = D products (3 D: fp32 queries in three parts) added one after another
           to partial sums that walk to s: at x of the way of variance
           x W^2 + x^2 s^2, W^2 the products' sum of squares, 1/2 and 1/3 of it on
           average.  dr^2 = u^2 T / 3 (W^2 / 2 + s^2 / 3)
  exp      its argument u |s - m| / sqrt(3), itself 2 u:  da^2 = u^2 (s - m)^2 / 3 + 4 u^2
  out      sum p^2 (dr^2 + da^2) |v - o|^2, as the row's sum goes along;
           h^2 / 3 sum p^2 |v|^2, h = 2^-8, where bf16 queries round their probabilities;
           half a step of the type, h^2 / 3 |o|^2 or u^2 / 3 |o|^2;
           n sums of products (3 n) added one after another, walking as the score does:
           u^2 n / 3 (sum p^2 |v|^2 / 2 + |o|^2 / 3);
           the scale 1 / sqrt(D), rounded once: u |sum p (s - mean s) v|;
           the parts' weights and the division, 4 u |o|.
  m + ln l sum p^2 (dr^2 + da^2) and the sum's n / 64 tiles and 32 values each,
           u^2 / 3 (n / 64 + 32); the scale u |mean s|, m's own rounding u |m|, 6 u.
A row may be off by 5 of these deviations (its largest key's score by 6), all rows of a
call together by 1.5."""

import numpy as np
import pytest

from oracle import paged as op
from tests.conftest import bf16_round
from tests.test_gpu_paged import ATTEND, _dtype, _i32, _pool, _table, _to_pages, _wide

U = 2.0 ** -24
H = 2.0 ** -8


def _inputs(case):
    hq, hkv, d, dtype, rows, past, n, counts, wider = case
    rng = np.random.default_rng(n * 17 + d)
    table, pages = _table(rng, past, n, rows, width=0)
    if wider:
        table = np.pad(table, ((0, 0), (0, wider)), constant_values=-7)
    pool = _pool(rng, pages, rows, hkv, d, spread=1)
    q = (1.5 * rng.standard_normal((len(past), n, hq, d))).astype(np.float32)
    return bf16_round(q) if dtype == "bf16" else q, pool, table, past, [n] * len(past) if counts is None else counts


def _rows_of(q, pool, table, past, counts):
    """For each token that is there and each KV head: (sequence, token, the group's query
    heads, their queries, the keys and the values that it sees), in 64 bits."""
    hkv, rows = pool["k"].shape[1:3]
    group = q.shape[2] // hkv
    for b, c in enumerate(counts):
        if past[b] < 0 or c == 0:
            continue
        at = np.arange(past[b] + c)
        page = table[b][at // rows]
        for g in range(hkv):
            k = pool["k"][page, g, at % rows] * pool["k_scale"][page, g][:, None]
            v = pool["v"][page, g, :, at % rows] * pool["v_scale"][page, g][:, None]
            heads = slice(g * group, (g + 1) * group)
            for i in range(c):
                n = past[b] + i + 1
                yield b, i, heads, q[b, i, heads].astype(np.float64), k[:n], v[:n]


def _expected(q, pool, table, past, counts, dtype):
    """(out, m, lse) and their deviations (of out: of a row's whole error vector), NaN in
    rows that there are not."""
    b_, n_, hq, d = q.shape
    parts, h = (1, H) if dtype == "bf16" else (3, U)
    out = np.full(q.shape, np.nan)
    m, lse, dev, dev_m, dev_lse, off_lse = (np.full((b_, n_, hq), np.nan) for _ in range(6))
    for b, i, at, x, k, v in _rows_of(q, pool, table, past, counts):
        n = len(k)
        s = x @ k.T / np.sqrt(d)
        top = s.max(1, keepdims=True)
        p = np.exp(s - top)
        l = p.sum(1, keepdims=True)
        p /= l
        o = p @ v
        w2 = (x * x) @ (k * k).T / d
        dr2 = U * U * parts * d / 3 * (w2 / 2 + s * s / 3)
        da2 = U * U * ((s - top) ** 2 / 3 + 4)
        v2, o2 = (v * v).sum(1), (o * o).sum(1)
        far = v2 - 2 * o @ v.T + o2[:, None]  # |v - o|^2
        pv = (p * p) @ v2
        mean = (p * s).sum(1, keepdims=True)
        scale = ((p * (s - mean)) @ v) ** 2
        var = (p * p * (dr2 + da2) * far).sum(1) + h * h / 3 * o2 + U * U * parts * n / 3 * (pv / 2 + o2 / 3)
        var += U * U * scale.sum(1) + 16 * U * U * o2
        if dtype == "bf16":
            var += H * H / 3 * pv
        out[b, i, at], m[b, i, at], lse[b, i, at] = o, top[:, 0], (top + np.log(l))[:, 0]
        dev[b, i, at] = np.sqrt(var)
        dev_m[b, i, at] = np.sqrt(dr2.max(1))
        dev_lse[b, i, at] = np.sqrt((p * p * (dr2 + da2)).sum(1) + U * U / 3 * (n / 64 + 32))
        off_lse[b, i, at] = U * (np.abs(mean) + np.abs(top) + 6)[:, 0]
    return out, m, lse, dev, dev_m, dev_lse, off_lse


def _faults(got, want):
    """What of (out [B, N, Hq, D], m, l [B, Hq, N]) is off by more than its roundings."""
    o, m, l = (np.asarray(x, np.float64) for x in got)
    m, l = m.transpose(0, 2, 1), l.transpose(0, 2, 1)
    eo, em, else_, dev, dev_m, dev_lse, off_lse = want
    there = ~np.isnan(em)
    bad = []
    if (o[~there] != 0).any() or (m[~there] != -np.inf).any() or (l[~there] != 0).any():
        bad.append("padding")
    if not np.isfinite(o).all() or not np.isfinite(m[there]).all() or not (l[there] > 0).all():
        return bad + ["not finite"]
    with np.errstate(invalid="ignore"):
        off = np.sqrt(((o - eo) ** 2).sum(-1))[there]
    # (a row over one key is exact, and has no deviation but that of its division)
    ratio = off / np.maximum(dev[there], 1e-300)
    if (ratio > 5).any():
        bad.append(f"out: {ratio.max():.2f} deviations of a row")
    if np.sqrt((ratio ** 2).mean()) > 1.5:
        bad.append(f"out: {np.sqrt((ratio ** 2).mean()):.2f} deviations of all rows")
    if (np.abs(m - em)[there] > (6 * dev_m + 2 * U * np.abs(em))[there]).any():
        bad.append("m")
    lse = m[there] + np.log(l[there])
    over = np.abs(lse - else_[there]) - (5 * dev_lse + off_lse)[there]
    if (over > 0).any():
        bad.append(f"lse by {over.max():.2e}")
    return bad


# ---------------------------------------------------------- the comparison --

def _computed(q, pool, table, past, counts, dtype, drop=None, shift=0, p_bits=None, q_bits=None):
    """The attention in fp32, as the kernels round it, with a mistake: the key `drop` of
    each row left out, values of `shift` rows on, or probabilities or queries of so many
    parts of bf16."""
    def cut(x, parts):
        got = np.zeros_like(x)
        for _ in range(parts):
            got += bf16_round(x - got)
        return got

    out = np.zeros(q.shape, np.float32)
    m = np.full((q.shape[0], q.shape[2], q.shape[1]), -np.inf)
    l = np.zeros(m.shape)
    for b, i, at, x, k, v in _rows_of(q, pool, table, past, counts):
        x = x.astype(np.float32)
        x = cut(x, q_bits) if q_bits else x
        keep = np.ones(len(k), bool)
        if drop is not None and len(k) > 1:
            keep[drop] = False
        s = (x @ k.T.astype(np.float32) * np.float32(q.shape[3] ** -0.5))[:, keep]
        top = s.max(1, keepdims=True)
        p = np.exp(s - top)
        m[b, at, i], l[b, at, i] = top[:, 0], p.sum(1, dtype=np.float64)
        if dtype == "bf16" or p_bits:
            p = cut(p, p_bits or 1)
        out[b, i, at] = (p @ np.roll(v, shift, 0)[keep].astype(np.float32)) / l[b, at, i][:, None].astype(np.float32)
    return bf16_round(out) if dtype == "bf16" else out, m.astype(np.float32), l.astype(np.float32)


SHORT = [c for c in ATTEND if max(c[5]) < 1000 and len(c[5]) < 10 and c[6] <= 20]
FP32 = [c for c in ATTEND if c[3] == "fp32" and c[6] <= 20]


@pytest.mark.parametrize("case", SHORT + [c for c in FP32 if c not in SHORT])
def test_the_comparison_accepts_roundings(case):
    args = *_inputs(case), case[3]
    assert _faults(_computed(*args), _expected(*args)) == []


@pytest.mark.parametrize("case", FP32)
def test_the_comparison_refuses_fewer_bits(case):
    args = *_inputs(case), "fp32"
    want = _expected(*args)
    assert _faults(_computed(*args, p_bits=1), want)
    assert _faults(_computed(*args, q_bits=1), want)
    assert _faults(_computed(*args, q_bits=2), want)
    # The third part of a probability is 2^-17 of it at most: 16 u, what a score's sum of
    # more than a few products is off by itself.
    if case[2] == 16:
        assert _faults(_computed(*args, p_bits=2), want)


@pytest.mark.parametrize("case", [c for c in ATTEND if c[5] in ([500], [777], [300], [3000], [313], [260])])
def test_the_comparison_refuses_a_lost_key(case):
    args = *_inputs(case), case[3]
    want = _expected(*args)
    for key in (0, -1):
        assert _faults(_computed(*args, drop=key), want), key


@pytest.mark.parametrize("case", [c for c in ATTEND if max(c[5]) >= 4000 and len(c[5]) == 1 and c[6] <= 3])
def test_the_comparison_refuses_other_rows_values(case):
    args = *_inputs(case), case[3]
    want = _expected(*args)
    assert _faults(_computed(*args), want) == []
    assert _faults(_computed(*args, shift=64), want)


# ------------------------------------------------------------- the kernels --

def _attend(gpu, q, p, table, past, counts, dtype):
    """The attention in outputs full of NaN, and a workspace of just the bytes that it is
    said to need, with others behind that stay as they are."""
    from longctx100m_amd import paged

    b, n, hq, _ = q.shape
    tq, tt = gpu.tensor(q).to(_dtype(gpu, dtype)).cuda(), _i32(gpu, table)
    nan = lambda *s, t=gpu.float32: gpu.full(s, float("nan"), dtype=t, device="cuda")  # noqa: E731
    need = paged.attention_workspace_bytes(tq, p, tt)
    room = gpu.full((need + 4096,), 0xff, dtype=gpu.uint8, device="cuda")  # (NaN, where it is read as floats)
    got = paged.attention(tq, p, tt, _i32(gpu, past), counts=_i32(gpu, counts), out=nan(*q.shape, t=tq.dtype),
                          m=nan(b, hq, n), l=nan(b, hq, n), workspace=room[:need])
    assert bool((room[need:] == 0xff).all()), "written behind the workspace"
    return [x.double().cpu().numpy() for x in got]


@pytest.mark.gpu
@pytest.mark.parametrize("case", ATTEND)
def test_attention_within_its_roundings(gpu, case):
    q, pool, table, past, counts = _inputs(case)
    dtype = case[3]
    want = _expected(q, pool, table, past, counts, dtype)
    p = _to_pages(gpu, pool)
    assert _faults(_attend(gpu, q, p, table, past, counts, dtype), want) == []
    if case[6] * case[0] // case[1] > 48 and dtype == "bf16":  # by tiles too
        assert _faults(_attend(gpu, q, p, _wide(table, q, pool), past, counts, dtype), want) == []
