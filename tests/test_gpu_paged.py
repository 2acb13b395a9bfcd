"""The paged 8-bit cache (longctx100m_amd/paged.py) against the float64 oracle.

Tolerances (u = 2^-24).  Codes: a value is rounded to e4m3, half a step of 2^-3
relative to it, 2^-10 of the scale at least; a rotated key is off by 7 u f (|x1| +
|x2|) before (tests/test_gpu_rotary.py); what is not rotated is exact to the code.
Attention: k and v are what codes and scales say, exactly.  A score is a sum of
T = D products of bf16 queries (3 D of the parts of fp32 ones), off by ds = (T +
4) u S, S the largest sum of |q k| / sqrt(D); its scaling and the exp's argument
add 4 u |s|.  A probability is then off by e = 2 (ds + 4 u max|s|) + 8 u
relatively, a sum of n of them by e + n u (3 n u for the parts).  An output is a mean of v with such weights: off by 2 (e + n u)
max|v|, for bf16 queries by another 2^-8 max|v| (each probability rounded to bf16),
and by half a step of its own type."""

import ctypes

import numpy as np
import pytest

from longctx100m_amd import _lib
from oracle import paged as op
from tests.conftest import bf16_round

U = 2.0 ** -24


def _i32(gpu, x):
    return None if x is None else gpu.tensor(x, dtype=gpu.int32).cuda()


def _dtype(gpu, dtype):
    return gpu.bfloat16 if dtype == "bf16" else gpu.float32


def _table(rng, past, n, rows, spare=3, width=0):
    """Pages in no order: (table, pages of the pool)."""
    need = [max(0, -(-(max(p, 0) + n) // rows)) for p in past]
    pages = sum(need) + spare
    order = rng.permutation(pages)
    table = np.full((len(past), max(max(need), width, 1)), -1, np.int64)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    return table, pages


def _pool(rng, pages, rows, hkv, d, spread=3):
    """A pool full of values, each page with scales of its own."""
    pool = {}
    for name, shape in (("k", (pages, hkv, rows, d)), ("v", (pages, hkv, d, rows))):
        x = rng.standard_normal(shape) * 2.0 ** rng.integers(-spread, spread + 1, (pages, hkv, 1, 1))
        s = np.array([[op.block_scale(np.abs(x[p, h]).max()) for h in range(hkv)] for p in range(pages)])
        pool[name], pool[name + "_scale"] = op.e4m3(x / s[..., None, None]), s
    return pool


def _to_pages(gpu, pool):
    from longctx100m_amd import paged
    codes = [gpu.tensor(pool[x], dtype=gpu.float32).to(gpu.float8_e4m3fn).cuda() for x in "kv"]
    return paged.Pages.of(*codes, *[gpu.tensor(pool[x + "_scale"], dtype=gpu.float32).cuda() for x in "kv"])


def _from_pages(p):
    return {"k": p.k.float().cpu().numpy().astype(np.float64), "v": p.v.float().cpu().numpy().astype(np.float64),
            "k_scale": p.k_scale.double().cpu().numpy(), "v_scale": p.v_scale.double().cpu().numpy()}


def _rows(gpu, rng, b, n, h, d, dtype, scale=1.0):
    x = (scale * rng.standard_normal((b, n, h, d))).astype(np.float32)
    x = bf16_round(x) if dtype == "bf16" else x
    return x, gpu.tensor(x).to(_dtype(gpu, dtype)).cuda()


# ------------------------------------------------------------------ append --

# hq, hkv, d, dtype, rows of a page, past of each sequence, tokens, counts
APPEND = [
    (8, 2, 64, "bf16", 16, [0], 1, None),
    (8, 2, 128, "bf16", 64, [5], 1, None),
    (32, 8, 128, "bf16", 64, [63, 64, 65, 127, 0], 1, [1, 1, 1, 0, 1]),
    (9, 3, 64, "fp32", 16, [0, 7, 16, 31, -1], 13, [13, 12, 1, 13, 13]),
    (4, 4, 128, "bf16", 128, [100, 1], 200, [200, 131]),
    (4, 2, 64, "bf16", 32, [3], 100, None),
    (2, 1, 16, "fp32", 16, [9, 0], 40, [40, 16]),
    (2, 2, 48, "bf16", 64, [1, 62], 70, None),
    (4, 2, 80, "bf16", 64, [13], 130, None),
    (2, 1, 112, "fp32", 128, [127, 5], 129, [129, 100]),
    (2, 1, 176, "bf16", 128, [2], 130, None),
    (2, 1, 240, "bf16", 32, [31], 33, None),
    (2, 1, 256, "fp32", 128, [0, 130], 131, None),
    (3, 3, 208, "bf16", 64, [60], 9, None),
]


def _check_codes(got, want, new, exact):
    """got, want: pools; new: for each (page, head, row) written the tolerance before
    rounding, by name."""
    for name in "kv":
        s, t = got[name + "_scale"], want[name + "_scale"]
        assert np.array_equal(s, t), name
        a = got[name] * s[..., None, None]
        b = want[name] * t[..., None, None]
        if exact or name == "v":
            assert np.array_equal(a, b, equal_nan=True), name
            continue
        off = np.abs(a - b)
        written = new > 0
        assert np.array_equal(a[~written], b[~written])
        # Codes may differ where rounding decides between two: by a step, if the value
        # before it was within its tolerance of the middle; a step is 2^-3 of a value's
        # binade, and 2^-9 of the scale at least.
        step = np.maximum(2.0 ** -3 * np.maximum(np.abs(a), np.abs(b)), 2.0 ** -9 * s[..., None, None])
        assert (off <= step * (1 + 1e-9))[written].all()
        assert (off[written] > 0).mean() <= 1e-3 + 2 / written.sum()


@pytest.mark.gpu
@pytest.mark.parametrize("turned", [None, "half", "interleaved"])
@pytest.mark.parametrize("case", APPEND)
def test_append(gpu, case, turned):
    from longctx100m_amd import paged, rotary

    hq, hkv, d, dtype, rows, past, n, counts = case
    rng = np.random.default_rng(d + n + rows)
    b = len(past)
    table, pages = _table(rng, past, n, rows)
    pool = _pool(rng, pages, rows, hkv, d)
    p = _to_pages(gpu, pool)
    # values that raise some pages' scales and not others'
    big = 2.0 ** rng.integers(-4, 6, (b, n, 1, 1))
    qkv = (rng.standard_normal((b, n, hq + 2 * hkv, d)) * big).astype(np.float32)
    qkv = bf16_round(qkv) if dtype == "bf16" else qkv
    t = gpu.tensor(qkv).to(_dtype(gpu, dtype)).cuda()
    tq, tk, tv = t.split((hq, hkv, hkv), 2)
    q, k, v = qkv[:, :, :hq], qkv[:, :, hq:hq + hkv], qkv[:, :, hq + hkv:]
    full = [n] * b if counts is None else counts
    kw = {}
    kk, r = k.astype(np.float64), None
    if turned:
        rd = d // 2 // 16 * 16 if turned == "interleaved" and d >= 32 else d
        r = rotary.Rotary(d, 10000.0, rotary_dim=rd, interleaved=turned == "interleaved")
        kk = np.stack([op.rotate(k[x], [past[x] + i for i in range(n)], r.inv_freq, 1.0, r.interleaved)
                       for x in range(b)])
        qo = gpu.full((b, n, hq, d), 7.0, dtype=t.dtype, device="cuda")
        kw = dict(rotary=r, q=tq, q_out=qo)
    got_q = paged.append(p, _i32(gpu, table), _i32(gpu, past), tk, tv, counts=_i32(gpu, counts), **kw)
    before = {x: y.copy() for x, y in pool.items()}
    op.append(pool, table, past, full, kk, v)
    got = _from_pages(p)
    # rows that were written, or rounded again
    new = np.zeros(pool["k"].shape)
    for x in range(b):
        if past[x] < 0 or full[x] == 0:
            continue
        for page in range(past[x] // rows, (past[x] + full[x] - 1) // rows + 1):
            hi = min(past[x] + full[x] - page * rows, rows)
            new[table[x][page], :, :hi] = 1
    _check_codes(got, pool, new, not turned)
    untouched = np.ones(pages, bool)
    untouched[[table[x][page] for x in range(b) if past[x] >= 0 and full[x] > 0
               for page in range(past[x] // rows, (past[x] + full[x] - 1) // rows + 1)]] = False
    for name in ("k", "v", "k_scale", "v_scale"):
        assert np.array_equal(got[name][untouched], before[name][untouched])
    if turned:
        assert got_q is qo
        want = np.stack([op.rotate(q[x], [past[x] + i for i in range(n)], r.inv_freq, 1.0, r.interleaved)
                         for x in range(b)])
        there = np.array([[past[x] >= 0 and i < full[x] for i in range(n)] for x in range(b)])
        g = got_q.float().cpu().numpy()
        assert (g[~there] == 7).all()
        most = np.abs(q).max(axis=-1, keepdims=True)
        tol = 14 * U * most + (2.0 ** -8 if dtype == "bf16" else U) * np.abs(want)
        assert (np.abs(g - want) <= tol)[there].all()
        # the same by the operator of its own
        at = gpu.tensor([[max(past[x], 0) + i for i in range(n)] for x in range(b)], dtype=gpu.int64).cuda()
        same = rotary.rotate(tq, at, r)
        where = gpu.tensor(there).cuda()
        assert gpu.equal(same[where], got_q[where])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_append_one_by_one(gpu, dtype):
    """Tokens one at a time: scales only rise, earlier rows follow; close to what one
    call of all gives."""
    from longctx100m_amd import paged

    rng = np.random.default_rng(8)
    hkv, d, rows, n = 2, 64, 16, 40
    table = np.array([[2, 0, 3]])
    pool = _pool(rng, 4, rows, hkv, d)
    x = _rows(gpu, rng, 1, n, hkv, d, dtype)[0] * (2.0 ** rng.integers(-12, 12, (1, n, hkv, 1))).astype(np.float32)
    y = _rows(gpu, rng, 1, n, hkv, d, dtype)[0] * (2.0 ** rng.integers(-12, 12, (1, n, hkv, 1))).astype(np.float32)
    tk, tv = (gpu.tensor(z).to(_dtype(gpu, dtype)).cuda() for z in (x, y))
    one, p = _to_pages(gpu, pool), _to_pages(gpu, pool)
    tt = _i32(gpu, table)
    paged.append(one, tt, _i32(gpu, [0]), tk, tv)
    for i in range(n):
        paged.append(p, tt, _i32(gpu, [i]), tk[:, i:i + 1], tv[:, i:i + 1])
        op.append(pool, table, [i], [1], x[:, i:i + 1], y[:, i:i + 1])
    got, whole = _from_pages(p), _from_pages(one)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert np.array_equal(got[name], pool[name]), name
    for name in "kv":
        assert np.array_equal(got[name + "_scale"], whole[name + "_scale"])
        # rounded twice: by another half step of the final scale's smallest at most
        off = np.abs(got[name] - whole[name])
        assert (off <= np.maximum(2.0 ** -9, 2.0 ** -3 * np.abs(whole[name]))).all()


@pytest.mark.gpu
def test_append_special_values(gpu):
    """Zeros, subnormals, the largest values, infinities and NaN."""
    from longctx100m_amd import paged

    d, rows = 16, 16
    inf, nan = float("inf"), float("nan")
    rng = np.random.default_rng(0)
    cases = [[0.0] * 4, [1e-45, 0.0, -3e-42, 1e-38], [3.4e38, -1.0, 1e30, 0.0], [inf, 1.0, -inf, nan], [nan] * 4,
             [448.0, -448.0, 449.0, 2.0 ** -9], [448.0, 2.0 ** -10, 1.5 * 2.0 ** -10, 2.0 ** -11], [-0.0, 1.0, 1.0625, 1.1875]]
    k = np.zeros((len(cases), 1, 1, d), np.float32)
    for i, c in enumerate(cases):
        k[i, 0, 0, :4] = c
    pool = _pool(rng, len(cases), rows, 1, d)
    p = _to_pages(gpu, pool)
    table = np.arange(len(cases))[:, None]
    tk = gpu.tensor(k).cuda()
    past = [0] * len(cases)
    paged.append(p, _i32(gpu, table), _i32(gpu, past), tk, tk)
    op.append(pool, table, past, [1] * len(cases), k, k)
    got = _from_pages(p)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert np.array_equal(got[name], pool[name], equal_nan=True), name


@pytest.mark.gpu
def test_append_bad_pages(gpu):
    """Entries that are no pages, and rows beyond the table: nothing is written
    there, everything else is."""
    from longctx100m_amd import paged, rotary

    rng = np.random.default_rng(11)
    hkv, d, rows, n = 2, 64, 16, 50
    pool = _pool(rng, 6, rows, hkv, d)
    table = np.array([[1, -1, 6, 0], [2 ** 31 - 1, 3, -2 ** 31, 4]])  # 64 rows each
    past, counts = [10, 40], [50, 50]
    k, tk = _rows(gpu, rng, 2, n, hkv, d, "bf16")
    v, tv = _rows(gpu, rng, 2, n, hkv, d, "bf16")
    p = _to_pages(gpu, pool)
    paged.append(p, _i32(gpu, table), _i32(gpu, past), tk, tv, counts=_i32(gpu, counts))
    op.append(pool, table, past, counts, k, v)
    got = _from_pages(p)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert np.array_equal(got[name], pool[name]), name
    # lengths that no table has, counts that no call has: clipped, or nothing
    for past, counts in (([2 ** 31 - 1, 2 ** 30], [50, 50]), ([-2 ** 31, -1], [50, 50]), ([0, 0], [0, -2 ** 31])):
        paged.append(p, _i32(gpu, table), _i32(gpu, past), tk, tv, counts=_i32(gpu, counts),
                     rotary=rotary.Rotary(d, 10000.0), q=tk)
        again = _from_pages(p)
        for name in ("k", "v", "k_scale", "v_scale"):
            assert np.array_equal(again[name], got[name]), name
    paged.append(p, _i32(gpu, table), _i32(gpu, [0, -1]), tk, tv, counts=_i32(gpu, [2 ** 31 - 1, 5]))  # 50
    op.append(pool, table, [0, -1], [50, 5], k, v)
    got = _from_pages(p)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert np.array_equal(got[name], pool[name]), name


# --------------------------------------------------------------- attention --

def _check_attention(got, want, q, pool, dtype):
    o, m, l = (x.float().cpu().numpy().astype(np.float64) for x in got)
    eo, em, el = want
    d, n = q.shape[3], int(np.prod(pool["k"].shape[::2]))  # (rows of the whole pool: no fewer than seen)
    parts = 1 if dtype == "bf16" else 3
    kmax = np.nan_to_num(np.abs(pool["k"] * pool["k_scale"][..., None, None])).max(axis=(0, 1, 2))
    vmax = np.nan_to_num(np.abs(pool["v"] * pool["v_scale"][..., None, None])).max()
    s = np.abs(q).astype(np.float64).max(axis=(0, 1, 2)) @ kmax / np.sqrt(d)
    ds = (parts * d + 4) * U * s
    e = 2 * (ds + 4 * U * s) + 8 * U + parts * n * U
    half = 2.0 ** -8 if dtype == "bf16" else U
    tol = (2 * e + (2.0 ** -8 if dtype == "bf16" else 0.0)) * vmax + half * np.abs(eo)
    there = np.isfinite(em)
    assert np.array_equal(np.isfinite(m), there)
    assert (l[~there] == 0).all()
    rows = there.transpose(0, 2, 1)
    assert (o[~rows] == 0).all()
    assert (np.abs(o - eo) <= tol)[rows].all(), (np.abs(o - eo)[rows].max(), tol[rows].min())
    assert (np.abs(m[there] - em[there]) <= ds + 4 * U * np.abs(em)[there]).all()
    assert (np.abs(l - el)[there] <= e * el[there]).all()


def _attend(gpu, q, p, table, past, counts, dtype, ws=True):
    from longctx100m_amd import paged

    b, n, hq, _ = q.shape
    tq = gpu.tensor(q).to(_dtype(gpu, dtype)).cuda()
    tt = _i32(gpu, table)
    nan = lambda *s, t=gpu.float32: gpu.full(s, float("nan"), dtype=t, device="cuda")  # noqa: E731
    work = nan(paged.attention_workspace_bytes(tq, p, tt) // 4 + 1) if ws else None
    return paged.attention(tq, p, tt, _i32(gpu, past), counts=_i32(gpu, counts), out=nan(*q.shape, t=tq.dtype),
                           m=nan(b, hq, n), l=nan(b, hq, n), workspace=work)


def _wide(table, q, pool):
    """The same table with entries of no page behind, so many that rows of a bf16 cache
    go by shared tiles instead of blocks of 16 (csrc/paged_attn.hip, make_plan)."""
    (b, n, hq, d), (_, hkv, rows, _) = q.shape, pool["k"].shape
    blocks = -(-n * hq // hkv // 16)
    width = (160 << 20) // (blocks * b * rows * hkv * d * 2) + 1
    return np.pad(table, ((0, 0), (0, max(0, width - table.shape[1]))), constant_values=-7)


# hq, hkv, d, dtype, rows of a page, past, tokens, counts, table wider by
ATTEND = [
    (8, 2, 64, "bf16", 16, [5], 1, None, 0),
    (8, 2, 128, "bf16", 64, [0], 1, None, 0),
    (32, 8, 128, "bf16", 64, [500], 1, None, 0),
    (32, 8, 128, "bf16", 128, [1200, 40, 0, 999, -1], 1, [1, 1, 1, 0, 1], 9),
    (9, 3, 64, "bf16", 16, [300, 7, 0, -1, 129], 16, [16, 3, 1, 16, 0], 4),
    (16, 16, 64, "bf16", 32, [260], 3, None, 0),
    (8, 2, 128, "bf16", 32, [63, 64, 65], 7, [7, 1, 7], 0),
    (8, 2, 128, "bf16", 64, [200], 64, None, 0),
    (4, 1, 128, "bf16", 16, [0, 33], 150, [150, 149], 2),
    (32, 1, 64, "bf16", 64, [450, 460], 5, None, 0),
    (6, 2, 64, "bf16", 64, [0, 1], 300, [299, 300], 0),
    (9, 3, 64, "fp32", 16, [512, 400], 13, [13, 12], 0),
    (8, 2, 128, "fp32", 64, [777], 17, None, 0),
    (4, 2, 128, "fp32", 32, [0, 10], 90, [90, 80], 0),
    (2, 1, 16, "fp32", 16, [33], 9, None, 0),
    (2, 1, 48, "bf16", 64, [100, 0], 6, None, 0),
    (4, 2, 80, "bf16", 32, [70], 33, None, 0),
    (4, 2, 112, "fp32", 128, [300], 5, None, 0),
    (4, 1, 256, "fp32", 16, [129, 64], 11, None, 0),
    (2, 2, 256, "bf16", 64, [313], 40, None, 0),
    (4, 2, 192, "bf16", 128, [90], 20, None, 0),
    # long ones: more than a run of 16 tiles a wave, several workgroups a sequence
    (4, 2, 128, "bf16", 128, [5000, 70, 2300], 2, None, 0),
    (4, 2, 64, "bf16", 128, [9100], 3, None, 0),
    (2, 1, 128, "fp32", 128, [3000], 2, None, 0),
    (8, 2, 128, "bf16", 16, [4200, 1], 1, None, 3),
    (4, 2, 64, "bf16", 32, [3000, 2999, 64], 1, None, 0),
    (2, 1, 64, "bf16", 64, [70000], 1, None, 0),
    (2, 1, 128, "bf16", 64, [70000], 2, None, 0),
    (8, 2, 128, "bf16", 64, [5000, 300], 70, [70, 33], 0),
    (2, 1, 64, "bf16", 128, [4000], 90, None, 0),
] + [(4, 2, 64, "bf16", 16, [(37 * i) % 91 - 1 for i in range(70)], 2, [i % 3 for i in range(70)], 0),
     (2, 1, 64, "bf16", 128, [(379 * i) % 2500 for i in range(67)], 1, None, 0),
     (2, 1, 128, "bf16", 64, [(379 * i) % 900 for i in range(70)], 40, None, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", ATTEND)
def test_attention(gpu, case):
    hq, hkv, d, dtype, rows, past, n, counts, wider = case
    rng = np.random.default_rng(n * 31 + d)
    table, pages = _table(rng, past, n, rows)
    if wider:
        table = np.pad(table, ((0, 0), (0, wider)), constant_values=-7)
    pool = _pool(rng, pages, rows, hkv, d, spread=1)
    q, _ = _rows(gpu, rng, len(past), n, hq, d, dtype, 1.5)
    full = [n] * len(past) if counts is None else counts
    want = op.attention(q, pool, table, past, full)
    p = _to_pages(gpu, pool)
    got = _attend(gpu, q, p, table, past, counts, dtype)
    _check_attention(got, want, q, pool, dtype)
    again = _attend(gpu, q, p, table, past, counts, dtype, ws=False)
    for x, y in zip(got, again):
        assert gpu.equal(x, y)
    if n * hq // hkv > 48 and dtype == "bf16":
        got = _attend(gpu, q, p, _wide(table, q, pool), past, counts, dtype)
        _check_attention(got, want, q, pool, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True], ids=["", "wide"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 6, 40, 130])
def test_rows_that_are_not_seen_do_not_matter(gpu, n, d, dtype, wide):
    """NaN codes and scales in pages and rows behind a token, also the next tokens'
    own, reach nobody; a seen one reaches its column alone."""
    rng = np.random.default_rng(5)
    hq, hkv, rows, past, counts = 8, 2, 32, [75, 0, 31], [n, max(n - 2, 1), n]
    table, pages = _table(rng, past, n, rows)
    pool = _pool(rng, pages, rows, hkv, d)
    q, _ = _rows(gpu, rng, 3, n, hq, d, dtype, 1.5)
    if wide:
        table = _wide(table, q, pool)
    want = op.attention(q, pool, table, past, counts)
    seen = np.zeros((pages, rows), bool)
    for b in range(3):
        for r in range(past[b] + counts[b]):
            seen[table[b][r // rows], r % rows] = True
    clean = {x: y.copy() for x, y in pool.items()}
    pool["k"].transpose(0, 2, 1, 3)[~seen] = np.nan
    pool["v"].transpose(0, 3, 1, 2)[~seen] = np.nan
    for name in ("k_scale", "v_scale"):
        pool[name][~seen.any(1)] = np.nan
    _check_attention(_attend(gpu, q, _to_pages(gpu, pool), table, past, counts, dtype), want, q, clean, dtype)
    # the last token's value: its own column of the last token, and nothing else
    last = past[0] + counts[0] - 1
    pool["v"][table[0][last // rows], 1, 3, last % rows] = np.nan
    got = _attend(gpu, q, _to_pages(gpu, pool), table, past, counts, dtype)
    nans = got[0].isnan().cpu().numpy()
    only = np.zeros(nans.shape, bool)
    only[0, counts[0] - 1, hq // 2:, 3] = True
    assert np.array_equal(nans, only)
    assert not got[1].isnan().any() and not got[2].isnan().any()
    # its key: the last token's rows, and nothing else
    pool["v"][table[0][last // rows], 1, 3, last % rows] = 1.0
    pool["k"][table[0][last // rows], 1, last % rows, 5] = np.nan
    got = _attend(gpu, q, _to_pages(gpu, pool), table, past, counts, dtype)
    only[0, counts[0] - 1, hq // 2:] = True
    assert np.array_equal(got[0].isnan().cpu().numpy(), only)


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True], ids=["", "wide"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [1, 20, 70])
def test_bad_pages_are_not_seen(gpu, n, dtype, wide):
    rng = np.random.default_rng(12)
    hq, hkv, d, rows = 8, 2, 128, 16
    past = [200, 90, 150]
    table, pages = _table(rng, past, n, rows)
    table[0, 3], table[0, 7], table[0, -1] = -1, pages, 2 ** 31 - 1
    table[1, :] = -5  # nothing there
    table[2, 0] = -2 ** 31
    pool = _pool(rng, pages, rows, hkv, d)
    q, _ = _rows(gpu, rng, 3, n, hq, d, dtype)
    want = op.attention(q, pool, table, past, [n] * 3)
    widen = (lambda t: _wide(t, q, pool)) if wide else (lambda t: t)
    _check_attention(_attend(gpu, q, _to_pages(gpu, pool), widen(table), past, None, dtype), want, q, pool, dtype)
    # a table that ends before the tokens
    short = widen(table[:, :9])
    want = op.attention(q, pool, short, past, [n] * 3)
    _check_attention(_attend(gpu, q, _to_pages(gpu, pool), short, past, None, dtype), want, q, pool, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("n,dtype", [(1, "bf16"), (3, "fp32"), (40, "bf16"), (40, "wide")])
def test_lengths_beyond_the_table(gpu, n, dtype):
    """A past of up to 2^31 - 1 rows sees what the table has."""
    rng = np.random.default_rng(19)
    pool = _pool(rng, 8, 16, 2, 64)
    table = np.array([[3, 5, 1, 7], [2, 0, 6, 4]])
    dtype, wide = ("bf16", True) if dtype == "wide" else (dtype, False)
    q, _ = _rows(gpu, rng, 2, n, 4, 64, dtype)
    want = op.attention(q, pool, table, [64, 64], [n] * 2)
    if wide:  # (more query heads' rows than kFewRows)
        table = _wide(table, q, pool)
    for past in ([2 ** 31 - 1, 2 ** 30], [64, 2 ** 30 + 5]):
        _check_attention(_attend(gpu, q, _to_pages(gpu, pool), table, past, None, dtype), want, q, pool, dtype)


@pytest.mark.gpu
def test_shared_pages(gpu):
    """Two sequences with the same prefix see the same pages."""
    rng = np.random.default_rng(13)
    pool = _pool(rng, 8, 16, 2, 64)
    table = np.array([[3, 5, 1], [3, 5, 6], [3, 3, 3]])
    past = [40, 44, 33]
    q, _ = _rows(gpu, rng, 3, 2, 4, 64, "bf16")
    want = op.attention(q, pool, table, past, [2] * 3)
    _check_attention(_attend(gpu, q, _to_pages(gpu, pool), table, past, None, "bf16"), want, q, pool, "bf16")


@pytest.mark.gpu
def test_extreme_scores(gpu):
    """Scores far apart, all the same, of the type's lowest values, and infinite."""
    rng = np.random.default_rng(14)
    hq, hkv, d, rows, past = 4, 2, 64, 16, [130]
    table, pages = _table(rng, past, 3, rows)
    pool = _pool(rng, pages, rows, hkv, d)
    for scale in (0.0, 40.0):
        q, _ = _rows(gpu, rng, 1, 3, hq, d, "bf16", scale)
        want = op.attention(q, pool, table, past, [3])
        _check_attention(_attend(gpu, q, _to_pages(gpu, pool), table, past, None, "bf16"), want, q, pool, "bf16")
    q = np.full((1, 3, hq, d), -3.3895e38, np.float32)  # the scores overflow
    got = _attend(gpu, bf16_round(q), _to_pages(gpu, pool), table, past, None, "bf16")
    assert got[0].isnan().any()  # as inf - inf would give
    q, _ = _rows(gpu, rng, 1, 3, hq, d, "bf16")
    q[0, 1, 2, 7] = np.nan
    got = _attend(gpu, q, _to_pages(gpu, pool), table, past, None, "bf16")
    nans = got[0].isnan().cpu().numpy()
    assert nans[0, 1, 2].all() and nans.sum() == d


@pytest.mark.gpu
def test_offsets_beyond_32_bits(gpu):
    """Pages whose bytes lie past 4 GiB of the pool, written and read."""
    from longctx100m_amd import paged

    rng = np.random.default_rng(15)
    hkv, d, rows, n = 8, 128, 128, 150
    count = (1 << 32) // (hkv * d * rows) + 40
    p = paged.Pages(count, rows, hkv, d)
    past = [0, 0]
    table = np.array([[count - 1, count - 3], [2, count - 17]])
    k, tk = _rows(gpu, rng, 2, n, hkv, d, "bf16")
    v, tv = _rows(gpu, rng, 2, n, hkv, d, "bf16")
    q, tq = _rows(gpu, rng, 2, n, 16, d, "bf16")
    tt = _i32(gpu, table)
    paged.append(p, tt, _i32(gpu, past), tk, tv)
    order = [count - 1, count - 3, 2, count - 17]
    small = {"k": np.zeros((4, hkv, rows, d)), "v": np.zeros((4, hkv, d, rows)), "k_scale": np.zeros((4, hkv)),
             "v_scale": np.zeros((4, hkv))}
    where = np.array([[0, 1], [2, 3]])
    op.append(small, where, past, [n] * 2, k, v)
    for name, t in (("k", p.k), ("v", p.v)):
        got = gpu.stack([t[i].view(gpu.uint8) for i in order]).view(gpu.float8_e4m3fn).float().cpu().numpy()
        assert np.array_equal(got, small[name])
    want = op.attention(q[:, -2:], small, where, [n - 2] * 2, [2] * 2)
    got = paged.attention(tq[:, -2:].contiguous(), p, tt, _i32(gpu, [n - 2] * 2))
    _check_attention(got, want, q[:, -2:], small, "bf16")
    rest = paged.attention(tq, p, tt, _i32(gpu, past))
    want = op.attention(q[:, [0, 77, 149]], small, where, past, [0] * 2)
    for i in (0, 77, 149):
        want = op.attention(q[:, i:i + 1], small, where, [i] * 2, [1] * 2)
        _check_attention([rest[0][:, i:i + 1], rest[1][..., i:i + 1], rest[2][..., i:i + 1]], want, q[:, i:i + 1],
                         small, "bf16")


@pytest.mark.gpu
def test_strides_and_alignment_of_the_append(gpu):
    """Rows that no vector fits, heads outside tokens, one row for all: the same codes."""
    from longctx100m_amd import paged, rotary

    rng = np.random.default_rng(16)
    hq, hkv, d, rows, n, past = 4, 2, 64, 16, 21, [7, 30]
    table, pages = _table(rng, past, n, rows)
    pool = _pool(rng, pages, rows, hkv, d)
    r = rotary.Rotary(d, 10000.0)
    for dtype in ("bf16", "fp32"):
        q, tq = _rows(gpu, rng, 2, n, hq, d, dtype)
        k, tk = _rows(gpu, rng, 2, n, hkv, d, dtype)
        v, tv = _rows(gpu, rng, 2, n, hkv, d, dtype)

        def run(q, k, v, **kw):
            p = _to_pages(gpu, pool)
            out = paged.append(p, _i32(gpu, table), _i32(gpu, past), k, v, rotary=r, q=q, **kw)
            return out, p.k.view(gpu.uint8), p.v.view(gpu.uint8), p.k_scale, p.v_scale

        want = run(tq, tk, tv)

        def odd(t):
            b, n, h, d = t.shape
            o = gpu.zeros(b * n * h * (d + 1) + 1, dtype=t.dtype, device="cuda")[1:].view(b, n, h, d + 1)[..., :d]
            return o.copy_(t)

        heads = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
        for f in (odd, heads):
            for x, y in zip(run(f(tq), f(tk), f(tv)), want):
                assert gpu.equal(x, y)
        same = tq.clone()
        got = run(same, tk, tv, q_out=same)
        assert got[0] is same
        for x, y in zip(got, want):
            assert gpu.equal(x, y)
        one = tk[:, :1].expand(2, n, hkv, d)
        for x, y in zip(run(tq, one, one), run(tq, one.contiguous(), one.contiguous())):
            assert gpu.equal(x, y)


@pytest.mark.gpu
def test_refusals(gpu):
    from longctx100m_amd import paged, rotary

    p = paged.Pages(6, 16, 2, 64)
    k = gpu.zeros(2, 3, 2, 64, device="cuda")
    q = gpu.zeros(2, 3, 4, 64, device="cuda")
    t, past = _i32(gpu, [[0, 1], [2, 3]]), _i32(gpu, [0, 0])
    r = rotary.Rotary(64, 10000.0)
    ok = dict(pages=p, table=t, past=past, k=k, v=k.clone(), counts=None, rotary=r, q=q, q_out=None)
    paged.append(**ok)
    for kw in (dict(k=k.half()), dict(k=k[..., :32]), dict(v=k[:1]), dict(v=k.bfloat16()), dict(q=q.bfloat16()),
               dict(q=q[:, :2]), dict(k=k.cpu()), dict(table=t.long()), dict(table=t[:1]), dict(table=t.t()),
               dict(table=t[0]), dict(past=past.long()), dict(past=past[:1]), dict(past=past.cpu()),
               dict(counts=past.float()), dict(counts=past[:1]), dict(rotary=None),
               dict(rotary=rotary.Rotary(128, 10000.0)), dict(q=None, q_out=q), dict(q_out=q.bfloat16()),
               dict(q_out=q[..., :32]), dict(k=gpu.zeros(2, 3, 2, 128, device="cuda")[..., ::2]),
               dict(q=gpu.zeros(2, 3, 3, 64, device="cuda")), dict(k=k[0])):
        with pytest.raises((ValueError, TypeError)):
            paged.append(**dict(ok, **kw))
    with pytest.raises(_lib.LcError, match="rotary_dim"):
        paged.append(**dict(ok, rotary=rotary.Rotary(64, 10000.0, rotary_dim=8)))
    ok = dict(q=q, pages=p, table=t, past=past, counts=None)
    for kw in (dict(q=q.half()), dict(q=q[:, ::2]), dict(q=q[..., :32]), dict(q=q.cpu()), dict(table=t.long()),
               dict(table=t[:1]), dict(past=past.long()), dict(counts=past[:1]), dict(out=q.bfloat16()),
               dict(out=q), dict(m=gpu.zeros(2, 3, 4, device="cuda")), dict(l=gpu.zeros(2, 4, 2, device="cuda")),
               dict(q=gpu.zeros(2, 3, 3, 64, device="cuda")), dict(workspace=gpu.zeros(8))):
        with pytest.raises((ValueError, TypeError)):
            paged.attention(**dict(ok, **kw))
    with pytest.raises(_lib.LcError, match="workspace"):
        paged.attention(**ok, workspace=gpu.zeros(1, dtype=gpu.uint8, device="cuda"))
    # nothing to do
    assert paged.append(p, t[:0], past[:0], k[:0], k[:0]) is None
    assert paged.append(p, t, past, k[:, :0], k[:, :0]) is None
    out, m, l = paged.attention(q[:, :0], p, t, past)
    assert out.shape == (2, 0, 4, 64) and m.shape == (2, 4, 0)


@pytest.mark.gpu
def test_a_decode_loop_and_its_graph(gpu):
    """The operators together: a prompt in two chunks, then tokens, of three
    sequences, eager, on another stream, and captured and replayed, all the same;
    and as plain attention of what the pool then holds."""
    from longctx100m_amd import paged, rotary

    rng = np.random.default_rng(17)
    hq, hkv, d, rows, lens, steps = 8, 2, 128, 32, [50, 1, 33], 9
    r = rotary.Rotary(d, 500000.0)
    n = max(lens)
    table, pages = _table(rng, lens, steps, rows)
    tt = _i32(gpu, table)
    _, prompt = _rows(gpu, rng, 3, n, hq + 2 * hkv, d, "bf16")
    _, tokens = _rows(gpu, rng, 3, steps, hq + 2 * hkv, d, "bf16")

    def split(x):
        return x.split((hq, hkv, hkv), 2)

    def step(p, x, past, counts, q_out, out, m, l, ws):
        q, k, v = split(x)
        q = paged.append(p, tt, past, k, v, counts=counts, rotary=r, q=q, q_out=q_out)
        return paged.attention(q, p, tt, past, counts=counts, out=out, m=m, l=l, workspace=ws)

    def buffers(x):
        b, n = x.shape[:2]
        q_out = gpu.zeros(b, n, hq, d, dtype=x.dtype, device="cuda")
        p = paged.Pages(pages, rows, hkv, d)
        ws = gpu.empty(paged.attention_workspace_bytes(q_out, p, tt), dtype=gpu.uint8, device="cuda")
        return [q_out, gpu.zeros_like(q_out), gpu.zeros(b, hq, n, device="cuda"), gpu.zeros(b, hq, n, device="cuda"), ws]

    def run(how):
        p = paged.Pages(pages, rows, hkv, d)
        outs = []
        past = _i32(gpu, [0, 0, 0])
        for lo, hi in ((0, 20), (20, n)):
            x = prompt[:, lo:hi]
            counts = _i32(gpu, [min(max(e - lo, 0), hi - lo) for e in lens])
            outs.append([t.clone() for t in step(p, x, past, counts, *buffers(x))])
            past += counts
        x = tokens[:, :1].clone()
        bufs = buffers(x)
        if how == "graph":
            g = gpu.cuda.CUDAGraph()
            gpu.cuda.synchronize()
            with gpu.cuda.graph(g):
                step(p, x, past, None, *bufs)
        for i in range(steps):
            x.copy_(tokens[:, i:i + 1])
            if how == "graph":
                g.replay()
                gpu.cuda.synchronize()
            else:
                step(p, x, past, None, *bufs)
            outs.append([t.clone() for t in bufs[1:4]])
            past += 1
        return outs, p

    outs, p = run("eager")
    s = gpu.cuda.Stream()
    s.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(s):
        other, p2 = run("stream")
    s.synchronize()
    captured, p3 = run("graph")
    for a, b, c in zip(outs, other, captured):
        for x, y, z in zip(a, b, c):
            assert gpu.equal(x, y) and gpu.equal(x, z)
    for a, b, c in zip(p._ptrs and (p.k, p.v, p.k_scale, p.v_scale), (p2.k, p2.v, p2.k_scale, p2.v_scale),
                       (p3.k, p3.v, p3.k_scale, p3.v_scale)):
        assert gpu.equal(a.view(gpu.uint8), b.view(gpu.uint8)) and gpu.equal(a.view(gpu.uint8), c.view(gpu.uint8))
    pool = _from_pages(p)
    at = [e + steps - 1 for e in lens]
    q = rotary.rotate(split(tokens[:, -1:])[0], gpu.tensor(at, dtype=gpu.int64).cuda()[:, None], r)
    want = op.attention(q.float().cpu().numpy(), pool, table, at, [1] * 3)
    _check_attention(outs[-1], want, q.float().cpu().numpy(), pool, "bf16")


@pytest.mark.gpu
def test_calls_that_overlap(gpu):
    """Two streams with a workspace each."""
    from longctx100m_amd import paged

    rng = np.random.default_rng(18)
    hq, hkv, d, rows, past = 8, 2, 64, 64, [3000, 20]
    table, pages = _table(rng, past, 2, rows)
    p = _to_pages(gpu, _pool(rng, pages, rows, hkv, d))
    q = [_rows(gpu, rng, 2, 2, hq, d, "bf16")[1] for _ in range(2)]
    tt, tp = _i32(gpu, table), _i32(gpu, past)
    want = [paged.attention(x, p, tt, tp) for x in q]
    streams = [gpu.cuda.Stream(), gpu.cuda.Stream()]
    gpu.cuda.synchronize()
    got = []
    for _ in range(5):
        for x, s in zip(q, streams):
            with gpu.cuda.stream(s):
                got.append(paged.attention(x, p, tt, tp))
    gpu.cuda.synchronize()
    for i, g in enumerate(got):
        for x, y in zip(g, want[i % 2]):
            assert gpu.equal(x, y)


def test_the_workspace_holds_what_the_query_says(monkeypatch):
    lib = _lib.load()
    c = _lib.Paged(1, 1, 32, 8, 128, 1, 4096, 64, 4096, 0)
    need = lib.lc_paged_attn_workspace_bytes(ctypes.byref(c))
    assert 0 < need < 1 << 26


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True], ids=["", "wide"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [64, 128])
@pytest.mark.parametrize("n", [1, 50, 140])
def test_pages_of_whole_tiles(gpu, n, rows, d, wide):
    """Pages that hold one or two 64-key tiles: missing ones in the middle and at the
    end, NaN and NaN scales wherever nobody looks, a NaN that some tokens see."""
    rng = np.random.default_rng(n + rows)
    hq, hkv, past, counts = 8, 2, [5 * rows + 3, 0, 2 * rows - 1], [n, max(n - 3, 1), n]
    table, pages = _table(rng, past, n, rows)
    table[0, 1], table[0, 4], table[2, 0] = -1, pages + 5, -3
    pool = _pool(rng, pages, rows, hkv, d)
    q, _ = _rows(gpu, rng, 3, n, hq, d, "bf16", 1.5)
    if wide:
        table = _wide(table, q, pool)
    want = op.attention(q, pool, table, past, counts)
    seen = np.zeros((pages, rows), bool)
    for b in range(3):
        for r in range(past[b] + counts[b]):
            if 0 <= table[b][r // rows] < pages:
                seen[table[b][r // rows], r % rows] = True
    clean = {x: y.copy() for x, y in pool.items()}
    pool["k"].transpose(0, 2, 1, 3)[~seen] = np.nan
    pool["v"].transpose(0, 3, 1, 2)[~seen] = np.nan
    for name in ("k_scale", "v_scale"):
        pool[name][~seen.any(1)] = np.nan
    _check_attention(_attend(gpu, q, _to_pages(gpu, pool), table, past, counts, "bf16"), want, q, clean, "bf16")
    # one token in the middle of the new ones, and one that all see
    for row, first in ((past[0] + n // 2, n // 2), (2 * rows + 5, 0)):
        at = table[0][row // rows], 1, 3, row % rows
        was, pool["v"][at] = pool["v"][at], np.nan
        got = _attend(gpu, q, _to_pages(gpu, pool), table, past, counts, "bf16")
        only = np.zeros(got[0].shape, bool)
        only[0, first:, hq // 2:, 3] = True
        assert np.array_equal(got[0].isnan().cpu().numpy(), only)
        pool["v"][at] = was
    # a table that ends inside the new tokens' rows, or before them
    short = table[:, :max(2, (past[0] + n // 2) // rows)]
    want = op.attention(q, clean, short, past, counts)
    _check_attention(_attend(gpu, q, _to_pages(gpu, pool), short, past, counts, "bf16"), want, q, clean, "bf16")
