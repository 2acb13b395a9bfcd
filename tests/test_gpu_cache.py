"""The KV-cache operators (longctx100m_amd/cache.py) against the float64 oracle.

Tolerances (u = 2^-24): a score is a sum of D exact or once-rounded products,
off by at most ds = (D + 4) u S, S the largest sum of |q k| / sqrt(D); its
scaling and the exp's argument add 4 u |s|.  A probability is then off by
e = 2 (ds + 4 u max|s|) + 8 u relatively (score and maximum), a sum of n of
them by e + n u.  An output is a mean of v with such weights: off by
2 (e + n u) max|v|, on the bf16 matrix cores by another 2^-8 max|v| (each
probability rounded to bf16, half a step of 2^-7), and by half a step of its
own type."""

import ctypes

import numpy as np
import pytest

from longctx100m_amd import _lib
from oracle import cache as oc
from tests.conftest import bf16_round

U = 2.0 ** -24


def _tree(rng, b, n, pad=0):
    """Random trees, several roots at times; the last ``pad`` nodes are padding."""
    p = [[-1] + [int(rng.integers(max(-1, i - 6), i)) for i in range(1, n)] for _ in range(b)]
    for row in p:
        for i in range(n - pad, n):
            row[i] = -2
    return p


def _data(rng, b, n, c, hq, hkv, d, dtype, scale=1.0):
    rnd = bf16_round if dtype == "bf16" else lambda x: np.asarray(x, np.float32)
    q = rnd(scale * rng.standard_normal((b, n, hq, d), dtype=np.float32))
    k = rnd(rng.standard_normal((b, c, hkv, d), dtype=np.float32))
    v = rnd(rng.standard_normal((b, c, hkv, d), dtype=np.float32))
    return q, k, v


def _to(gpu, x, dtype, layout="rows"):
    t = gpu.tensor(x).to(gpu.bfloat16 if dtype == "bf16" else gpu.float32).cuda()
    if layout == "heads":  # [B, H, C, D] in memory
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "slice":  # rows and heads of a larger cache
        b, c, h, d = t.shape
        big = gpu.full((b + 1, c + 3, h + 2, d), float("nan"), dtype=t.dtype, device="cuda")
        big[1:, 2:2 + c, 1:1 + h] = t
        return big[1:, 2:2 + c, 1:1 + h]
    if layout == "rows_first":  # [C, B, H, D] in memory
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    return t


def _i32(gpu, x):
    return None if x is None else gpu.tensor(x, dtype=gpu.int32).cuda()


def _nan(gpu, *shape, dtype=None):
    return gpu.full(shape, float("nan"), dtype=dtype or gpu.float32, device="cuda")


def _bounds(q, k, d, n):
    s = np.abs(q).astype(np.float64).max(axis=(0, 1, 2)) @ np.abs(k).astype(np.float64).max(axis=(0, 1, 2))
    s /= np.sqrt(d)
    ds = (d + 4) * U * s
    return ds, 2 * (ds + 4 * U * s) + 8 * U + n * U


def _check_attention(got, want, q, k, v, dtype, mfma):
    o, m, l = (x.float().cpu().numpy().astype(np.float64) for x in got)
    eo, em, el = want
    d = q.shape[3]
    kk, vv = np.nan_to_num(k, posinf=0, neginf=0), np.nan_to_num(v, posinf=0, neginf=0)
    ds, e = _bounds(q, kk, d, k.shape[1])
    half = 2.0 ** -8 if dtype == "bf16" else U
    tol = (2 * e + (2.0 ** -8 if mfma else 0.0)) * np.abs(vv).max() + half * np.abs(eo)
    there = np.isfinite(em)
    assert np.array_equal(np.isfinite(m), there)
    assert (l[~there] == 0).all()
    rows = there.transpose(0, 2, 1)
    assert (o[~rows] == 0).all()
    assert (np.abs(o - eo) <= tol)[rows].all(), np.abs(o - eo)[rows].max()
    assert (np.abs(m - em)[there] <= ds + 4 * U * np.abs(em)[there]).all()
    assert (np.abs(l - el)[there] <= e * el[there]).all()


def _run(gpu, q, k, v, past, parents, dtype, layout="rows", precise=False, ws="nan"):
    from longctx100m_amd import cache as kv

    b, n, hq, _ = q.shape
    tq, tk, tv = _to(gpu, q, dtype), _to(gpu, k, dtype, layout), _to(gpu, v, dtype, layout)
    out = _nan(gpu, *q.shape, dtype=tq.dtype)
    m, l = _nan(gpu, b, hq, n), _nan(gpu, b, hq, n)
    need = kv.tree_attention_workspace_bytes(tq, tk, precise)
    work = _nan(gpu, need // 4) if ws == "nan" else None
    return kv.tree_attention(tq, tk, tv, _i32(gpu, past), _i32(gpu, parents), out=out, m=m, l=l,
                             workspace=work, precise=precise)


# hq, hkv, d, dtype, past of each sequence, tokens, padding, capacity beyond the longest, layout
ATTENTION = [
    (8, 2, 64, "bf16", [5], 1, 0, 0, "rows"),               # one token, a handful of keys
    (8, 2, 128, "bf16", [0], 7, 0, 0, "rows"),              # nothing before the tree
    (4, 4, 128, "bf16", [63, 64, 65], 4, 1, 9, "rows"),     # tile edges
    (32, 8, 128, "bf16", [500], 8, 0, 0, "rows"),
    (9, 3, 64, "bf16", [300, 7, 0, -1, 129], 16, 3, 70, "heads"),  # ragged, a slot without a sequence
    (32, 8, 128, "bf16", [2111, 40], 26, 0, 0, "slice"),    # 104 rows per KV head
    (8, 2, 128, "bf16", [1200], 64, 5, 33, "heads"),        # 256 rows per KV head
    (4, 1, 128, "bf16", [777], 256, 0, 0, "rows"),          # the largest tree, 1,024 rows
    (32, 1, 64, "bf16", [450, 460], 5, 0, 1, "rows"),       # all heads share one KV head
    (6, 2, 64, "bf16", [1000, 1], 70, 2, 0, "rows_first"),
    (8, 2, 128, "bf16", [90, 1000], 6, 0, -4, "rows"),      # the longest has no room for its last nodes
    (4, 2, 128, "bf16", [4001, 3, 2000, 64, 0, 900, 1, 17], 9, 2, 0, "rows"),
    (16, 16, 64, "bf16", [260], 3, 0, 0, "rows"),
    (9, 3, 64, "fp32", [512, 400], 13, 2, 0, "heads"),
    (8, 2, 128, "fp32", [1000], 17, 0, 5, "rows"),
    (2, 1, 16, "fp32", [33], 9, 0, 0, "slice"),
    (2, 1, 48, "bf16", [100, 0], 6, 1, 0, "rows"),
    (4, 2, 80, "fp32", [70], 33, 0, 0, "rows"),
    (4, 2, 112, "bf16", [300], 5, 0, 0, "heads"),
    (4, 1, 256, "fp32", [129, 64], 11, 0, 0, "rows"),
    (2, 2, 256, "bf16", [513], 20, 3, 0, "rows"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
@pytest.mark.parametrize("case", ATTENTION)
def test_tree_attention(gpu, case, tree):
    hq, hkv, d, dtype, past, n, pad, extra, layout = case
    rng = np.random.default_rng(n * 31 + d)
    b, c = len(past), max(past) + n + extra
    q, k, v = _data(rng, b, n, c, hq, hkv, d, dtype, 1.5)
    parents = _tree(rng, b, n, pad) if tree else None
    want = oc.tree_attention(q, k, v, past, parents)
    got = _run(gpu, q, k, v, past, parents, dtype, layout)
    _check_attention(got, want, q, k, v, dtype, dtype == "bf16")
    if dtype == "bf16":
        got = _run(gpu, q, k, v, past, parents, dtype, layout, precise=True, ws=None)
        _check_attention(got, want, q, k, v, dtype, False)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,dtype", [(32, 8, 128, "bf16"), (9, 3, 64, "bf16"),
                                            (4, 2, 64, "fp32")])
def test_what_is_not_seen_does_not_matter(gpu, hq, hkv, d, dtype):
    """NaN and infinities in rows behind the tokens, in padded nodes and in other
    branches reach nobody; a seen infinite value reaches its column alone."""
    rng = np.random.default_rng(5)
    past, n = [130, 64], 12
    c = 190
    q, k, v = _data(rng, 2, n, c, hq, hkv, d, dtype)
    parents = _tree(rng, 2, n)
    for p in parents:
        p[4], p[5], p[6] = 0, -2, 5  # 5 and its child 6 are padding
        for i in range(7, n):
            p[i] = 0 if p[i] in (4, 5, 6) else p[i]
    want = oc.tree_attention(q, k, v, past, parents)
    for x in range(2):
        k[x, past[x] + n:] = np.nan
        v[x, past[x] + n:] = np.inf
        k[x, past[x] + 5], v[x, past[x] + 5] = np.inf, np.nan
        k[x, past[x] + 6], v[x, past[x] + 6] = np.nan, -np.inf
        v[x, past[x] + 4, :, 3] = np.inf   # seen by node 4 alone
    o, m, l = _run(gpu, q, k, v, past, parents, dtype)
    eo = want[0].copy()
    col = o[:, 4, :, 3].float().cpu().numpy()
    assert (col == np.inf).all()
    o = o.clone()
    o[:, 4, :, 3] = 0
    eo[:, 4, :, 3] = 0
    _check_attention((o, m, l), (eo, want[1], want[2]), q, k, v, dtype, dtype == "bf16")
    # in the past, seen by all: its column becomes infinite, the others stay
    v[0, 100, 0, 7] = -np.inf
    o, _, _ = _run(gpu, q, k, v, past, parents, dtype)
    g = hq // hkv
    col = o[0, :, :g, 7].float().cpu().numpy()
    there = np.isfinite(want[1][0, :g]).T
    assert (col[there] == -np.inf).all() and (col[~there] == 0).all()
    o[0, :, :g, 7] = 0
    o[:, 4, :, 3] = 0
    eo[0, :, :g, 7] = 0
    _check_attention((o, m, l), (eo, want[1], want[2]), q, k, v, dtype, dtype == "bf16")


@pytest.mark.gpu
def test_odd_lengths_and_parents_on_the_device(gpu):
    """Lengths beyond the capacity, the type's extremes and wild parents stay in
    bounds: such tokens are not there."""
    rng = np.random.default_rng(6)
    big = 2 ** 31 - 1
    past, n, c = [200, big, -big - 1, 195, 190], 8, 200
    q, k, v = _data(rng, 5, n, c, 8, 2, 128, "bf16")
    parents = [[-1, 0, big, -big - 1, 4, 5, 7, 1] for _ in past]
    want = oc.tree_attention(q, k, v, past, parents)
    got = _run(gpu, q, k, v, past, parents, "bf16")
    _check_attention(got, want, q, k, v, "bf16", True)
    assert np.isfinite(want[1]).any(axis=(1, 2)).tolist() == [False, False, False, True, True]
    got = _run(gpu, q, k, v, past, None, "bf16")
    _check_attention(got, oc.tree_attention(q, k, v, past), q, k, v, "bf16", True)


@pytest.mark.gpu
def test_shared_cache_and_missing_statistics(gpu):
    """One cache for all sequences (stride 0), and m and l left out."""
    from longctx100m_amd import cache as kv

    rng = np.random.default_rng(7)
    q, k, v = _data(rng, 3, 1, 300, 8, 2, 128, "bf16")
    k[1:], v[1:] = k[:1], v[:1]
    past = [299, 100, 5]
    want = oc.tree_attention(q, k, v, past)
    tq, tk, tv = (_to(gpu, x, "bf16") for x in (q, k[:1], v[:1]))
    tk, tv = tk.expand(3, -1, -1, -1), tv.expand(3, -1, -1, -1)
    got = kv.tree_attention(tq, tk, tv, _i32(gpu, past))
    _check_attention(got, want, q, k, v, "bf16", True)
    lib = _lib.load()
    c = kv._describe(tk, 1, 8)
    need = lib.lc_cache_attn_workspace_bytes(c)
    ws = gpu.empty(need, dtype=gpu.uint8, device="cuda")
    out = gpu.zeros_like(tq)
    rc = lib.lc_cache_attn(c, _i32(gpu, past).data_ptr(), None, tq.data_ptr(), tk.data_ptr(),
                           tv.data_ptr(), out.data_ptr(), None, None, ws.data_ptr(), need,
                           gpu.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert gpu.equal(out, got[0])


@pytest.mark.gpu
def test_more_sequences_than_a_wave_has_lanes(gpu):
    rng = np.random.default_rng(8)
    past = [int(x) for x in rng.integers(0, 200, 150)]
    past[70] = -1
    q, k, v = _data(rng, 150, 2, 202, 2, 1, 64, "bf16")
    want = oc.tree_attention(q, k, v, past)
    _check_attention(_run(gpu, q, k, v, past, None, "bf16"), want, q, k, v, "bf16", True)


# As ATTENTION: batches of unequal lengths, and the row blocks of head_dim 64.
UNEQUAL = [
    (4, 2, 64, "bf16", [30] * 20 + [3000] + [0, -1, 7] * 6, 6, 1, 0, "rows"),
    (4, 2, 128, "bf16", [100] * 11 + [2500, 64], 9, 0, 2, "heads"),
    (8, 1, 128, "bf16", [65] * 69 + [2000, -1, 3], 4, 0, 0, "rows"),
    (2, 2, 32, "fp32", [20] * 63 + [900], 2, 0, 0, "rows"),
    (4, 1, 64, "bf16", [700, 90], 12, 0, 0, "rows"),     # 48 rows per KV head
    (4, 1, 64, "bf16", [1300], 16, 2, 0, "heads"),       # 64
    (8, 2, 128, "bf16", [1300, 0, 65], 9, 0, 0, "slice"),   # 36
    (8, 2, 128, "bf16", [700], 16, 1, 3, "heads"),       # 64
    (4, 1, 64, "bf16", [1300, 128], 17, 2, 0, "rows"),   # 68
    (3, 3, 64, "bf16", [640], 256, 7, 1, "rows"),
    (8, 2, 256, "fp32", [300, 65], 20, 2, 0, "rows"),    # fp32 products, more than 32 rows
    (8, 2, 112, "bf16", [200, 3], 30, 0, 0, "heads"),
    (4, 1, 16, "fp32", [129], 40, 0, 0, "rows"),
    (4, 1, 32, "bf16", [77, 64, 15], 64, 6, 0, "rows"),
    (12, 3, 128, "fp32", [1000, 0, 17, -1], 17, 1, 0, "slice"),
    (4, 2, 80, "fp32", [500, 480], 100, 0, 2, "rows"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", UNEQUAL)
def test_unequal_lengths_and_row_blocks(gpu, case):
    hq, hkv, d, dtype, past, n, pad, extra, layout = case
    rng = np.random.default_rng(n + d + len(past))
    q, k, v = _data(rng, len(past), n, max(past) + n + extra, hq, hkv, d, dtype)
    parents = _tree(rng, len(past), n, pad)
    want = oc.tree_attention(q, k, v, past, parents)
    got = _run(gpu, q, k, v, past, parents, dtype, layout)
    _check_attention(got, want, q, k, v, dtype, dtype == "bf16")


# hq, hkv, d, past of each sequence, tokens, padding, capacity, layout
LARGE = [
    (4, 1, 64, [900], 12, 0, 530_000, "rows"),
    (4, 1, 64, [900], 4, 1, 530_000, "rows"),
    (4, 1, 64, [900], 40, 0, 530_000, "heads"),
    (4, 1, 128, [900], 10, 2, 250_000, "rows"),                    # 40 rows per KV head
    (32, 8, 128, [2111], 26, 0, 16_000, "rows"),                   # 104
    (4, 1, 128, [0, 1, 63, 64, 65, 127, 128, 129, -1], 17, 3, 40_000, "rows"),
    (4, 2, 128, [1, 700], 64, 1, 40_000, "heads"),                 # 128
    (4, 2, 128, [777], 70, 4, 60_000, "rows"),                     # 140
    (4, 1, 128, [1200, 0, 65, 128, 40], 64, 5, 30_000, "heads"),   # 256
    (9, 3, 128, [2300, 64, 191], 85, 0, 10_000, "rows"),           # 255, three heads a KV head
    (4, 1, 128, [777, 1300], 256, 9, 32_000, "rows"),              # 1,024
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", LARGE)
def test_little_of_a_large_cache(gpu, case):
    """Short pasts in caches of a large capacity, whose other rows are NaN: the
    forms that read each row once."""
    from longctx100m_amd import cache as kv

    hq, hkv, d, past, n, pad, c, layout = case
    rng = np.random.default_rng(n + d)
    b, used = len(past), max(past) + n
    q, k, v = _data(rng, b, n, used, hq, hkv, d, "bf16")
    if layout == "heads":
        tk, tv = (_nan(gpu, b, hkv, c, d, dtype=gpu.bfloat16).transpose(1, 2) for _ in range(2))
    else:
        tk, tv = (_nan(gpu, b, c, hkv, d, dtype=gpu.bfloat16) for _ in range(2))
    tk[:, :used] = _to(gpu, k, "bf16")
    tv[:, :used] = _to(gpu, v, "bf16")
    parents = _tree(rng, b, n, pad)
    got = kv.tree_attention(_to(gpu, q, "bf16"), tk, tv, _i32(gpu, past), _i32(gpu, parents))
    _check_attention(got, oc.tree_attention(q, k, v, past, parents), q, k, v, "bf16", True)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(gpu):
    """Every operator on caches whose sequences, heads and rows lie gigabytes apart."""
    from longctx100m_amd import cache as kv

    rng = np.random.default_rng(42)
    b, c, hq, hkv, d, n, past = 2, 80, 4, 2, 64, 8, [72, 41]
    strides = (2 ** 32 + 64, 2 ** 22, 2 ** 31 + 128, 1)
    size = sum(s * (x - 1) for s, x in zip(strides, (b, c, hkv, d))) + 1
    q, k, v = _data(rng, b, n, c, hq, hkv, d, "bf16")
    big = [gpu.empty(size, dtype=gpu.bfloat16, device="cuda") for _ in range(2)]
    tk, tv = (x.as_strided((b, c, hkv, d), strides) for x in big)
    tk.copy_(_to(gpu, k, "bf16"))
    tv.copy_(_to(gpu, v, "bf16"))
    parents = _tree(rng, b, n)
    tq, tpast, tpar = _to(gpu, q, "bf16"), _i32(gpu, past), _i32(gpu, parents)
    got = kv.tree_attention(tq, tk, tv, tpast, tpar)
    _check_attention(got, oc.tree_attention(q, k, v, past, parents), q, k, v, "bf16", True)
    m, l = (x.cpu().numpy() for x in got[1:])
    for rows in (1, n):  # one token a sequence, and all of them
        w = kv.key_weights(tq[:, :rows].contiguous(), tk, tpast, got[1][:, :, :rows].contiguous(),
                           got[2][:, :, :rows].contiguous())
        want = oc.key_weights(q[:, :rows], k, past, m[:, :, :rows], l[:, :, :rows], None,
                              np.zeros((b, hkv, c), np.float32))
        _check_weights(w, want, q, k, m, n * hq)
    path = [[1, 3, 4, 7] + [-1] * 4, [0, 5] + [-1] * 6]
    lens = kv.commit(kv.Layers([tk], [tv]), tpast, _i32(gpu, path))
    ek, ev, en = oc.commit(k, v, past, path)
    assert gpu.equal(tk.cpu().float(), gpu.tensor(ek)) and lens.tolist() == en
    weights = rng.random((b, hkv, c), dtype=np.float32)
    _, _, gn = kv.evict(tk, tv, gpu.tensor(weights).cuda(), lens, 40, sinks=2, recent=6)
    ek, ev, _, _, fn = oc.evict(ek, ev, weights, en, 40, 2, 6, None, None, None)
    assert gn.tolist() == fn
    assert gpu.equal(tk.cpu().float(), gpu.tensor(ek)) and gpu.equal(tv.cpu().float(), gpu.tensor(ev))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_no_tokens(gpu, dtype):
    """Nothing to attend with; key weights pass the earlier ones on."""
    from longctx100m_amd import cache as kv

    rng = np.random.default_rng(43)
    q, k, v = _data(rng, 2, 0, 70, 4, 2, 64, dtype)
    tq, tk, past = _to(gpu, q, dtype), _to(gpu, k, dtype), _i32(gpu, [66, 3])
    out, m, l = kv.tree_attention(tq, tk, tk, past)
    assert out.shape == (2, 0, 4, 64) and m.shape == l.shape == (2, 4, 0)
    old = gpu.rand(2, 2, 70, device="cuda")
    hold = gpu.rand(2, 2, 70, device="cuda")
    got = kv.key_weights(tq, tk, past, m, l, old, out=hold.clone())
    for x, n in enumerate((66, 3)):
        assert gpu.equal(got[x, :, :n], old[x, :, :n])
        assert gpu.equal(got[x, :, n:], hold[x, :, n:])
    layers = kv.Layers([tk], [tk.clone()])
    lens = kv.commit(layers, past, gpu.zeros(2, 0, dtype=gpu.int32, device="cuda"))
    assert lens.tolist() == [66, 3]


@pytest.mark.gpu
@pytest.mark.parametrize("d,n,dtype", [(128, 3, "bf16"), (128, 40, "bf16"), (64, 20, "bf16"),
                                       (64, 4, "fp32")])
def test_lengths_beyond_the_capacity(gpu, d, n, dtype):
    """A past that counts more rows than there are: its tokens have no place, and
    every row is a past one."""
    from longctx100m_amd import cache as kv

    rng = np.random.default_rng(44)
    past, c = [2 ** 31 - 1, 90, 200, 199], 200
    q, k, v = _data(rng, 4, n, c, 4, 2, d, dtype)
    got = _run(gpu, q, k, v, past, None, dtype)
    want = oc.tree_attention(q, k, v, past)
    assert not np.isfinite(want[1][0]).any() and np.isfinite(want[1][3]).any()
    _check_attention(got, want, q, k, v, dtype, dtype == "bf16")
    old = rng.random((4, 2, c), dtype=np.float32)
    m, l = (x.cpu().numpy() for x in got[1:])
    w = kv.key_weights(_to(gpu, q, dtype), _to(gpu, k, dtype), _i32(gpu, past), *got[1:],
                       gpu.tensor(old).cuda())
    want = oc.key_weights(q, k, past, m, l, old, np.zeros_like(old))
    _check_weights(w, want, q, k, m, 4 * n)
    assert np.array_equal(w[0].cpu().numpy(), old[0])


# ------------------------------------------------------------- key weights --

WEIGHTS = [
    (8, 2, 64, "bf16", [5], 1, 0, 0, "rows"),
    (32, 8, 128, "bf16", [1000], 1, 0, 6, "rows"),
    (32, 8, 128, "bf16", [63, 64, 128, 127], 4, 1, 0, "heads"),
    (9, 3, 64, "bf16", [300, 7, 0, -1, 129], 16, 3, 70, "slice"),
    (8, 2, 128, "bf16", [700], 26, 2, 0, "rows_first"),
    (4, 1, 128, "bf16", [90], 256, 9, 0, "rows"),
    (8, 2, 128, "bf16", [90, 300], 33, 0, -4, "rows"),
    (3, 3, 64, "bf16", [31, 500], 64, 0, 0, "rows"),
    (9, 3, 64, "fp32", [512, 400], 13, 2, 0, "heads"),
    (8, 2, 128, "fp32", [200], 17, 0, 5, "rows"),
    (2, 1, 16, "fp32", [33], 9, 0, 0, "slice"),
    (4, 2, 80, "bf16", [70], 33, 0, 0, "rows"),
    (4, 1, 256, "fp32", [129, 64], 11, 0, 0, "rows"),
    (16, 1, 128, "bf16", [400, 1], 1, 0, 0, "rows"),          # all heads share one KV head
    (32, 1, 64, "bf16", [400, 64], 3, 0, 0, "rows"),
    (8, 1, 128, "bf16", [30] * 70 + [1500], 2, 0, 0, "rows"),  # one long sequence among many
    (8, 2, 128, "bf16", [150], 40, 3, 66000, "rows"),         # 160 rows, a large cache
    (8, 2, 64, "bf16", [300, 64], 33, 0, 33000, "heads"),
]


def _check_weights(got, want, q, k, m, n_rows):
    kk = np.nan_to_num(k, posinf=0, neginf=0)
    ds, e = _bounds(q, kk, q.shape[3], n_rows)
    fin = np.abs(m[np.isfinite(m)]).max() if np.isfinite(m).any() else 0.0
    e += 8 * U * (fin + 16)  # m log2(e) + log2(l) in fp32: values up to |m| and log2(l) < 16
    g = got.cpu().numpy().astype(np.float64)
    assert (np.abs(g - want) <= e * np.abs(want) + 1e-36).all(), np.abs(g - want).max()


def _weights_case(gpu, case, parents, rng):
    from longctx100m_amd import cache as kv

    hq, hkv, d, dtype, past, n, _, extra, layout = case
    b, c = len(past), max(past) + n + extra
    q, k, v = _data(rng, b, n, c, hq, hkv, d, dtype, 1.5)
    _, m, l = oc.tree_attention(q, k, v, past, parents)
    m, l = m.astype(np.float32), l.astype(np.float32)
    old = rng.random((b, hkv, c), dtype=np.float32)
    hold = rng.random((b, hkv, c), dtype=np.float32)
    args = (_to(gpu, q, dtype), _to(gpu, k, dtype, layout), _i32(gpu, past),
            gpu.tensor(m).cuda(), gpu.tensor(l).cuda())
    for given in (old, None):
        out = gpu.tensor(hold).cuda()
        w = None if given is None else gpu.tensor(given).cuda()
        got = kv.key_weights(*args, w, _i32(gpu, parents), out=out)
        assert got is out
        want = oc.key_weights(q, k, past, m, l, given, hold, parents)
        _check_weights(got, want, q, k, m, n * hq)
        for x in range(b):  # rows behind the tokens, and absent sequences, as they were
            end = 0 if past[x] < 0 else min(past[x] + n, c)
            assert np.array_equal(got[x, :, end:].cpu().numpy(), hold[x, :, end:])
    w = gpu.tensor(old).cuda()  # in place
    kv.key_weights(*args, w, _i32(gpu, parents), out=w)
    want = oc.key_weights(q, k, past, m, l, old, old, parents)
    _check_weights(w, want, q, k, m, n * hq)


@pytest.mark.gpu
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
@pytest.mark.parametrize("case", WEIGHTS)
def test_key_weights(gpu, case, tree):
    rng = np.random.default_rng(case[5] * 17 + case[2])
    parents = _tree(rng, len(case[4]), case[5], case[6]) if tree else None
    _weights_case(gpu, case, parents, rng)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    (8, 2, 128, "bf16", [0], 300, 0, 0, "rows"),            # a whole prompt
    (6, 3, 64, "bf16", [100, 0], 401, 0, 30, "heads"),
    (4, 2, 64, "fp32", [17, 0], 290, 0, 0, "rows"),
])
def test_key_weights_of_a_prompt(gpu, case):
    _weights_case(gpu, case, None, np.random.default_rng(11))


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype", [(128, "bf16"), (64, "bf16"), (64, "fp32")])
def test_key_weights_nan_stays_where_it_is(gpu, d, dtype):
    """A NaN key gives its own weight NaN; in rows nobody sees it gives nothing,
    and so does a query row without statistics."""
    from longctx100m_amd import cache as kv

    rng = np.random.default_rng(12)
    past, n, c = [130], 8, 150
    q, k, v = _data(rng, 1, n, c, 4, 2, d, dtype)
    parents = [[-1, 0, 0, -2, 1, 4, -1, 6]]
    _, m, l = oc.tree_attention(q, k, v, past, parents)
    m, l = m.astype(np.float32), l.astype(np.float32)
    l[0, 1, 5] = 0.0            # a row that gives nothing
    m[0, 2, 7] = -np.inf
    q[0, 3] = np.nan            # a padded token's query
    want = oc.key_weights(q, k, past, m, l, None, np.zeros((1, 2, c)), parents)
    k[0, 133] = np.inf          # the padded token's row
    k[0, 138:] = np.nan         # behind the tokens
    k[0, 40, 1] = np.nan        # a seen key of KV head 1
    got = kv.key_weights(_to(gpu, q, dtype), _to(gpu, k, dtype), _i32(gpu, past),
                         gpu.tensor(m).cuda(), gpu.tensor(l).cuda(), None, _i32(gpu, parents))
    assert np.isnan(got[0, 1, 40].item())
    got[0, 1, 40] = 0
    want[0, 1, 40] = 0
    assert got[0, :, 133].abs().max().item() == 0
    _check_weights(got, want, np.nan_to_num(q), k, m, n * 4)


# ---------------------------------------------------------------- eviction --

EVICT = [
    # lens, capacity, hkv, d, budget, sinks, recent, dtype, layout, earlier
    ([100], 100, 2, 64, 40, 4, 8, "bf16", "rows", 0),
    ([1], 5, 1, 16, 1, 0, 0, "fp32", "rows", 0),
    ([9, 10, 11, 0, -3, 40], 40, 3, 16, 10, 2, 3, "fp32", "heads", 0),
    ([300, 299, 20], 320, 2, 128, 300, 0, 300, "bf16", "slice", 0),
    ([300, 299, 20], 320, 2, 128, 299, 5, 0, "bf16", "rows_first", 150),
    ([5000, 4097, 4096], 5003, 2, 32, 4096, 4, 64, "bf16", "rows", 4000),
    ([9000], 9000, 1, 16, 1, 0, 1, "bf16", "heads", 0),
    ([9000, 8500], 9000, 2, 16, 8191, 1, 1, "fp32", "rows", 8190),
    ([20001], 20011, 3, 16, 5000, 16, 100, "bf16", "rows", 3),
    ([70000], 70000, 1, 16, 33000, 4, 1000, "bf16", "rows", 0),
    ([50], 64, 2, 256, 400, 4, 8, "fp32", "rows", 0),   # more room than rows
    ([600000], 600000, 1, 16, 250000, 4, 64, "bf16", "rows", 0),
    ([300000, 5, 270001], 300000, 1, 16, 269000, 0, 9, "bf16", "heads", 0),
]


def _evict_inputs(rng, case, ties):
    lens, c, hkv, d, budget, sinks, recent, dtype, layout, earlier = case
    b = len(lens)
    _, k, v = _data(rng, b, 1, c, hkv, hkv, d, dtype)
    w = np.exp(3 * rng.standard_normal((b, hkv, c))).astype(np.float32)
    if ties:
        w = rng.choice(np.array([0.0, -0.0, 1.0, 2.5, np.inf, np.nan, -1.0, 1e-42], np.float32),
                       (b, hkv, c))
    pos = rng.permuted(np.tile(np.arange(2 * c, dtype=np.int32), (b, hkv, 1)), axis=-1)[..., :c]
    kept = [min(earlier, max(n, 0)) for n in lens] if earlier else None
    ends = [max(n, 0) + earlier for n in lens] if earlier else None
    return k, v, w, pos, kept, ends


@pytest.mark.gpu
@pytest.mark.parametrize("ties", [False, True], ids=["distinct", "ties"])
@pytest.mark.parametrize("case", EVICT)
def test_evict(gpu, case, ties):
    from longctx100m_amd import cache as kv

    lens, c, hkv, d, budget, sinks, recent, dtype, layout, earlier = case
    rng = np.random.default_rng(budget + c)
    k, v, w, pos, kept, ends = _evict_inputs(rng, case, ties)
    p = pos if earlier else None
    ek, ev, ew, ep, en = oc.evict(k, v, w, lens, budget, sinks, recent, p, kept, ends)
    for in_place in (False, True):
        tk, tv = _to(gpu, k, dtype, layout), _to(gpu, v, dtype, layout)
        tw = gpu.tensor(w).cuda()
        tp = gpu.tensor(pos).cuda() if earlier else None
        out = dict(weights_out=tw, positions_out=tp) if in_place else {}
        if in_place and tp is None:
            out["positions_out"] = gpu.zeros(pos.shape, dtype=gpu.int32, device="cuda")
        gw, gp, gn = kv.evict(tk, tv, tw, _i32(gpu, lens), budget, sinks=sinks, recent=recent,
                              positions=tp, kept=_i32(gpu, kept), ends=_i32(gpu, ends), **out)
        assert gn.tolist() == en
        np.testing.assert_array_equal(tk.float().cpu().numpy(), ek)
        np.testing.assert_array_equal(tv.float().cpu().numpy(), ev)
        for x, n in enumerate(en):
            np.testing.assert_array_equal(gw[x, :, :n].cpu().numpy(), ew[x, :, :n])
            np.testing.assert_array_equal(gp[x, :, :n].cpu().numpy(), ep[x, :, :n])
            if in_place:  # behind the kept rows as it was
                np.testing.assert_array_equal(gw[x, :, n:].cpu().numpy(), w[x, :, n:])
            else:
                assert (gw[x, :, n:] == 0).all() and (gp[x, :, n:] == 0).all()
                np.testing.assert_array_equal(tw.cpu().numpy(), w)


@pytest.mark.gpu
@pytest.mark.parametrize("c", [70, 20000])
def test_evict_extremes(gpu, c):
    """Lengths and kept counts beyond the cache, infinities and NaN of both signs."""
    from longctx100m_amd import cache as kv

    rng = np.random.default_rng(45)
    lens, kept, ends = [2 ** 31 - 1, c, -5, c - 1], [c + 9, 2 ** 31 - 1, 4, -1], [c + 50, c, 0, 7]
    _, k, v = _data(rng, 4, 1, c, 2, 2, 16, "bf16")
    w = rng.choice(np.array([-np.inf, np.inf, np.nan, -np.nan, -0.0, 0.0, 3e38, -3e38, 1e-45, -1e-45],
                            np.float32), (4, 2, c))
    pos = rng.integers(0, c + 40, (4, 2, c)).astype(np.int32)
    budget, sinks, recent = c - 30, 5, 20
    want = oc.evict(k, v, w, lens, budget, sinks, recent, pos, kept, ends)
    tk, tv = _to(gpu, k, "bf16"), _to(gpu, v, "bf16")
    got = kv.evict(tk, tv, gpu.tensor(w).cuda(), _i32(gpu, lens), budget, sinks=sinks,
                   recent=recent, positions=gpu.tensor(pos).cuda(), kept=_i32(gpu, kept),
                   ends=_i32(gpu, ends))
    assert got[2].tolist() == want[4]
    np.testing.assert_array_equal(tk.float().cpu().numpy(), want[0])
    np.testing.assert_array_equal(tv.float().cpu().numpy(), want[1])
    for x, n in enumerate(want[4]):
        np.testing.assert_array_equal(got[0][x, :, :n].cpu().numpy(), want[2][x, :, :n])
        np.testing.assert_array_equal(got[1][x, :, :n].cpu().numpy(), want[3][x, :, :n])


@pytest.mark.gpu
def test_long_caches_in_a_graph(gpu):
    """Attention, weights, commit and an eviction of several launches, captured
    once and replayed with other tensors, lengths and trees, beside eager calls."""
    from longctx100m_amd import cache as kv

    rng = np.random.default_rng(47)
    b, c, n, hq, hkv, d, budget = 2, 18000, 8, 4, 2, 64, 9000

    def inputs(past):
        q, k, v = (_to(gpu, x, "bf16") for x in _data(rng, b, n, c, hq, hkv, d, "bf16"))
        w = gpu.tensor(rng.random((b, hkv, c), dtype=np.float32)).cuda()
        path = [[0, 3, -1, -1], [1, 2, 6, -1]]
        return [q, k, v, w, _i32(gpu, past), _i32(gpu, _tree(rng, b, n)), _i32(gpu, path)]

    def step(q, k, v, w, past, parents, path, ws):
        out, m, l = kv.tree_attention(q, k, v, past, parents, workspace=ws[0])
        kv.key_weights(q, k, past, m, l, w, parents, out=w)
        lens = kv.commit(kv.Layers([k], [v]), past, path)
        return (out, m, l, k, v, *kv.evict(k, v, w, lens, budget, sinks=4, recent=60, workspace=ws[1]))

    static = inputs([0, 0])
    ws = [gpu.empty(s, dtype=gpu.uint8, device="cuda") for s in
          (kv.tree_attention_workspace_bytes(static[0], static[1]), kv.evict_workspace_bytes(static[1]))]
    step(*[x.clone() for x in static], ws)
    gpu.cuda.synchronize()
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph):
        got = step(*static, ws)
    for past in ([17000, 3], [17992, 12000], [8995, -1], [400, 17999]):
        fresh = inputs(past)
        want = step(*[x.clone() for x in fresh], [w.clone() for w in ws])
        for x, y in zip(static, fresh):
            x.copy_(y)
        graph.replay()
        gpu.cuda.synchronize()
        for x, y in zip(got, want):
            assert gpu.equal(x, y), past


@pytest.mark.gpu
def test_other_operators_on_two_streams(gpu):
    """Weights, evictions and commits that overlap, each on tensors of its own."""
    from longctx100m_amd import cache as kv

    rng = np.random.default_rng(46)
    c, n = 20000, 8
    runs = []
    for _ in range(2):
        q, k, v = _data(rng, 1, n, c, 8, 2, 64, "bf16")
        runs.append((_to(gpu, q, "bf16"), _to(gpu, k, "bf16"), _to(gpu, v, "bf16")))

    def go(q, k, v):
        k, v = k.clone(), v.clone()
        past = _i32(gpu, [c - n])
        _, m, l = kv.tree_attention(q, k, v, past)
        w = kv.key_weights(q, k, past, m, l)
        lens = kv.commit(kv.Layers([k], [v]), past, _i32(gpu, [[1, 2, 5, -1]]))
        return (k, v, *kv.evict(k, v, w, lens, 12000, sinks=4, recent=30))

    alone = [go(*r) for r in runs]
    gpu.cuda.synchronize()
    streams = [gpu.cuda.Stream(), gpu.cuda.Stream()]
    outs = [[], []]
    for _ in range(5):
        for i in (0, 1):
            with gpu.cuda.stream(streams[i]):
                outs[i].append(go(*runs[i]))
    gpu.cuda.synchronize()
    for i in (0, 1):
        for got in outs[i]:
            assert all(gpu.equal(x, y) for x, y in zip(got, alone[i]))


# ------------------------------------------------------------------ commit --

@pytest.mark.gpu
@pytest.mark.parametrize("layers,hkv,d,dtype,past,n,extra,layout", [
    (1, 2, 64, "bf16", [5], 4, 0, "rows"),
    (3, 3, 128, "fp32", [0, 17, -1, 40], 20, 0, "heads"),
    (33, 1, 16, "bf16", [7, 3], 64, 2, "rows"),
    (2, 2, 256, "fp32", [30, 60, 2 ** 31 - 1], 9, 0, "slice"),
    (2, 2, 32, "bf16", [10], 200, 0, "rows_first"),
])
def test_commit(gpu, layers, hkv, d, dtype, past, n, extra, layout):
    from longctx100m_amd import cache as kv

    rng = np.random.default_rng(d + n)
    b, c = len(past), max(p for p in past if p < 1000) + n + extra
    paths = []
    for x in range(b):
        p = sorted(rng.choice(n, rng.integers(1, n + 1), replace=False).tolist())
        paths.append(p + [-1] * (n - len(p)))
    paths[0] = list(range(n))                  # all of a chain: nothing moves
    if b > 1:
        paths[1] = [n - 1] + [n - 2] * (n - 1)     # ends at the second entry: not ascending
    if b > 3:
        paths[3] = [0, 2, 3, 2 ** 31 - 1] + [n] * (n - 4)
    ks, vs, want = [], [], []
    for _ in range(layers):
        _, k, v = _data(rng, b, 1, c, hkv, hkv, d, dtype)
        want.append(oc.commit(k, v, past, paths))
        ks.append(_to(gpu, k, dtype, layout))
        vs.append(_to(gpu, v, dtype, layout))
    lens = kv.commit(kv.Layers(ks, vs), _i32(gpu, past), _i32(gpu, paths))
    for k, v, (ek, ev, en) in zip(ks, vs, want):
        np.testing.assert_array_equal(k.float().cpu().numpy(), ek)
        np.testing.assert_array_equal(v.float().cpu().numpy(), ev)
        assert lens.tolist() == en


# ---------------------------------------------------------------- together --

def _steps(gpu, rng, b, c, hq, hkv, d, steps):
    """Inputs of a run: queries, keys and values of each step's drafted tokens."""
    return [_data(rng, b, n, n, hq, hkv, d, "bf16") for n in steps]


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
def test_run_together(gpu, graph):
    """A bounded cache over several rounds of drafting: attend the tree, commit a
    path, accumulate the accepted tokens' weights, evict, against the oracle
    doing the same on the exact values.  As a captured graph the same launches
    replay with each round's lengths, trees and paths."""
    from longctx100m_amd import cache as kv

    rng = np.random.default_rng(21)
    b, c, hq, hkv, d, n, budget, sinks, recent = 3, 120, 8, 2, 128, 8, 40, 2, 12
    i32 = lambda x: gpu.tensor(x, dtype=gpu.int32).cuda()  # noqa: E731
    _, k, v = _data(rng, b, 1, c, hq, hkv, d, "bf16")
    lens, ends, kept = [60, 33, 0], [60, 33, 0], [0, 0, 0]
    w = rng.random((b, hkv, c), dtype=np.float32)
    pos = np.zeros((b, hkv, c), np.int32)
    s = dict(k=_to(gpu, k, "bf16"), v=_to(gpu, v, "bf16"), w=gpu.tensor(w).cuda(), pos=i32(pos),
             past=i32(lens), ends=i32(ends), kept=i32(kept), parents=i32([[-1] * n] * b),
             chain=i32([[-1] * n] * b), path=i32([[-1] * n] * b),
             q=gpu.zeros(b, n, hq, d, dtype=gpu.bfloat16, device="cuda"))
    layers = kv.Layers([s["k"]], [s["v"]])
    lens_out, kept_out = i32(lens), i32(kept)

    def step():
        o, m, l = kv.tree_attention(s["q"], s["k"], s["v"], s["past"], s["parents"])
        at = s["path"].clamp(min=0).long()
        new = kv.commit(layers, s["past"], s["path"], lens_out=lens_out)
        # the accepted tokens as a chain of their own, padded
        qa = s["q"].gather(1, at[:, :, None, None].expand(-1, -1, hq, d)).contiguous()
        ma, la = (t.gather(2, at[:, None].expand(-1, hq, -1)).contiguous() for t in (m, l))
        kv.key_weights(qa, s["k"], s["past"], ma, la, s["w"], s["chain"], out=s["w"])
        kv.evict(s["k"], s["v"], s["w"], new, budget, sinks=sinks, recent=recent,
                 positions=s["pos"], kept=s["kept"], ends=s["ends"], weights_out=s["w"],
                 positions_out=s["pos"], lens_out=kept_out)
        return o, m, l

    g = None
    if graph:
        save = {x: t.clone() for x, t in s.items()}
        side = gpu.cuda.Stream()
        side.wait_stream(gpu.cuda.current_stream())
        with gpu.cuda.stream(side):
            step()
        gpu.cuda.current_stream().wait_stream(side)
        g = gpu.cuda.CUDAGraph()
        with gpu.cuda.graph(g):
            outs = step()
        for x, t in s.items():
            t.copy_(save[x])
    for rnd in range(5):
        q, kn, vn = _data(rng, b, n, n, hq, hkv, d, "bf16", 1.5)
        parents = _tree(rng, b, n, rnd % 3)
        paths, chains = [], []
        for x in range(b):
            leaf = int(rng.integers(0, n - rnd % 3))
            p = [leaf]
            while parents[x][p[0]] >= 0:
                p.insert(0, parents[x][p[0]])
            paths.append(p + [-1] * (n - len(p)))
            chains.append([j - 1 if j < len(p) else -2 for j in range(n)])
        for x in range(b):
            k[x, lens[x]:lens[x] + n], v[x, lens[x]:lens[x] + n] = kn[x], vn[x]
        # the oracle's round
        eo, em, el = oc.tree_attention(q, k, v, lens, parents)
        k1, v1, new = oc.commit(k, v, lens, paths)
        at = np.maximum(paths, 0)
        qa = np.take_along_axis(q, at[:, :, None, None], 1)
        ma, la = (np.take_along_axis(t, at[:, None], 2) for t in (em, el))
        w1 = oc.key_weights(qa, k1, lens, ma, la, w, w, chains)
        # the device's
        s["k"].copy_(_to(gpu, k, "bf16"))
        s["v"].copy_(_to(gpu, v, "bf16"))
        ends = [e + len([p for p in row if p >= 0]) for e, row in zip(ends, paths)]
        for name, val in (("past", lens), ("parents", parents), ("path", paths),
                          ("chain", chains), ("ends", ends), ("kept", kept)):
            s[name].copy_(i32(val))
        s["q"].copy_(_to(gpu, q, "bf16"))
        pos_in = s["pos"].cpu().numpy()
        if graph:
            g.replay()
            got = outs
        else:
            got = step()
        gpu.cuda.synchronize()
        _check_attention(got, (eo, em, el), q, k, v, "bf16", True)
        assert lens_out.tolist() == new
        # the weights decide what goes: compare the eviction on the device's own
        k2, v2, _, _, kept = oc.evict(k1, v1, w1, new, budget, sinks, recent, pos_in, kept, ends)
        assert kept_out.tolist() == kept
        np.testing.assert_array_equal(s["k"].float().cpu().numpy(), k2)
        np.testing.assert_array_equal(s["v"].float().cpu().numpy(), v2)
        k, v, lens = k2, v2, kept
        w, pos = s["w"].cpu().numpy(), s["pos"].cpu().numpy()
        for x in range(b):  # positions are distinct and below the sequence's end
            for h in range(hkv):
                p = pos[x, h, :kept[x]]
                assert len(set(p.tolist())) == kept[x] and (p < ends[x]).all() and (p >= 0).all()


@pytest.mark.gpu
def test_two_streams_at_once(gpu):
    """Two calls that overlap, each with its own workspace, on streams of their own."""
    from longctx100m_amd import cache as kv

    rng = np.random.default_rng(31)
    args = []
    for past in ([3000, 10], [700, 2500]):
        q, k, v = _data(rng, 2, 8, 3100, 8, 2, 128, "bf16")
        args.append((_to(gpu, q, "bf16"), _to(gpu, k, "bf16"), _to(gpu, v, "bf16"),
                     _i32(gpu, past), _i32(gpu, _tree(rng, 2, 8))))
    alone = [kv.tree_attention(*a) for a in args]
    gpu.cuda.synchronize()
    streams = [gpu.cuda.Stream(), gpu.cuda.Stream()]
    outs = [[], []]
    for _ in range(10):
        for i in (0, 1):
            with gpu.cuda.stream(streams[i]):
                outs[i].append(kv.tree_attention(*args[i]))
    gpu.cuda.synchronize()
    for i in (0, 1):
        for got in outs[i]:
            assert all(gpu.equal(x, y) for x, y in zip(got, alone[i]))


@pytest.mark.gpu
def test_python_checks(gpu):
    from longctx100m_amd import cache as kv

    q = gpu.zeros(1, 2, 4, 64, device="cuda")
    k = gpu.zeros(1, 8, 2, 64, device="cuda")
    past = gpu.zeros(1, dtype=gpu.int32, device="cuda")
    ok = dict(out=None)
    for bad, kw in [((q.bfloat16(), k, k, past), ok), ((q, k, k[:, :4], past), ok),
                    ((q, k, k.transpose(1, 2).contiguous().transpose(1, 2), past), ok),
                    ((q, k, k, past.long()), ok), ((q, k, k, past.cpu()), ok),
                    ((q[:, :, :, :32], k, k, past), ok), ((q[..., ::2], k, k, past), ok),
                    ((q, k, k, past, gpu.zeros(1, 3, dtype=gpu.int32, device="cuda")), ok),
                    ((q, k, k, past), dict(out=gpu.zeros(1, 2, 4, 32, device="cuda"))),
                    ((q, k, k, past), dict(m=gpu.zeros(1, 2, 4, device="cuda"))),
                    ((q, k.half(), k.half(), past), ok)]:
        with pytest.raises(ValueError):
            kv.tree_attention(*bad, **kw)
    with pytest.raises(_lib.LcError, match="workspace"):
        kv.tree_attention(q, k, k, past, workspace=gpu.empty(16, dtype=gpu.uint8, device="cuda"))
    w = gpu.zeros(1, 2, 8, device="cuda")
    with pytest.raises(ValueError, match="budget"):
        kv.evict(k, k.clone(), w, past, 0)
    with pytest.raises(ValueError, match="positions"):
        kv.evict(k, k.clone(), w, past, 4, kept=past)
    with pytest.raises(ValueError, match="same shape"):
        kv.Layers([k, k.clone()], [k.clone(), k[:, :4]])
    with pytest.raises(ValueError, match="listed twice"):
        kv.Layers([k, k.clone()], [k.clone(), k])
    m = gpu.zeros(1, 4, 2, device="cuda")
    with pytest.raises(ValueError):
        kv.key_weights(q, k, past, m, m, gpu.zeros(1, 2, 9, device="cuda"))
