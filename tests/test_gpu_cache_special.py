"""Infinities and NaN in the caches of the KV-cache operators, in every form of
the kernels, against the float64 oracle (tolerances: test_gpu_cache.py)."""

import numpy as np
import pytest

from oracle import cache as oc
from tests.conftest import bf16_round
from tests.test_gpu_cache import _check_attention, _check_weights, _data, _i32, _nan, _to, _tree

pytestmark = pytest.mark.gpu


# hq, hkv, d, tokens, capacity, dtype: query rows of a KV head and the form that takes them
@pytest.mark.parametrize("hq,hkv,d,n,c,dtype", [
    (4, 2, 128, 8, 170, "bf16"),      # 16: in registers
    (4, 2, 128, 13, 170, "bf16"),     # 26: in LDS, one tile of 32
    (4, 2, 64, 20, 170, "bf16"),      # 40
    (4, 2, 128, 32, 170, "bf16"),     # 64, no filler
    (8, 2, 128, 50, 70000, "bf16"),   # 200
    (8, 2, 64, 64, 70000, "bf16"),    # 256
    (8, 2, 128, 64, 300, "bf16"),     # 256, streamed
    (4, 2, 64, 150, 300, "bf16"),     # 300
    (4, 2, 64, 20, 170, "fp32"),
])
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
def test_rows_that_give_nothing_give_no_nan(gpu, hq, hkv, d, n, c, dtype, tree):
    """An infinite key gives those rows that give nothing (padding, l not above 0,
    m = -inf) a NaN or infinite score, and every other row -inf: its weight is 0."""
    from longctx100m_amd import cache as kv

    rng = np.random.default_rng(n + d)
    past = [130]
    q, k, v = _data(rng, 1, n, past[0] + n, hq, hkv, d, dtype)
    q[..., 3] = -np.abs(q[..., 3]) - 1
    q = bf16_round(q) if dtype == "bf16" else q  # what the kernel is given
    parents = _tree(rng, 1, n, 3) if tree else None
    _, m, l = oc.tree_attention(q, k, v, past, parents)
    m, l = m.astype(np.float32), l.astype(np.float32)
    for i, h in ((5, 1), (6, 0), (7, hq - 1)):
        q[0, i, h, 3] = (0, 2, 1)[i - 5]
    l[0, 1, 5] = 0.0
    l[0, 0, 6] = np.nan
    m[0, hq - 1, 7] = -np.inf
    if tree:
        q[0, n - 3:, :, 3] = (0, 1, -1)[n % 3]
    k[0, [20, 70, 129], :, 3] = np.inf
    zeros = np.zeros((1, hkv, past[0] + n), np.float32)
    want = oc.key_weights(q, k, past, m, l, None, zeros, parents)
    assert (want[0, :, [20, 70, 129]] == 0).all()
    tk = gpu.zeros(1, c, hkv, d, dtype=gpu.bfloat16 if dtype == "bf16" else gpu.float32,
                   device="cuda")
    tk[:, :past[0] + n] = _to(gpu, k, dtype)
    args = (_i32(gpu, past), gpu.tensor(m).cuda(), gpu.tensor(l).cuda(), None, _i32(gpu, parents))
    got = kv.key_weights(_to(gpu, q, dtype), tk, *args)[..., :past[0] + n]
    _check_weights(got, want, q, k, m, n * hq)
    tk[0, 40, 1, 7] = float("nan")  # a seen key: NaN in its own weight alone
    got = kv.key_weights(_to(gpu, q, dtype), tk, *args)[..., :past[0] + n]
    assert np.isnan(got[0, 1, 40].item())
    got[0, 1, 40] = float(want[0, 1, 40])
    _check_weights(got, want, q, k, m, n * hq)


# hq, hkv, d, past of each sequence, tokens, padding, capacity, dtype
@pytest.mark.parametrize("hq,hkv,d,past,n,pad,c,dtype", [
    (32, 8, 128, [130, 1, 31], 3, 0, 200, "bf16"),
    (8, 2, 64, [65, 700, 129], 4, 1, 710, "bf16"),
    (8, 2, 128, [1201, 33], 8, 0, 1300, "bf16"),
    (9, 3, 64, [300, 7, 190], 9, 2, 400, "bf16"),
    (4, 1, 64, [900], 12, 0, 530_000, "bf16"),
    (4, 1, 128, [900, 65], 10, 2, 120_000, "bf16"),
    (4, 2, 128, [777], 70, 4, 60_000, "bf16"),
    (4, 1, 128, [777, 1301], 160, 9, 48_000, "bf16"),
    (8, 2, 80, [130, 17], 9, 0, 200, "bf16"),
    (9, 3, 64, [300, 7], 9, 2, 400, "fp32"),
])
def test_infinities_in_a_tile_that_the_past_ends_in(gpu, hq, hkv, d, past, n, pad, c, dtype):
    """An infinite value in the past's last row makes its column infinite, a NaN one
    NaN, and no other; an infinite key that all rows score -inf has no part."""
    from longctx100m_amd import cache as kv

    rng = np.random.default_rng(n + d)
    b, used = len(past), max(past) + n
    q, k, v = _data(rng, b, n, used, hq, hkv, d, dtype)
    q[..., 3] = -np.abs(q[..., 3]) - 1
    q = bf16_round(q) if dtype == "bf16" else q
    for x in range(b):
        if past[x] > 1:
            k[x, past[x] - 2, :, 3] = np.inf
    parents = _tree(rng, b, n, pad)
    eo, em, el = oc.tree_attention(q, k, v, past, parents)
    there = np.isfinite(em[:, 0])
    for x in range(b):
        v[x, past[x] - 1, :, 7], v[x, past[x] - 1, :, d - 1] = np.inf, -np.inf
        v[x, past[x] - 1, :, 5] = np.nan
    tk, tv = (_nan(gpu, b, c, hkv, d, dtype=gpu.bfloat16 if dtype == "bf16" else gpu.float32)
              for _ in range(2))
    tk[:, :used], tv[:, :used] = _to(gpu, k, dtype), _to(gpu, v, dtype)
    for precise in ((False, True) if dtype == "bf16" and c < 1000 else (False,)):
        o, m, l = kv.tree_attention(_to(gpu, q, dtype), tk, tv, _i32(gpu, past),
                                    _i32(gpu, parents), precise=precise)
        col = o.float().cpu().numpy()
        assert (col[there][..., 7] == np.inf).all() and (col[there][..., d - 1] == -np.inf).all()
        assert np.isnan(col[there][..., 5]).all()
        o, want = o.clone(), eo.copy()
        for x in (5, 7, d - 1):
            o[..., x], want[..., x] = 0, 0
        _check_attention((o, m, l), (want, em, el), q, k, v, dtype,
                         dtype == "bf16" and not precise)


# hq, hkv, d, tokens, capacity: forms, each with several tiles of keys a wave
@pytest.mark.parametrize("hq,hkv,d,n,c", [
    (4, 1, 128, 4, 120_000), (4, 1, 128, 8, 120_000), (4, 1, 64, 8, 120_000),
    (4, 1, 64, 16, 530_000),
    (4, 1, 128, 10, 250_000), (4, 1, 128, 32, 130_000),   # 128 rows in two halves
    (4, 1, 128, 64, 70_000), (4, 1, 128, 256, 70_000),    # 256 rows
])
def test_the_largest_probability_is_not_rounded(gpu, hq, hkv, d, n, c):
    """Probabilities go to the matrix cores in bf16, relative to their row's largest
    so far: where one key has nearly all of a row's weight, its value comes out
    exactly.  Here key 133 has it, and a key of the tiles before has 2^-5 of that
    at most and the same value; the others have less than 2^-26 together.  The
    rounding of the small ones (2^-8 each) moves the output by 2^-13 of the value,
    less than half a step (2^-9 at least), which is the output's rounding."""
    from longctx100m_amd import cache as kv

    gen = gpu.Generator(device="cuda").manual_seed(n + d)
    k = gpu.full((1, c, hkv, d), -3.0, device="cuda")
    k[:, 5], k[:, 133] = 0.625 if d == 128 else 0.5, 1.0
    v = gpu.randn(1, c, hkv, d, generator=gen, device="cuda").bfloat16()
    v[:, 5] = v[:, 133]
    scale = 1 + gpu.arange(n * hq, device="cuda") % 32 / 128
    q = scale.view(1, n, hq, 1).expand(-1, -1, -1, d)
    out, _, _ = kv.tree_attention(q.bfloat16().contiguous(), k.bfloat16(), v, _i32(gpu, [c - n]))
    assert gpu.equal(out, v[:, 133:134].expand(-1, n, -1, -1).repeat(1, 1, hq, 1))
