"""The float64 oracle of the KV-cache operators (oracle/cache.py) pinned to the
dense attention oracle and to hand-made cases; the C ABI's refusals, before any
device work; the Python layer's checks.  Runs without a GPU."""

import ctypes

import numpy as np
import pytest

from longctx100m_amd import _lib
from longctx100m_amd import cache as kv
from oracle import cache as oc
from oracle import dense


def test_chain_is_causal_attention():
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal(s) for s in ((2, 5, 4, 16), (2, 12, 2, 16), (2, 12, 2, 16)))
    out, m, l = oc.tree_attention(q, k, v, [7, 7])
    eo, em, el = dense.attention_fwd(q, k, v, q_pos0=7, k_pos0=0, valid_length=None)
    assert np.abs(out - eo).max() < 1e-12 and np.abs(m - em).max() < 1e-12
    assert np.abs(l - el).max() < 1e-12


def test_tree_is_the_chain_of_each_path():
    """Node 4 of the tree 0-1-4, 0-2, 3 (padding) sees what the third token of
    the chain 0, 1, 4 sees."""
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal(s) for s in ((1, 6, 2, 16), (1, 11, 2, 16), (1, 11, 2, 16)))
    parents = [[-1, 0, 0, -2, 1, 3]]
    out, m, l = oc.tree_attention(q, k, v, [5], parents)
    rows = [0, 1, 2, 3, 4, 5, 6, 9]
    eo, em, el = oc.tree_attention(q[:, [0, 1, 4]], k[:, rows], v[:, rows], [5])
    assert np.allclose(out[:, 4], eo[:, 2]) and np.allclose(m[..., 4], em[..., 2])
    assert np.allclose(l[..., 4], el[..., 2])
    for i in (3, 5):  # padding, and a child of padding
        assert (out[:, i] == 0).all() and (m[..., i] == -np.inf).all() and (l[..., i] == 0).all()
    # each query row gives its keys a weight of one in all
    w = oc.key_weights(q, k, [5], m, l, None, np.zeros((1, 2, 11)), parents)
    assert abs(w.sum() - 4 * 2) < 1e-12 and (w[:, :, 8] == 0).all()


def test_evict_by_hand():
    k = np.arange(8, dtype=np.float32).reshape(1, 8, 1, 1)
    w = np.array([[[5, 1, 3, 3, 9, 3, 0, 2]]], np.float32)
    k2, _, w2, p2, n2 = oc.evict(k, k, w, [8], 4, sinks=0, recent=1)
    # row 7 is protected; 4 and 0 by weight; of the three 3s the lowest row
    assert n2 == [4] and k2[0, :4, 0, 0].tolist() == [0, 4, 2, 7]
    assert w2[0, 0, :4].tolist() == [5, 9, 3, 2] and p2[0, 0, :4].tolist() == [0, 4, 2, 7]


def test_commit_by_hand():
    k = np.arange(8, dtype=np.float32).reshape(1, 8, 1, 1)
    k2, _, n = oc.commit(k, k, [2], [[0, 2, 3, -1, 5]])
    assert n == [5] and k2[0, :, 0, 0].tolist() == [0, 1, 2, 4, 5, 5, 6, 7]


def test_tree_depths():
    assert kv.tree_depths([-1, 0, 0, 1, -2, 4, -1, 6, 9]) == [0, 1, 1, 2, -1, -1, 0, 1, -1]


# ------------------------------------------------------------- refusals --

P = 1 << 20  # a pointer that is never read: the calls below return before any device work


def _cache(**kw):
    c = dict(batch=2, tokens=4, capacity=100, heads_q=8, heads_kv=2, head_dim=64,
             dtype=_lib.LC_DTYPE_BF16, flags=0, seq_stride=100 * 128, row_stride=128,
             head_stride=64)
    c.update(kw)
    return _lib.Cache(**c)


def _calls(lib, c):
    ks, vs = (ctypes.c_void_p * 1)(P), (ctypes.c_void_p * 1)(2 * P)
    pp, vv = (ctypes.cast(x, ctypes.POINTER(ctypes.c_void_p)) for x in (ks, vs))
    big = 1 << 40
    return {
        "attn": lambda: lib.lc_cache_attn(c, P, None, P, P, P, P, P, P, P, big, None),
        "weights": lambda: lib.lc_cache_weights(c, P, None, P, P, P, P, None, P, None),
        "evict": lambda: lib.lc_cache_evict(c, 10, 1, 1, P, None, None, P, P, P, None, 2 * P,
                                            3 * P, 4 * P, P, big, None),
        "commit": lambda: lib.lc_cache_commit(c, 1, pp, vv, P, 2 * P, 3 * P, None),
    }


READS = ("attn", "weights")
ALL = ("attn", "weights", "evict", "commit")


@pytest.mark.parametrize("kw,code,who", [
    (dict(batch=0), _lib.LC_ERR_INVALID, ALL),
    (dict(tokens=-1), _lib.LC_ERR_INVALID, ALL),
    (dict(capacity=0), _lib.LC_ERR_INVALID, ALL),
    (dict(heads_kv=0), _lib.LC_ERR_INVALID, ALL),
    (dict(heads_q=7), _lib.LC_ERR_INVALID, READS),
    (dict(dtype=2), _lib.LC_ERR_UNSUPPORTED, ALL),
    (dict(flags=_lib.LC_FLAG_ACCUMULATE), _lib.LC_ERR_INVALID, ALL),
    (dict(head_dim=72), _lib.LC_ERR_UNSUPPORTED, ALL),
    (dict(head_dim=272), _lib.LC_ERR_UNSUPPORTED, ALL),
    (dict(row_stride=132), _lib.LC_ERR_INVALID, ALL),
    (dict(head_stride=-64), _lib.LC_ERR_INVALID, ALL),
    (dict(row_stride=1 << 25, seq_stride=1 << 40), _lib.LC_ERR_UNSUPPORTED, ALL),
    (dict(batch=1 << 20, capacity=1 << 20), _lib.LC_ERR_UNSUPPORTED, ALL),
    (dict(heads_q=2 << 24), _lib.LC_ERR_UNSUPPORTED, READS),
    (dict(batch=1 << 20, heads_kv=4, head_stride=64, row_stride=256), _lib.LC_ERR_UNSUPPORTED, ALL),
    (dict(tokens=256, batch=1 << 12, heads_q=8), _lib.LC_ERR_UNSUPPORTED, ("attn",)),
    (dict(tokens=1 << 28, heads_q=8), _lib.LC_ERR_UNSUPPORTED, READS),
    (dict(seq_stride=0), _lib.LC_ERR_INVALID, ("evict", "commit")),      # sequences share rows
    (dict(row_stride=64), _lib.LC_ERR_INVALID, ("evict", "commit")),     # rows overlap heads
    (dict(seq_stride=(1 << 40) + 8), _lib.LC_ERR_UNSUPPORTED, ("attn", "weights", "evict", "commit")),
    (dict(head_stride=(1 << 40) + 8), _lib.LC_ERR_UNSUPPORTED, ("attn", "weights", "evict", "commit")),
    (dict(head_stride=32), _lib.LC_ERR_INVALID, ("evict", "commit")),
])
def test_cache_refusals(kw, code, who):
    lib = _lib.load()
    for name in who:
        assert _calls(lib, _cache(**kw))[name]() == code, name
    if "attn" in who:
        assert lib.lc_cache_attn_workspace_bytes(_cache(**kw)) == 0
    if "evict" in who:
        assert lib.lc_cache_evict_workspace_bytes(_cache(**kw)) == 0


def test_argument_refusals():
    lib = _lib.load()
    c = _cache()
    err = lambda: lib.lc_last_error().decode()  # noqa: E731
    inv = _lib.LC_ERR_INVALID
    big = 1 << 40
    # attention
    assert lib.lc_cache_attn(None, P, None, P, P, P, P, P, P, P, big, None) == inv
    assert lib.lc_cache_attn(c, None, None, P, P, P, P, P, P, P, big, None) == inv
    assert lib.lc_cache_attn(c, P, None, P, P + 2, P, P, P, P, P, big, None) == inv
    assert "16-byte" in err()
    assert lib.lc_cache_attn(c, P + 2, None, P, P, P, P, P, P, P, big, None) == inv
    need = lib.lc_cache_attn_workspace_bytes(c)
    assert need > 0
    assert lib.lc_cache_attn(c, P, None, P, P, P, P, P, P, P, need - 1, None) == \
        _lib.LC_ERR_WORKSPACE and str(need) in err()
    assert lib.lc_cache_attn(c, P, None, P, P, P, P, P, P, None, big, None) == _lib.LC_ERR_WORKSPACE
    assert lib.lc_cache_attn(c, P, None, P, P, P, P, P, P, P + 4, big, None) == inv
    long = _cache(tokens=257)
    assert lib.lc_cache_attn(long, P, None, P, P, P, P, P, P, P, big, None) == \
        _lib.LC_ERR_UNSUPPORTED
    assert lib.lc_cache_attn(_cache(tokens=0), P, None, None, P, P, None, None, None, None, 0,
                             None) == 0  # nothing to do
    # weights
    assert lib.lc_cache_weights(long, P, P, P, P, P, P, None, P, None) == _lib.LC_ERR_UNSUPPORTED
    assert lib.lc_cache_weights(c, P, None, P, P, P, None, None, P, None) == inv
    assert lib.lc_cache_weights(c, P, None, P, P, P, P, P + 4, P, None) == inv
    assert "overlap" in err()
    # eviction
    ev = lambda b=10, s=1, r=1, lens=P, kept=None, ends=None, w=5 * P, pos=None, wo=2 * P,\
        po=3 * P, lo=4 * P, ws=big: lib.lc_cache_evict(  # noqa: E731
            c, b, s, r, lens, kept, ends, P, P, w, pos, wo, po, lo, P, ws, None)
    assert ev(b=0) == inv and "budget" in err()
    assert ev(s=-1) == inv and ev(s=6, r=5) == inv and "fit the budget" in err()
    assert ev(s=2**31 - 1, r=2**31 - 1) == inv
    assert ev(kept=6 * P) == inv and "positions" in err()
    assert ev(lo=P) == inv and ev(lo=2 * P + 4) == inv and ev(wo=5 * P + 4) == inv
    assert ev(pos=2 * P) == inv and ev(po=5 * P) == inv
    assert ev(ws=lib.lc_cache_evict_workspace_bytes(c) - 1) == _lib.LC_ERR_WORKSPACE
    # commit
    ks, vs = (ctypes.c_void_p * 2)(P, None), (ctypes.c_void_p * 2)(2 * P, 3 * P)
    pp, vv = (ctypes.cast(x, ctypes.POINTER(ctypes.c_void_p)) for x in (ks, vs))
    assert lib.lc_cache_commit(c, 2, pp, vv, P, 2 * P, 3 * P, None) == inv and "layer 1" in err()
    assert lib.lc_cache_commit(c, -1, pp, vv, P, 2 * P, 3 * P, None) == inv
    assert lib.lc_cache_commit(c, 1, pp, vv, P, 2 * P, P + 4, None) == inv
    assert lib.lc_cache_commit(c, 1, pp, vv, P, 2 * P, 2 * P + 28, None) == inv
    assert lib.lc_cache_commit(c, 1, None, pp, P, 2 * P, 3 * P, None) == inv
    assert lib.lc_cache_commit(c, 1, pp, pp, P, 2 * P, 3 * P, None) == inv and "same cache" in err()


def test_python_refuses_cpu_tensors():
    import torch

    k = torch.zeros(1, 8, 2, 16)
    q = torch.zeros(1, 2, 4, 16)
    past = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        kv.tree_attention(q, k, k, past)
    with pytest.raises(ValueError, match="GPU"):
        kv.key_weights(q, k, past, q, q)
    with pytest.raises(ValueError, match="GPU"):
        kv.evict(k, k, torch.zeros(1, 2, 8), past, 4)
    with pytest.raises(ValueError, match="GPU"):
        kv.Layers([k], [k])
    with pytest.raises(ValueError, match="one k and one v"):
        kv.Layers([], [])


def test_workspace_does_not_grow_with_the_capacity_alone():
    """The partials of the splits are bounded by what the chip holds at once."""
    lib = _lib.load()
    size = lambda **kw: lib.lc_cache_attn_workspace_bytes(_cache(**kw))  # noqa: E731
    long = dict(capacity=1 << 20, seq_stride=(1 << 20) * 128)
    assert size(**long) == size(capacity=1 << 19, seq_stride=(1 << 19) * 128)
    assert size(tokens=0) == 0
    assert size(tokens=64, **long) < 64 << 20
