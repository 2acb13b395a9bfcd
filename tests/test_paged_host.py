"""The paged cache and rotary positions where no GPU is needed: frequencies and
turns, the scale arithmetic and page lookup of csrc/e4m3.h compiled for the
host, the oracle's e4m3 against torch's, and refusals of the C ABI, which return
before any device work."""

import ctypes
import math
import shutil
import subprocess
from fractions import Fraction
from pathlib import Path

import numpy as np
import pytest
import torch

from longctx100m_amd import _lib, layer, paged, rotary
from oracle import paged as op

CSRC = Path(__file__).resolve().parents[1] / "longctx100m_amd" / "csrc"

HOST = r'''
#include <cstring>
#include "e4m3.h"
static uint32_t bits(float f) { uint32_t u; std::memcpy(&u, &f, 4); return u; }
static float value(uint32_t u) { float f; std::memcpy(&f, &u, 4); return f; }
extern "C" {
float scale_of(float amax) { return value(lc::scale_bits(bits(amax))); }
float inverse_of(float scale) { return value(lc::inverse_bits(bits(scale))); }
float ratio_of(float was, float now) { return value(lc::ratio_bits(bits(was), bits(now))); }
int page_of(const int32_t* table, int width, int pages, int64_t at) { return lc::page_of(table, width, pages, at); }
}
'''


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("e4m3")
    (d / "h.cpp").write_text(HOST)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-O1", f"-I{CSRC}", str(d / "h.cpp"), "-o",
                    str(d / "h.so")], check=True)
    lib = ctypes.CDLL(str(d / "h.so"))
    for name, n in (("scale_of", 1), ("inverse_of", 1), ("ratio_of", 2)):
        getattr(lib, name).restype = ctypes.c_float
        getattr(lib, name).argtypes = [ctypes.c_float] * n
    lib.page_of.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_int64]
    return lib


def test_scale_is_the_smallest_power_of_two(host):
    rng = np.random.default_rng(1)
    amax = np.float32(2.0) ** rng.uniform(-149, 127.99, 4000).astype(np.float32)
    edge = np.float32([448.0 * 2.0 ** e for e in range(-140, 119)])
    amax = np.concatenate([amax, edge, np.nextafter(edge, np.float32(np.inf)), np.nextafter(edge, np.float32(0)),
                           np.float32([0.0, 1e-45, 3.4028235e38, 2.0 ** -126, 448.0, 1.0])])
    for a in amax.astype(np.float32):
        s = host.scale_of(a)
        assert s == op.block_scale(float(a)), a
        assert float(a) <= 448.0 * s
        assert s == 2.0 ** -126 or float(a) > 224.0 * s
        assert host.inverse_of(s) == 1.0 / s


def test_ratio_of_scales(host):
    for was in (-126, -125, -10, 0, 33, 120):
        for now in range(was, 121):
            want = 2.0 ** (was - now) if was - now >= -126 else 0.0
            assert host.ratio_of(2.0 ** was, 2.0 ** now) == want


def test_page_lookup_refuses_what_is_no_page(host):
    table = (ctypes.c_int32 * 6)(3, -1, 7, 0, 2 ** 31 - 1, -2 ** 31)
    at = ctypes.addressof(table)
    assert [host.page_of(at, 6, 7, i) for i in range(6)] == [3, -1, -1, 0, -1, -1]
    for i in (-1, 6, 7, 2 ** 40, -2 ** 40):  # beyond the table: not read
        assert host.page_of(at, 6, 7, i) == -1
    assert host.page_of(None, 0, 7, 0) == -1


def test_oracle_rounds_as_e4m3():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    codes = np.unique(codes[np.isfinite(codes)])
    mid = (codes[1:] + codes[:-1]) / 2
    x = np.concatenate([codes, mid, mid * (1 + 1e-7), mid * (1 - 1e-7),
                        np.random.default_rng(2).uniform(-448, 448, 5000)])
    x = x.astype(np.float32)
    want = torch.tensor(x).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(op.e4m3(x), want)
    assert np.isnan(op.e4m3([np.inf, -np.inf, np.nan])).all()


TAU = Fraction("6.283185307179586476925286766559005768394338798750211641949889184615632812572417997256069650684234")


def test_turns_are_exact_fractions_of_a_turn():
    f = [1.0, 0.5, 1e-3, 500000.0 ** (-126 / 128), 2.0 * math.pi, 100.0, 0.0, -0.25, 1e-30, 3e5]
    turns = (ctypes.c_uint64 * len(f))()
    _lib.check(_lib.load().lc_rotary_turns(len(f), (ctypes.c_double * len(f))(*f), turns))
    for x, t in zip(f, turns):
        want = Fraction(x) / TAU * 2 ** 64
        # half a unit of rounding, and the quotient's 64 significant bits
        off = (t - want) % 2 ** 64
        assert min(off, 2 ** 64 - off) <= Fraction(1, 2) + abs(want) / 2 ** 63
    lib = _lib.load()
    assert lib.lc_rotary_turns(0, (ctypes.c_double * 1)(1.0), turns) == _lib.LC_ERR_INVALID
    assert lib.lc_rotary_turns(1, None, turns) == _lib.LC_ERR_INVALID
    for bad in (math.nan, math.inf):
        assert lib.lc_rotary_turns(1, (ctypes.c_double * 1)(bad), turns) == _lib.LC_ERR_INVALID


def test_frequencies():
    f, factor = rotary.frequencies(8, 10000.0)
    assert f == [1.0, 10000.0 ** -0.25, 10000.0 ** -0.5, 10000.0 ** -0.75] and factor == 1.0
    assert rotary.frequencies(8, 10000.0, dict(type="default"))[0] == f
    g, factor = rotary.frequencies(8, 10000.0, dict(rope_type="linear", factor=4.0))
    assert g == [x / 4 for x in f] and factor == 1.0
    # llama3: short wavelengths stay, long ones stretch, monotonous between
    sc = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
              original_max_position_embeddings=8192)
    f, _ = rotary.frequencies(128, 500000.0)
    g, factor = rotary.frequencies(128, 500000.0, sc)
    for a, b in zip(f, g):
        turns = 8192 * a / (2 * math.pi)
        if turns >= 4:
            assert b == a
        elif turns <= 1:
            assert b == a / 8
        else:
            k = (turns - 1) / 3
            assert b == pytest.approx(a * k + a / 8 * (1 - k), rel=1e-12)
    assert factor == 1.0
    # without scaling as the layer's fp32 ones: exp of an fp32 argument of at most ln theta
    inv, _ = layer.rope_inv_freq(layer.rope_params(128, 500000.0))
    assert np.allclose(inv, f, rtol=2 * math.log(500000.0) * 2.0 ** -24 + 2.0 ** -23, atol=0)
    sc = dict(rope_type="yarn", factor=32.0, original_max_position_embeddings=4096)
    f, _ = rotary.frequencies(128, 10000.0)
    g, factor = rotary.frequencies(128, 10000.0, sc)
    assert factor == pytest.approx(0.1 * math.log(32) + 1)
    lo = math.floor(128 * math.log(4096 / (64 * math.pi)) / (2 * math.log(10000)))
    hi = math.ceil(128 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000)))
    for i, (a, b) in enumerate(zip(f, g)):
        if i <= lo:
            assert b == pytest.approx(a, rel=1e-12)
        elif i >= hi:
            assert b == pytest.approx(a / 32, rel=1e-12)
        else:
            assert a / 32 < b < a
    assert rotary.frequencies(128, 10000.0, dict(sc, attention_factor=1.5))[1] == 1.5
    assert rotary.frequencies(128, 10000.0, dict(sc, factor=0.5))[1] == 1.0


@pytest.mark.parametrize("args,match", [
    ((7, 1e4), "even"), ((0, 1e4), "even"), ((-2, 1e4), "even"), ((8, 1.0), "theta"), ((8, math.nan), "theta"),
    ((8, 1e4, dict(type="wavy")), "unsupported"), ((8, 1e4, dict(type="linear", factor=0.0)), "factor"),
    ((8, 1e4, dict(type="linear", factor=math.nan)), "factor"),
    ((8, 1e4, dict(type="yarn", factor=2.0)), "original"),
    ((8, 1e4, dict(type="yarn", factor=2.0, original_max_position_embeddings=0)), "positive"),
    ((8, 1e4, dict(type="yarn", factor=2.0, original_max_position_embeddings=64, beta_fast=1.0)), "beta_fast"),
    ((8, 1e4, dict(type="llama3", factor=2.0, original_max_position_embeddings=64)), "low/high"),
    ((8, 1e4, dict(type="llama3", factor=2.0, original_max_position_embeddings=64, low_freq_factor=2.0,
                   high_freq_factor=2.0)), "above"),
])
def test_frequencies_refuse(args, match):
    with pytest.raises(ValueError, match=match):
        rotary.frequencies(*args)


def test_rotary_refuses():
    for kw, match in ((dict(head_dim=64, rotary_dim=66), "at most head_dim"), (dict(head_dim=300), "256"),
                      (dict(head_dim=64, inv_freq=[1.0] * 33), "at most head_dim"),
                      (dict(head_dim=64, inv_freq=[1.0], rotary_dim=4), "rotary_dim / 2"),
                      (dict(head_dim=64, inv_freq=[1.0], scaling=dict(type="linear")), "in place of"),
                      (dict(head_dim=64, inv_freq=[math.inf]), "finite")):
        with pytest.raises(ValueError, match=match):
            rotary.Rotary(device="cpu", **kw)
    r = rotary.Rotary(64, rotary_dim=32, device="cpu")
    assert r.rotary_dim == 32 and len(r.inv_freq) == 16 and r.turns.dtype is torch.int64
    with pytest.raises(ValueError, match="live on the GPU"):
        rotary.rotate(torch.zeros(3, 2, 64), 0, r)


def test_struct_layouts():
    assert ctypes.sizeof(_lib.Paged) == 40 and ctypes.sizeof(_lib.Rows) == 24 and ctypes.sizeof(_lib.Rotary) == 24
    assert _lib.Rotary.turns.offset == 16 and _lib.Paged.flags.offset == 36


def test_rotary_of_the_layers_profile():
    for sc in (None, dict(type="linear", factor=4.0),
               dict(type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                    original_max_position_embeddings=8192)):
        rope = layer.rope_params(128, 500000.0, sc)
        inv, _ = layer.rope_inv_freq(rope)
        r = rotary.Rotary.of(rope, device="cpu")
        assert r.inv_freq == [x / 4.0 if sc and sc["type"] == "linear" else x for x in inv]
        assert (r.head_dim, r.rotary_dim, r.interleaved, r.factor) == (128, 128, False, 1.0)
    sc["attention_factor"] = 1.5  # of cos alone: no rotation
    with pytest.raises(ValueError, match="cos alone"):
        rotary.Rotary.of(layer.rope_params(128, 500000.0, sc), device="cpu")


def test_pages_refuse():
    f8 = torch.float8_e4m3fn
    good = (torch.zeros(3, 2, 16, 32, dtype=torch.uint8).view(f8), torch.zeros(3, 2, 32, 16, dtype=torch.uint8).view(f8),
            torch.zeros(3, 2), torch.zeros(3, 2))
    p = paged.Pages.of(*good)
    assert (p.count, p.kv_heads, p.rows, p.head_dim) == (3, 2, 16, 32)
    with pytest.raises(ValueError, match="live on the GPU"):
        p.device()
    for i, bad in ((0, good[0].view(torch.uint8)), (0, good[1]), (1, good[0]), (2, torch.zeros(3, 3)),
                   (3, torch.zeros(3, 2, dtype=torch.float64)), (0, good[0][:, :, ::2]), (2, None)):
        args = list(good)
        args[i] = bad
        with pytest.raises(ValueError):
            paged.Pages.of(*args)
    with pytest.raises(ValueError, match="rows"):
        paged.Pages(2, 48, 1, 64, device="cpu")


def _desc(**kw):
    d = dict(batch=2, tokens=3, heads_q=4, heads_kv=2, head_dim=64, dtype=_lib.LC_DTYPE_BF16, pages=9, page_rows=16,
             table_width=4, flags=0)
    d.update(kw)
    return _lib.Paged(**d)


I, U, W = _lib.LC_ERR_INVALID, _lib.LC_ERR_UNSUPPORTED, _lib.LC_ERR_WORKSPACE


@pytest.mark.parametrize("kw,code", [
    (dict(batch=0), I), (dict(tokens=-1), I), (dict(heads_kv=0), I), (dict(heads_q=0), I), (dict(heads_q=3), I),
    (dict(head_dim=0), I), (dict(head_dim=24), U), (dict(head_dim=272), U), (dict(pages=0), I),
    (dict(page_rows=0), U), (dict(page_rows=48), U), (dict(page_rows=256), U), (dict(table_width=0), I),
    (dict(flags=1), I), (dict(dtype=5), U), (dict(table_width=1 << 27), U), (dict(batch=1 << 20), U),
    (dict(tokens=(1 << 24) + 1), U), (dict(tokens=1 << 24, batch=64), U), (dict(tokens=1 << 23, heads_q=6, heads_kv=6), U),
    (dict(heads_q=1 << 18, heads_kv=1), U),
])
def test_paged_descriptions_are_checked(kw, code):
    lib = _lib.load()
    d = _desc(**kw)
    a = 1 << 20  # never dereferenced
    rows = _lib.Rows(1 << 16, 1 << 10, 64)
    assert lib.lc_paged_attn_workspace_bytes(d) == 0
    assert lib.lc_paged_attn(d, *[a] * 12, 1 << 30, None) == code
    rc = lib.lc_paged_append(d, None, a, a, a, None, None, None, a, rows, a, rows, a, a, a, a, None)
    # (without queries, heads_q is not read)
    assert rc == code or ("heads_q" in kw and rc == I)
    assert lib.lc_paged_attn(None, *[a] * 12, 1 << 30, None) == I


def test_paged_attention_pointers_are_checked():
    lib = _lib.load()
    d = _desc()
    need = lib.lc_paged_attn_workspace_bytes(d)
    assert need > 0
    apart = [(i + 1) << 24 for i in range(12)]  # addresses that are never dereferenced
    # (table, past, counts, q, k, v, ks, vs, out, m, l, workspace)
    call = lambda ptrs, n=need: lib.lc_paged_attn(d, *ptrs, n, None)  # noqa: E731
    assert call(apart, need - 1) == W
    for i in (0, 1, 3, 4, 5, 6, 7, 8):
        assert call([None if j == i else p for j, p in enumerate(apart)]) == I, i
    assert call([None if j == 11 else p for j, p in enumerate(apart)]) == W
    for i, by in ((0, 2), (1, 1), (2, 2), (3, 8), (4, 8), (5, 4), (6, 2), (7, 1), (8, 8), (9, 2), (10, 1), (11, 8)):
        assert call([p + by if j == i else p for j, p in enumerate(apart)]) == I, i
    for i, j in ((8, 3), (9, 8), (10, 9), (11, 8), (11, 3), (8, 4), (9, 6), (10, 0), (11, 1), (8, 2), (4, 5), (6, 7), (4, 7)):
        assert call([apart[j] if x == i else p for x, p in enumerate(apart)]) == I, (i, j)
    assert lib.lc_paged_attn(_desc(tokens=0), *[None] * 12, 0, None) == _lib.LC_OK


def test_append_pointers_are_checked():
    lib = _lib.load()
    d = _desc()
    rows = _lib.Rows(3 * 512, 512, 64)
    rot = _lib.Rotary(64, 64, 0, 1.0, 1 << 30)
    apart = [(i + 1) << 24 for i in range(11)]  # table past counts q q_out k v kp vp ks vs

    def call(ptrs, rot=rot, d=d, r=(rows, rows, rows)):
        t, p, c, q, qo, k, v, kp, vp, ks, vs = ptrs
        return lib.lc_paged_append(d, rot, t, p, c, q, r[0], qo, k, r[1], v, r[2], kp, vp, ks, vs, None)

    for i in (0, 1, 4, 5, 6, 7, 8, 9, 10):
        assert call([None if j == i else p for j, p in enumerate(apart)]) == I, i
    assert call(apart, rot=None) == I  # queries without a rotation
    for bad in (dict(head_dim=32), dict(rotary_dim=63), dict(rotary_dim=0), dict(rotary_dim=66), dict(interleaved=2),
                dict(factor=math.nan), dict(turns=None), dict(turns=(1 << 30) + 4)):
        kw = dict(head_dim=64, rotary_dim=64, interleaved=0, factor=1.0, turns=1 << 30)
        kw.update(bad)
        assert call(apart, rot=_lib.Rotary(*kw.values())) == I, bad
    assert call(apart, rot=_lib.Rotary(64, 40, 0, 1.0, 1 << 30)) == U
    for i, by in ((0, 2), (1, 2), (2, 1), (3, 1), (4, 1), (5, 1), (6, 1), (7, 8), (8, 8), (9, 2), (10, 2)):
        assert call([p + by if j == i else p for j, p in enumerate(apart)]) == I, i
    for i, j in ((4, 5), (4, 6), (4, 0), (4, 1), (4, 2), (4, 7), (4, 9), (7, 8), (9, 10), (7, 5), (8, 6), (9, 1), (10, 0), (7, 3)):
        assert call([apart[j] if x == i else p for x, p in enumerate(apart)]) == I, (i, j)
    for r in (None, _lib.Rows(-1, 512, 64), _lib.Rows(1536, (1 << 40) + 1, 64)):
        for i in range(3):
            rr = [rows, rows, rows]
            rr[i] = r
            assert call(apart, r=rr) == I, (i, r)
    # q in place only where it is laid out as q_out: [2, 3, 4, 64] dense
    assert call([apart[3] if x == 4 else p for x, p in enumerate(apart)]) == I


def test_rotary_apply_is_checked():
    lib = _lib.load()
    rot = _lib.Rotary(64, 64, 0, 1.0, 1 << 30)
    rows = _lib.Rows(5 * 128, 128, 64)

    def call(rot=rot, dtype=1, batch=2, tokens=5, heads=2, pos=2 << 24, inverse=0, x=3 << 24, xr=rows, out=4 << 24,
             outr=rows):
        return lib.lc_rotary_apply(rot, dtype, batch, tokens, heads, pos, 0, inverse, x, xr, out, outr, None)

    for kw in (dict(rot=None), dict(batch=-1), dict(tokens=-1), dict(heads=0), dict(inverse=2), dict(x=None),
               dict(out=None), dict(xr=None), dict(outr=None), dict(pos=(2 << 24) + 4), dict(x=(3 << 24) + 1),
               dict(out=(4 << 24) + 1), dict(out=(3 << 24) + 2), dict(out=2 << 24), dict(out=1 << 30),
               dict(outr=_lib.Rows(5 * 128, 128, 32)), dict(outr=_lib.Rows(0, 128, 64)),
               dict(out=3 << 24, outr=_lib.Rows(5 * 256, 256, 64)), dict(xr=_lib.Rows(5 * 128, -128, 64)),
               dict(rot=_lib.Rotary(64, 62 + 3, 0, 1.0, 1 << 30))):
        assert call(**kw) == I, kw
    for kw in (dict(dtype=2), dict(batch=1 << 20, tokens=1 << 10), dict(rot=_lib.Rotary(512, 64, 0, 1.0, 1 << 30))):
        assert call(**kw) == U, kw
    assert call(batch=0, x=None, out=None) == _lib.LC_OK
    assert call(tokens=0) == _lib.LC_OK


def test_extents_beyond_64_bits_are_refused():
    """Strides within their bounds whose products with the sizes are not."""
    lib = _lib.load()
    far = _lib.Rows(1 << 40, 1 << 40, 64)
    near = _lib.Rows(64, 64, 64)
    rot = _lib.Rotary(64, 64, 0, 1.0, 1 << 30)
    n = 1 << 23  # n 2^40 is 2^63
    for x, out in ((far, near), (near, far)):
        for batch, tokens in ((n + 1, 1), (1, n + 1), (2, 1)):
            assert lib.lc_rotary_apply(rot, 1, batch, tokens, 1, None, 0, 0, 1 << 50, x, 1 << 52, out, None) == I
    d = _desc(tokens=n + 1, batch=1, heads_q=1, heads_kv=1)
    apart = [i << 24 for i in range(1, 8)]
    for k, v in ((far, near), (near, far)):
        rc = lib.lc_paged_append(d, None, *apart[:2], None, None, None, None, 1 << 50, k, 1 << 52, v, 1 << 54, 1 << 55,
                                 1 << 56, 1 << 57, None)
        assert rc == I


def test_tiles_of_all_sequences_are_counted_in_31_bits():
    """Sequences that share pages may have more rows together than the pool."""
    lib = _lib.load()
    a = 1 << 20  # never dereferenced
    for d in (_desc(batch=65, table_width=1 << 26), _desc(batch=1 << 10, table_width=(1 << 22) + 1)):
        assert lib.lc_paged_attn_workspace_bytes(d) == 0
        assert lib.lc_paged_attn(d, *[a] * 12, 1 << 30, None) == U
    assert lib.lc_paged_attn_workspace_bytes(_desc(batch=64, table_width=1 << 26)) > 0
