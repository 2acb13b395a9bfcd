"""Sizes and counts beyond the C ABI's 32 bits, which ctypes would cut to their
low bits without an error: refused by the Python layer (longctx100m_amd/cache.py)."""

import pytest
import torch

from longctx100m_amd import cache as kv


@pytest.mark.parametrize("x", [2 ** 31, 2 ** 32 + 10, -2 ** 31 - 1, -2 ** 32 + 10])
def test_int32(x):
    with pytest.raises(ValueError, match="32 bits"):
        kv._int32(x, "budget")


def test_int32_takes_its_range():
    assert [kv._int32(x, "n") for x in (-2 ** 31, 0, 2 ** 31 - 1)] == [-2 ** 31, 0, 2 ** 31 - 1]


@pytest.mark.parametrize("shape,tokens,heads", [
    ((2 ** 32 + 5, 4, 2, 16), 1, 2), ((1, 2 ** 32 + 5, 2, 16), 1, 2), ((1, 4, 2 ** 31, 16), 1, 2),
    ((1, 4, 2, 16), 2 ** 31, 2), ((1, 4, 2, 16), 1, 2 ** 32 + 2)])
def test_shapes(shape, tokens, heads):
    """(A dimension of stride 0 holds so many rows in little memory.)"""
    k = torch.zeros(1, 1, 1, 16).expand(shape)
    with pytest.raises(ValueError, match="32 bits"):
        kv._describe(k, tokens, heads)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(budget=2 ** 32 + 4), dict(budget=-2 ** 32 + 4),
                                dict(budget=4, sinks=2 ** 32 + 1), dict(budget=4, recent=-2 ** 32 + 1)])
def test_evict_refuses_them(gpu, kw):
    k = gpu.rand(1, 8, 2, 64, device="cuda")
    was, lens = k.clone(), gpu.full((1,), 8, dtype=gpu.int32, device="cuda")
    with pytest.raises(ValueError, match="32 bits"):
        kv.evict(k, k.clone(), gpu.zeros(1, 2, 8, device="cuda"), lens, **kw)
    assert gpu.equal(k, was)
