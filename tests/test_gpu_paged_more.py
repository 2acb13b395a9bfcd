"""The paged 8-bit cache and rotary positions: copies of their handles, and calls that
other tests of them do not make."""

import copy

import pytest

pytestmark = pytest.mark.gpu


def _i32(gpu, x):
    return gpu.tensor(x, dtype=gpu.int32).cuda()


def _bytes(gpu, p):
    return [t.view(gpu.uint8).clone() for t in (p.k, p.v, p.k_scale, p.v_scale)]


def test_a_copied_pool_is_a_pool_of_its_own(gpu):
    """An append to a copy of a pool leaves the pool as it was, and attention over the
    copy sees the copy's rows."""
    from longctx100m_amd import paged

    gen = gpu.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: gpu.randn(*s, generator=gen, device="cuda").bfloat16()  # noqa: E731
    p = paged.Pages(4, 16, 2, 64)
    table, past = _i32(gpu, [[2, 0]]), _i32(gpu, [0])
    paged.append(p, table, past, rand(1, 20, 2, 64), rand(1, 20, 2, 64))
    q, before = rand(1, 20, 4, 64), _bytes(gpu, p)
    want = paged.attention(q, p, table, past)
    other = copy.deepcopy(p)
    for x, y in zip(want, paged.attention(q, other, table, past)):
        assert gpu.equal(x, y)
    k, v = rand(1, 20, 2, 64), rand(1, 20, 2, 64)
    paged.append(other, table, past, k, v)
    for x, y in zip(_bytes(gpu, p), before):
        assert gpu.equal(x, y)
    for x, y in zip(want, paged.attention(q, p, table, past)):
        assert gpu.equal(x, y)
    fresh = paged.Pages(4, 16, 2, 64)
    paged.append(fresh, table, past, k, v)
    for x, y in zip(paged.attention(q, fresh, table, past), paged.attention(q, other, table, past)):
        assert gpu.equal(x, y)
