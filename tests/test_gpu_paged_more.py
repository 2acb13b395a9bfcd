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


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
def test_gradients_reach_what_was_rotated(gpu, interleaved, dtype):
    """Queries and keys rotated before the ring's attention: their gradients are the
    rotation's backward pass of those that the attention gives."""
    from longctx100m_amd import ring_attention as ra
    from longctx100m_amd import rotary

    gen = gpu.Generator(device="cuda").manual_seed(2)
    rand = lambda h: gpu.randn(1, 128, h, 64, generator=gen, device="cuda").to(getattr(gpu, dtype))  # noqa: E731
    r = rotary.Rotary(64, 500000.0, rotary_dim=32, interleaved=interleaved)
    q, k, v = rand(4).requires_grad_(), rand(2).requires_grad_(), rand(2).requires_grad_()
    at = 10 ** 8 + gpu.arange(128, device="cuda")[None]
    qr, kr = rotary.rotate(q, at, r), rotary.rotate(k, 10 ** 8, r)
    assert gpu.equal(qr, rotary.rotate(q.detach(), at, r)) and qr.requires_grad
    for t in (qr, kr):
        t.retain_grad()
    out = ra.RingCausalAttention.apply(qr, kr, v, [(qr, kr, v)], 0, True, None)
    out.backward(rand(4))
    for x, y in ((q, qr), (k, kr)):
        assert x.grad.abs().max() > 0
        assert gpu.equal(x.grad, rotary.rotate_backward(y.grad, at, r))
    # a gradient whose rows are no vectors, and a whole shard's sum
    (g,) = gpu.autograd.grad(rotary.rotate(k, at, r).sum(), k)
    assert gpu.equal(g, rotary.rotate_backward(gpu.ones_like(k), at, r))
    (g,) = gpu.autograd.grad(rotary.rotate(k, at, r).transpose(1, 3).contiguous().sum(1), k,
                             gpu.ones(1, 2, 128, dtype=k.dtype, device="cuda"))
    assert gpu.equal(g, rotary.rotate_backward(gpu.ones_like(k), at, r))
    with pytest.raises(ValueError, match="no_grad"):
        rotary.rotate(q, at, r, out=gpu.empty_like(q))
    assert rotary.rotate(q[:, :0], at[:, :0], r).shape == (1, 0, 4, 64)


def test_a_captured_training_step_of_a_rotation(gpu):
    """Forward and backward in one graph, replayed with other rows, positions and
    gradients, beside eager work."""
    from longctx100m_amd import rotary

    gen = gpu.Generator(device="cuda").manual_seed(3)
    rand = lambda: gpu.randn(33, 6, 128, generator=gen, device="cuda").bfloat16()  # noqa: E731
    r = rotary.Rotary(128, 500000.0)
    x, g, at = rand().requires_grad_(), rand(), gpu.arange(33, device="cuda")
    gpu.cuda.synchronize()
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph):
        y = rotary.rotate(x, at, r)
        (dx,) = gpu.autograd.grad(y, x, g)
    y = y.detach()
    for shift in (0, 7, 10 ** 8):
        with gpu.no_grad():
            x.copy_(rand())
        g.copy_(rand())
        at.copy_(gpu.arange(33, device="cuda") + shift)
        graph.replay()
        gpu.cuda.synchronize()
        assert gpu.equal(y, rotary.rotate(x.detach(), at, r))
        assert gpu.equal(dx, rotary.rotate_backward(g, at, r))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_drafts_that_are_taken_back(gpu, dtype):
    """A past that is lowered: the rows behind it are not seen, the next append writes over
    them and the rows before stay, also where the drafts raised their page's scale."""
    import numpy as np

    from longctx100m_amd import paged
    from oracle import paged as op
    from tests.test_gpu_paged import _from_pages, _pool, _rows, _to_pages
    from tests.test_paged_bounds import _attend, _expected, _faults

    rng = np.random.default_rng(21)
    hkv, d, rows = 2, 64, 16
    table = np.array([[4, 1, 3], [0, 2, 5]])
    pool = _pool(rng, 6, rows, hkv, d)
    p = _to_pages(gpu, pool)
    for past, n, scale in (([0, 0], 20, 1.0), ([20, 20], 9, 60.0), ([22, 15], 4, 1.0), ([3, 16], 13, 0.1)):
        k, tk = _rows(gpu, rng, 2, n, hkv, d, dtype, scale)
        v, tv = _rows(gpu, rng, 2, n, hkv, d, dtype, scale)
        paged.append(p, _i32(gpu, table), _i32(gpu, past), tk, tv)
        op.append(pool, table, past, [n] * 2, k, v)
        got = _from_pages(p)
        for name in ("k", "v", "k_scale", "v_scale"):
            assert np.array_equal(got[name], pool[name]), name
        q, _ = _rows(gpu, rng, 2, n, 4, d, dtype, 1.5)
        want = _expected(q, pool, table, past, [n] * 2, dtype)
        assert _faults(_attend(gpu, q, p, table, past, None, dtype), want) == []
