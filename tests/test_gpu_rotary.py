"""Rotary positions (longctx100m_amd/rotary.py) against the float64 oracle.

Tolerance (u = 2^-24): the angle within its quarter turn, at most pi/4, is off by
three roundings of a factor each, so by 3 u pi/4 < 2.4 u, and by 2^-34 of a turn,
< 0.01 u; cos and sin by as much, by two roundings of the last steps of their
series (2 u) and the series' end (0.03 u), and times the factor by another u / 2:
5 u.  An element x1 c - x2 s is then off by 5 u f (|x1| + |x2|), by the
rounding of its two products and its difference, 2 u f (|x1| + |x2|), and by half
a step of its type.  The oracle's own angles are off by |pos| f 2^-53 + 2^-50."""

import numpy as np
import pytest

from longctx100m_amd import rotary
from oracle import paged as op
from tests.conftest import bf16_round

U = 2.0 ** -24
SCALING = {"default": None, "linear": dict(type="linear", factor=4.0),
           "yarn": dict(type="yarn", factor=32.0, original_max_position_embeddings=4096)}


def _tolerance(x, want, r, positions, dtype):
    half, n = r.rotary_dim // 2, r.rotary_dim
    pair = np.abs(x.astype(np.float64))
    a, b = (pair[..., 0:n:2], pair[..., 1:n:2]) if r.interleaved else (pair[..., :half], pair[..., half:n])
    s = a + b
    both = np.stack((s, s), -1).reshape(*s.shape[:-1], n) if r.interleaved else np.concatenate((s, s), -1)
    far = np.abs(np.asarray(positions, np.float64)).max(initial=0.0) * max(r.inv_freq) * 2.0 ** -53 + 2.0 ** -50
    far += np.abs(np.asarray(positions, np.float64)).max(initial=0.0) * 2 * np.pi * 2.0 ** -65
    tol = np.zeros(x.shape)
    tol[..., :n] = (7 * U + far) * abs(r.factor) * both
    return tol + (2.0 ** -8 if dtype == "bf16" else U) * np.abs(want)


def _data(gpu, rng, shape, dtype):
    x = rng.standard_normal(shape, dtype=np.float32)
    x = bf16_round(x) if dtype == "bf16" else x
    return x, gpu.tensor(x).to(gpu.bfloat16 if dtype == "bf16" else gpu.float32).cuda()


# tokens, heads, head_dim, rotary_dim, dtype, positions
CASES = [
    (1, 1, 128, 128, "bf16", [0]),
    (1, 40, 128, 128, "bf16", [100_000_000]),
    (7, 12, 64, 64, "bf16", [0, 1, 2, 3, 2 ** 31, 2 ** 40 + 1, -5]),
    (5, 9, 64, 64, "fp32", [99_999_999, 17, 17, 4095, 1]),
    (3, 3, 64, 16, "bf16", [5, 1000, 1_000_003]),
    (4, 16, 128, 64, "fp32", [7, 8, 9, 10]),
    (4, 2, 80, 48, "bf16", [1, 2, 3, 4]),
    (3, 5, 256, 256, "bf16", [10, 20, 30]),
    (3, 2, 256, 32, "fp32", [10, 20, 30]),
    (6, 3, 64, 20, "bf16", [0, 5, 2, 8, 9, 77]),      # pairs that are no whole vectors
    (2, 4, 50, 50, "fp32", [3, 12345]),               # a head that is none
    (2, 3, 10, 2, "bf16", [1, 2]),
    (1030, 3, 64, 32, "bf16", None),                  # tokens in groups of four, the last smaller
    (1027, 1, 16, 16, "fp32", None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("scaling", sorted(SCALING))
@pytest.mark.parametrize("case", CASES)
def test_rotate(gpu, case, scaling, interleaved):
    tokens, heads, d, rd, dtype, positions = case
    rng = np.random.default_rng(tokens + d)
    if positions is None:
        positions = rng.integers(-2 ** 33, 2 ** 33, tokens).tolist()
    x, tx = _data(gpu, rng, (tokens, heads, d), dtype)
    r = rotary.Rotary(d, 500000.0, rotary_dim=rd, interleaved=interleaved, scaling=SCALING[scaling])
    tp = gpu.tensor(positions, dtype=gpu.int64).cuda()
    for turn, backward in ((rotary.rotate, False), (rotary.rotate_backward, True)):
        # (few enough tokens for the oracle's loops)
        at = np.arange(tokens) if tokens < 100 else np.concatenate([np.arange(6), np.arange(tokens - 6, tokens)])
        some = [positions[i] for i in at]
        want = op.rotate(x[at], some, r.inv_freq, r.factor, interleaved, backward)
        tol = _tolerance(x[at], want, r, some, dtype)
        out = gpu.full_like(tx, float("nan"))
        got = turn(tx, tp, r, out=out)
        assert got is out
        assert (np.abs(got.float().cpu().numpy()[at] - want) <= tol).all()
        assert gpu.equal(turn(tx, tp, r), out)
        same = tx.clone()  # in place
        assert gpu.equal(turn(same, tp, r, out=same), out)
        assert gpu.equal(out[..., rd:], tx[..., rd:])
        assert not out.isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strides_and_first_positions(gpu, dtype):
    """Columns of a fused projection, heads outside tokens, rows that no vector fits,
    and positions that follow from the first."""
    rng = np.random.default_rng(3)
    b, n, h, d = 3, 11, 5, 64
    x, tx = _data(gpu, rng, (b, n, h, d), dtype)
    r = rotary.Rotary(d, 10000.0)
    at = gpu.arange(1000, 1000 + n, device="cuda").repeat(b, 1)
    want = rotary.rotate(tx, at, r)
    assert gpu.equal(rotary.rotate(tx, 1000, r), want)
    assert gpu.equal(rotary.rotate(tx[1], 1000, r), want[1])
    big = gpu.full((b, n, h + 3, d), float("nan"), dtype=tx.dtype, device="cuda")
    big[:, :, 2:2 + h] = tx
    odd = gpu.zeros(b * n * h * (d + 1) + 1, dtype=tx.dtype, device="cuda")[1:].view(b, n, h, d + 1)[..., :d]
    odd.copy_(tx)
    for view in (big[:, :, 2:2 + h], tx.transpose(1, 2).contiguous().transpose(1, 2), odd):
        assert gpu.equal(rotary.rotate(view, 1000, r), want)
        assert gpu.equal(rotary.rotate(tx, at, r, out=gpu.empty_like(view.transpose(1, 2).contiguous()).transpose(1, 2)),
                         want)
    inner = big[:, :, 2:2 + h]
    rotary.rotate(inner, 1000, r, out=inner)
    assert gpu.equal(inner, want) and big[:, :, :2].isnan().all() and big[:, :, 2 + h:].isnan().all()
    spread = rotary.rotate(tx[:1, :1].expand(b, n, h, d), 1000, r)  # one row for all
    one = rotary.rotate(tx[:1, :1].expand(b, n, h, d).contiguous(), 1000, r)
    assert gpu.equal(spread, one)
    assert rotary.rotate(tx[:, :0], 5, r).shape == (b, 0, h, d)
    assert rotary.rotate(tx[:0], 5, r).shape == (0, n, h, d)


@pytest.mark.gpu
def test_backward_is_the_gradient(gpu):
    """<rotate_backward(g), x> = <g, rotate(x)>, and differences of a loss along
    directions: the map is linear, so they are exact but for rounding."""
    rng = np.random.default_rng(4)
    for interleaved in (False, True):
        r = rotary.Rotary(64, 500000.0, rotary_dim=32, interleaved=interleaved, scaling=SCALING["yarn"])
        _, x = _data(gpu, rng, (9, 4, 64), "fp32")
        _, g = _data(gpu, rng, (9, 4, 64), "fp32")
        _, v = _data(gpu, rng, (9, 4, 64), "fp32")
        at = gpu.tensor(rng.integers(0, 10 ** 8, 9), dtype=gpu.int64).cuda()
        dx = rotary.rotate_backward(g, at, r).double()
        n = x.numel()
        # each of n products of elements off by 8 u f (|x1| + |x2|) at most
        tol = 2 * n * 8 * U * r.factor * 2 * float(x.abs().max() * g.abs().max())
        assert abs(float((dx * x.double()).sum() - (g.double() * rotary.rotate(x, at, r).double()).sum())) <= tol
        loss = lambda y: (g.double() * rotary.rotate(y, at, r).double()).sum()  # noqa: E731
        diff = float(loss(x + v) - loss(x - v)) / 2
        tol = 4 * n * 8 * U * r.factor * 2 * float((x.abs() + v.abs()).max() * g.abs().max())
        assert abs(diff - float((dx * v.double()).sum())) <= tol


@pytest.mark.gpu
def test_special_values_and_far_positions(gpu):
    r = rotary.Rotary(64, 10000.0, rotary_dim=32)
    x = gpu.ones(2, 3, 64, device="cuda")
    x[0, 1, 3] = float("nan")
    x[1, 2, 40] = float("inf")
    y = rotary.rotate(x, 9, r)
    assert y[0, 1, [3, 19]].isnan().all() and y.isnan().sum() == 2
    assert y[1, 2, 40] == float("inf")
    # 2^62 positions on: the turns of whole numbers of 2^-64 come round
    a, b = rotary.rotate(x, 2 ** 62 - 2, r)[1, 0], rotary.rotate(x, 2 ** 62 - 1, r)[0, 0]
    assert gpu.equal(a, b) and not a.isnan().any()
    with pytest.raises(ValueError, match="62 bits"):
        rotary.rotate(x, 2 ** 62, r)


@pytest.mark.gpu
def test_refusals(gpu):
    r = rotary.Rotary(64, 10000.0)
    x = gpu.zeros(2, 3, 64, device="cuda")
    at = gpu.zeros(2, dtype=gpu.int64, device="cuda")
    for args, kw in (((x.half(), at, r), {}), ((x[..., :32], at, r), {}), ((x[0], at, r), {}),
                     ((x, at.int(), r), {}), ((x, at[:1], r), {}), ((x, at.cpu(), r), {}), ((x.cpu(), at, r), {}),
                     ((x, gpu.zeros(4, dtype=gpu.int64, device="cuda")[::2], r), {}),
                     ((gpu.zeros(2, 3, 128, device="cuda")[..., ::2], at, r), {}),
                     ((x, at, r), dict(out=x.bfloat16())), ((x, at, r), dict(out=x[:1])),
                     ((x, at, r), dict(out=x.cpu())), ((x, at, r), dict(out=x[:1].expand(2, 3, 64))),
                     ((x, at, rotary.Rotary(64, 10000.0, device="cpu")), {})):
        with pytest.raises(ValueError):
            rotary.rotate(*args, **kw)
    flat = gpu.zeros(2 * 3 * 64 + 64, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        rotary.rotate(flat[:384].view(2, 3, 64), at, r, out=flat[64:].view(2, 3, 64))
    with pytest.raises(ValueError, match="overlap"):
        rotary.rotate(x, x.view(gpu.int64).view(-1)[:2], r, out=x)


@pytest.mark.gpu
def test_streams_and_graphs(gpu):
    rng = np.random.default_rng(6)
    r = rotary.Rotary(128, 500000.0)
    _, x = _data(gpu, rng, (33, 40, 128), "bf16")
    at = gpu.arange(33, device="cuda")
    want = rotary.rotate(x, at, r)
    s = gpu.cuda.Stream()
    s.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(s):
        got = rotary.rotate(x, at, r)
    s.synchronize()
    assert gpu.equal(got, want)
    out = gpu.zeros_like(x)
    g = gpu.cuda.CUDAGraph()
    gpu.cuda.synchronize()
    with gpu.cuda.graph(g):
        rotary.rotate(x, at, r, out=out)
    for shift in (0, 5, 10 ** 8):
        at.copy_(gpu.arange(33, device="cuda") + shift)
        g.replay()
        gpu.cuda.synchronize()
        assert gpu.equal(out, rotary.rotate(x, at, r))


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d,rd", [(80, 40), (40, 24), (128, 100), (90, 90), (33, 32), (65, 6), (255, 254), (2, 2), (3, 2)])
@pytest.mark.parametrize("heads", [1, 7, 300])
def test_pairs_that_are_no_vectors(gpu, heads, d, rd, dtype, interleaved):
    """Four pairs at a time, or one; heads of odd size; more heads than a workgroup takes
    at once; rows of 8-byte alignment."""
    rng = np.random.default_rng(d + heads)
    tokens = 1030 if heads == 7 else 3
    x, tx = _data(gpu, rng, (tokens, heads, d), dtype)
    r = rotary.Rotary(d, 500000.0, rotary_dim=rd, interleaved=interleaved)
    positions = rng.integers(-2 ** 30, 2 ** 30, tokens).tolist()
    tp = gpu.tensor(positions, dtype=gpu.int64).cuda()
    at = [0, tokens // 2, tokens - 1]
    some = [positions[i] for i in at]
    for turn, backward in ((rotary.rotate, False), (rotary.rotate_backward, True)):
        want = op.rotate(x[at], some, r.inv_freq, r.factor, interleaved, backward)
        out = gpu.full_like(tx, float("nan"))
        turn(tx, tp, r, out=out)
        assert (np.abs(out.float().cpu().numpy()[at] - want) <= _tolerance(x[at], want, r, some, dtype)).all()
        assert gpu.equal(out[..., rd:], tx[..., rd:]) and not out.isnan().any()
        same = tx.clone()
        assert gpu.equal(turn(same, tp, r, out=same), out)
        # the same rows 8 bytes on, with 8 bytes between the heads
        pad = 8 // tx.element_size()
        room = gpu.full((tokens * heads * (d + pad) + pad,), float("nan"), dtype=tx.dtype, device="cuda")
        view = room[pad:].view(tokens, heads, d + pad)[..., :d]
        view.copy_(tx)
        assert gpu.equal(turn(view, tp, r, out=view), out)
        assert int(room.isnan().sum()) == pad * (tokens * heads + 1)
