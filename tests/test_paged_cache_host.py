"""What layer.PagedCache decides on the host: slots, pages, tables, and what a
refused or failing call leaves behind.  The layers are replaced by a recorder, so
this runs without a GPU."""

import pytest
import torch

from longctx100m_amd import layer as ly
from longctx100m_amd import paged
from longctx100m_amd import rotary as rot

CFG = ly.ModelConfig(hidden_size=64, num_heads=4, num_key_value_heads=2, intermediate_size=64, num_layers=2,
                     vocab_size=50)


@pytest.fixture
def cache(monkeypatch):
    calls = []

    def layer(x, w, cfg, rotary, pages, table, past, counts, residual=None, workspace=None):
        if w.get("fail"):
            raise RuntimeError("a layer failed")
        calls.append((x.shape[0], table.tolist(), past.tolist(), None if counts is None else counts.tolist()))
        return x + 1, x * 2

    monkeypatch.setattr(ly, "layer_extend_paged", layer)
    monkeypatch.setattr(ly, "rmsnorm", lambda x, w, eps, residual=None: x + residual)
    c = ly.PagedCache(CFG, pages=6, sequences=3, device="cpu", page_rows=16)
    weights = {"embed": torch.randn(50, 64), "lm_head": torch.randn(50, 64), "final_norm": torch.ones(64),
               "layers": [{}, {}]}
    return c, weights, calls


def ids(n):
    return torch.arange(n) % 50


def test_pages_follow_the_rows(cache):
    c, w, calls = cache
    a, b = c.open(), c.open()
    assert (a, b) == (0, 1) and c.free_pages == 6
    out = c.extend([a, b], [ids(16), ids(3)], w)
    assert out.shape == (2, 50) and c.rows[:2] == [16, 3] and c.free_pages == 4
    assert len(calls) == 2  # layers
    rows, table, past, counts = calls[0]
    assert rows == 32 and past == [0, 0] and counts == [16, 3]
    assert len({x for t in table for x in t}) == 2 and len(table[0]) == 1
    c.extend([b, a], [ids(1), ids(1)], w)  # a's next page
    rows, table, past, counts = calls[-1]
    assert past == [3, 16] and counts is None and table[0][1] == -1
    assert table[1][0] == calls[0][1][0][0] and table[0][0] == calls[0][1][1][0]
    assert c.rows[:2] == [17, 4] and c.free_pages == 3
    # the logits are those of the last tokens: each layer adds one, the last residual twice x
    x = w["embed"][ids(1)]
    assert torch.allclose(c.extend([b], [ids(1)], w), (x + 2 + 2 * (x + 1)) @ w["lm_head"].t(), atol=1e-5)


def test_last_tokens_of_a_padded_batch(cache):
    c, w, _ = cache
    a, b = c.open(), c.open()
    out = c.extend([a, b], [ids(5) + 7, ids(2) + 20], w)
    x = w["embed"][[11, 21]]
    assert torch.allclose(out, (x + 2 + 2 * (x + 1)) @ w["lm_head"].t(), atol=1e-5)


def test_closed_sequences_give_their_pages_back(cache):
    c, w, _ = cache
    a = c.open()
    c.extend([a], [ids(90)], w)
    assert c.free_pages == 0
    with pytest.raises(ValueError, match="pages are needed"):
        c.extend([a], [ids(7)], w)
    assert c.rows[a] == 90
    c.extend([a], [ids(6)], w)  # the last page's rows
    c.close(a)
    assert c.free_pages == 6 and c.rows[a] == 0
    for bad in (a, 1, 3, -1):
        with pytest.raises(ValueError, match="no sequence"):
            c.close(bad)
    assert [c.open() for _ in range(3)] == [0, 1, 2]
    with pytest.raises(ValueError, match="all 3"):
        c.open()


def test_refused_and_failing_calls_leave_everything(cache):
    c, w, calls = cache
    a, b = c.open(), c.open()
    c.extend([a], [ids(20)], w)
    before = (list(c.rows), list(c._free), [None if p is None else list(p) for p in c._pages], len(calls))
    for slots, toks in (([], []), ([a, a], [ids(1), ids(1)]), ([a], [ids(1), ids(1)]), ([a], [ids(0)]),
                        ([a], [ids(4).view(2, 2)]), ([2], [ids(1)]), ([a, b], [ids(1), ids(80)])):
        with pytest.raises(ValueError):
            c.extend(slots, toks, w)
    bad = dict(w, layers=[{}, {"fail": True}])
    with pytest.raises(RuntimeError, match="a layer failed"):
        c.extend([a, b], [ids(20), ids(5)], bad)
    after = (list(c.rows), list(c._free), [None if p is None else list(p) for p in c._pages])
    assert after == before[:3]
    c.extend([b, a], [ids(1), ids(1)], w)
    assert c.rows[:2] == [21, 1]
    held = [x for p in c._pages if p for x in p] + c._free
    assert sorted(held) == list(range(6))


def test_sizes(monkeypatch):
    for kw in (dict(pages=0, sequences=1), dict(pages=1, sequences=0), dict(pages=-1, sequences=1)):
        with pytest.raises(ValueError):
            ly.PagedCache(CFG, device="cpu", **kw)
    r = rot.Rotary(16, 100.0, device="cpu")
    c = ly.PagedCache(CFG, 2, 1, "cpu", rotary=r)
    assert c.rotary is r and len(c.pools) == 2 and c.pools[0].rows == 64
    assert ly.PagedCache(CFG, 2, 1, "cpu").rotary.inv_freq[0] == 1.0


def test_runs_on_its_own_device(cache, monkeypatch):
    """Layers and the final norm run with the tensors' device current, and tables are
    made where the cache was, not where the current device is by then."""
    from contextlib import contextmanager

    c, w, calls = cache
    inside = []

    @contextmanager
    def device_of(t):
        inside.append(t.device)
        yield
        inside.pop()

    monkeypatch.setattr(torch.cuda, "device_of", device_of)
    for name in ("layer_extend_paged", "rmsnorm"):
        was = getattr(ly, name)

        def checked(*args, was=was, **kw):
            assert inside == [torch.device("cpu")]
            return was(*args, **kw)

        monkeypatch.setattr(ly, name, checked)
    c.extend([c.open()], [ids(3)], w)
    assert len(calls) == 2 and not inside
    assert isinstance(c._device, torch.device)


def test_a_layer_needs_tokens_of_every_sequence():
    for rows, b in ((5, 2), (0, 2), (3, 0)):
        with pytest.raises(ValueError, match="sequences"):
            ly.layer_extend_paged(torch.zeros(rows, 64), {}, CFG, None, None, torch.zeros(b, 1), None)


def test_a_pool_has_its_own_addresses():
    """Copies of a pool are pools of their own tensors, and a pool's tensors and sizes,
    which the kernels' addresses and bounds come from, cannot be replaced."""
    import copy
    import io

    p = paged.Pages(3, 16, 2, 64, device="cpu")
    file = io.BytesIO()
    torch.save(p, file)
    file.seek(0)
    for q in (copy.deepcopy(p), torch.load(file, weights_only=False)):
        assert q._ptrs == tuple(t.data_ptr() for t in (q.k, q.v, q.k_scale, q.v_scale))
        assert not set(q._ptrs) & set(p._ptrs)
        assert (q.count, q.kv_heads, q.rows, q.head_dim) == (3, 2, 16, 64)
    assert copy.copy(p)._ptrs == p._ptrs
    for name in ("k", "v", "k_scale", "v_scale", "rows", "count", "kv_heads", "head_dim"):
        with pytest.raises(AttributeError, match="Pages.of"):
            setattr(p, name, getattr(p, name))
    p.k.set_(torch.zeros(3, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn))
    assert p._ptrs[0] == p.k.data_ptr()


def test_a_rotation_stays_as_it_is_made(monkeypatch):
    """What the C ABI is given follows from the attributes, of which none can be set,
    and a copy of a rotation that was used has frequencies of its own."""
    import copy

    r = rot.Rotary(64, 10000.0, rotary_dim=32, interleaved=True, factor=0.5, device="cpu")
    for name, value in (("factor", 2.0), ("turns", r.turns.clone()), ("interleaved", False), ("rotary_dim", 64),
                        ("head_dim", 128), ("inv_freq", [1.0] * 16)):
        with pytest.raises(AttributeError, match="another Rotary"):
            setattr(r, name, value)
    with pytest.raises(ValueError, match="live on cpu"):
        r.on(0)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    for x in (r, copy.deepcopy(r), copy.copy(r)):
        c = x.on(0)
        assert (c.head_dim, c.rotary_dim, c.interleaved, c.factor) == (64, 32, 1, 0.5)
        assert c.turns == x.turns.data_ptr()
    assert copy.deepcopy(r).on(0).turns != r.on(0).turns


def test_rotate_is_differentiable(monkeypatch):
    """Autograd reaches x through rotate and rotate_backward, by the kernel of the other,
    twice if asked; a result in ``out`` has no graph, so it is refused where a gradient is
    wanted."""
    calls = []

    def turn(x, positions, rotary, out, inverse):  # what the kernel does: (half layout, whole head)
        assert x.stride(-1) == 1
        at = positions if isinstance(positions, torch.Tensor) else positions + torch.arange(x.shape[0])
        angle = at.double()[:, None, None] * torch.tensor(rotary.inv_freq, dtype=torch.float64) * (-1) ** inverse
        a, b = x.detach().chunk(2, -1)
        calls.append(inverse)
        return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1) * rotary.factor

    monkeypatch.setattr(rot, "_turn", turn)
    r = rot.Rotary(8, 100.0, factor=1.5, device="cpu")
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(5, 3, 8, dtype=torch.float64, generator=gen, requires_grad=True)
    for at in (torch.tensor([4, 0, 100, -3, 7]), 9):
        for f in (rot.rotate, rot.rotate_backward):
            assert torch.autograd.gradcheck(lambda y: f(y, at, r), (x,))
            assert torch.autograd.gradgradcheck(lambda y: f(y, at, r), (x,))
            calls.clear()
            (g,) = torch.autograd.grad(f(x, at, r).sum(), x)  # the gradient of a sum: strides of zero
            assert torch.equal(g, turn(torch.ones_like(x), at, r, None, int(f is rot.rotate)))
            with pytest.raises(ValueError, match="no_grad"):
                f(x, at, r, out=torch.empty_like(x))
            with torch.no_grad():
                assert not f(x, at, r, out=torch.empty_like(x)).requires_grad
            assert not f(x.detach(), at, r, out=torch.empty_like(x)).requires_grad
    at = torch.tensor([4, 0, 100, -3, 7])
    y = rot.rotate(x, at, r).sum()
    at += 1  # the backward pass would take other angles
    with pytest.raises(RuntimeError, match="modified"):
        y.backward()


def test_scales_are_powers_of_two():
    """A pool of scales that are none would be read wrongly without a word."""
    def pool(name, value):
        p = paged.Pages(3, 16, 2, 64, device="cpu")
        scales = {"k_scale": p.k_scale.clone(), "v_scale": p.v_scale.clone()}
        scales[name][2, 1] = value
        return paged.Pages.of(p.k, p.v, **scales)

    for name in ("k_scale", "v_scale"):
        for good in (0.0, 1.0, 2.0 ** -126, 2.0 ** 120, 0.25, float("nan")):
            pool(name, good)
        for bad in (3.1 / 448, 3.0, 1.0 + 2.0 ** -23, 2.0 ** 121, 2.0 ** -127, 1e-45, -1.0, float("inf"), -0.25):
            with pytest.raises(ValueError, match=rf"{name}\[2, 1\].*power of two"):
                pool(name, bad)


def test_rows_that_are_taken_back(cache):
    """A sequence with fewer rows than its pages hold takes none from the others, keeps its
    pages and writes into them again; rows that it never had are refused."""
    c, w, calls = cache
    a, b = c.open(), c.open()
    c.extend([a, b], [ids(40), ids(3)], w)
    pa, pb = list(c._pages[a]), list(c._pages[b])
    c.rows[a] = 10  # two pages more than it needs
    c.extend([a, b], [ids(1), ids(30)], w)
    _, table, past, counts = calls[-1]
    assert past == [10, 3] and counts == [1, 30]
    assert table[0] == pa and table[1][0] == pb[0]
    assert all(0 <= x < 6 for x in table[1]) and len(set(table[0] + table[1])) == 6
    assert c.rows[:2] == [11, 33] and c.free_pages == 0
    c.extend([a], [ids(37)], w)
    assert calls[-1][1] == [pa] and c.rows[a] == 48
    for rows in (-1, 49):
        c.rows[a] = rows
        before = len(calls)
        with pytest.raises(ValueError, match="do not hold"):
            c.extend([b, a], [ids(1), ids(1)], w)
        assert len(calls) == before
    c.close(a)
    c.close(b)
    assert sorted(c._free) == list(range(6))


def test_weights_of_as_many_layers(cache):
    c, w, calls = cache
    a = c.open()
    for layers in ([{}], [{}, {}, {}]):
        with pytest.raises(ValueError, match="2 layers"):
            c.extend([a], [ids(1)], dict(w, layers=layers))
    assert not calls and c.rows[a] == 0 and c.free_pages == 6
