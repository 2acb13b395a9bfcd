"""What layer.BoundedCache decides on the host: which trees and paths it takes
and what a refused call leaves behind.  The kernels are replaced by recorders,
so this runs without a GPU."""

import pytest
import torch

from longctx100m_amd import layer as ly


class Recorder:
    """Stands for longctx100m_amd.cache: notes the calls that reach it."""

    def __init__(self, real):
        self.real, self.calls = real, []

    def __getattr__(self, name):
        if name in ("tree_depths", "MAX_TOKENS"):
            return getattr(self.real, name)
        return lambda *a, **kw: self.calls.append(name)


def _bounded(monkeypatch, past=10, capacity=100, layers=2):
    kv = Recorder(ly.kv)
    monkeypatch.setattr(ly, "kv", kv)
    c = object.__new__(ly.BoundedCache)
    c.cfg = ly.ModelConfig(hidden_size=64, num_heads=4, num_key_value_heads=2,
                           intermediate_size=64, num_layers=layers, vocab_size=50)
    c.capacity, c.past, c.kept, c.end = capacity, past, 0, past
    c.caches = ly.new_cache(c.cfg, capacity, "cpu", torch.float32)
    c.layers = None
    c.weights = [torch.zeros(1, 2, capacity) for _ in c.caches]
    c.positions = [torch.zeros(1, 2, capacity, dtype=torch.int32) for _ in c.caches]
    c._device = torch.device("cpu")
    c._drafts, c._parents = [], []
    return c, kv


def _drafted(c, parents):
    """As after a decode of this tree."""
    n = len(parents)
    c._parents = list(parents)
    c._drafts = [(torch.zeros(1, n, 4, 16), torch.zeros(1, 4, n), torch.ones(1, 4, n))
                 for _ in c.caches]


@pytest.mark.parametrize("parents,path", [
    ([-1, 2, 0], [0, 2, 1]),        # node 1 names a later node: padding
    ([1, -1], [1, 0]),
    ([-1, 1, 0], [0, 1]),           # node 1 names itself
    ([-1, 3, 0, 2], [0, 2, 3, 1]),
    ([-1, -2, 0], [1]),
    ([-1, 0, 1], [0, 2]),
    ([-1, 0, 1], [1]),
    ([-1, 0], [0, -1]),
    ([-1, 0], [0, 2]),
])
def test_commit_refuses_paths_through_padding(monkeypatch, parents, path):
    c, kv = _bounded(monkeypatch)
    _drafted(c, parents)
    with pytest.raises(ValueError, match="chain"):
        c.commit(path)
    assert kv.calls == [] and (c.past, c.end) == (10, 10)
    c.commit([parents.index(-1)])  # the tree is still there
    assert kv.calls == ["commit", "key_weights", "key_weights"] and (c.past, c.end) == (11, 11)


@pytest.mark.parametrize("parents", [[-2], [5, -2], [-1, -2], [-1, 0]])
def test_decode_refuses_a_table_that_ends_at_the_tree(monkeypatch, parents):
    """Padding takes a row of the table too, where its tree has no other node."""
    c, kv = _bounded(monkeypatch, past=20)
    table = torch.zeros(20 + max(ly.kv.tree_depths(parents) + [0]), 2, 8)
    with pytest.raises(ValueError, match="RoPE"):
        c.decode(torch.zeros(len(parents), dtype=torch.long), parents, {}, table)
    assert kv.calls == [] and c.past == 20


def test_a_decode_that_fails_leaves_no_tree(monkeypatch):
    """A tree whose rows not every layer has cannot be committed, nor the one
    before it, whose rows are overwritten; a call that is refused leaves it."""
    c, kv = _bounded(monkeypatch)
    _drafted(c, [-1, 0])
    layers = []

    def one_layer(x, *a, observe=None, **kw):
        layers.append(x)
        if len(layers) > 1:
            raise RuntimeError("out of memory")
        observe(torch.zeros(1, 3, 4, 16), torch.zeros(1, 4, 3), torch.ones(1, 4, 3))
        return x, x

    monkeypatch.setattr(ly, "layer_decode_tree", one_layer)
    ids, table = torch.zeros(3, dtype=torch.long), torch.zeros(100, 2, 8)
    weights = {"embed": torch.zeros(50, 64), "layers": [{}, {}]}
    with pytest.raises(ValueError, match="parent"):
        c.decode(ids, [-1, 0], weights, table)
    assert len(c._parents) == len(c._drafts) == 2
    with pytest.raises(RuntimeError, match="memory"):
        c.decode(ids, [-1, 0, 0], weights, table)
    for path in ([0], [0, 1], [0, 2]):
        with pytest.raises(ValueError, match="chain"):
            c.commit(path)
    assert kv.calls == [] and c.past == 10


@pytest.mark.parametrize("kw", [dict(budget=0), dict(budget=-3), dict(budget=20, recent=17),
                                dict(budget=20, sinks=-1, recent=2), dict(budget=39, recent=-1)])
def test_evict_refuses_before_it_drops_the_tree(monkeypatch, kw):
    c, kv = _bounded(monkeypatch, past=40)
    _drafted(c, [-1, 0])
    with pytest.raises(ValueError, match="budget"):
        c.evict(**kw)
    assert kv.calls == [] and (c.past, c.kept) == (40, 0)
    c.commit([0, 1])
    assert c.past == 42


def test_evict_within_the_budget_drops_the_tree(monkeypatch):
    c, kv = _bounded(monkeypatch, past=40)
    _drafted(c, [-1, 0])
    c.evict(40)
    assert kv.calls == [] and (c.past, c.kept) == (40, 0)
    with pytest.raises(ValueError, match="chain"):
        c.commit([0])
