"""layer.BoundedCache: a model decoded by trees of drafted tokens over caches that
are held to a budget, against the full prefill of the same tokens (bf16 bar 2e-2,
as the decode step's) and against the rows that the caches have to hold."""

import numpy as np
import pytest

from tests.conftest import norm_rel

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ly(gpu):
    from longctx100m_amd import layer

    return layer


def _model(ly, gpu, heads=(4, 2), layers=2):
    cfg = ly.ModelConfig(hidden_size=128 * heads[0], num_heads=heads[0],
                         num_key_value_heads=heads[1], intermediate_size=1024, num_layers=layers,
                         vocab_size=1000, rope_theta=500000.0)
    gen = gpu.Generator(device="cuda")
    gen.manual_seed(31)
    return cfg, ly.init_model_weights(cfg, gen, "cuda", std=0.05), gen


def _np(t):
    return t.detach().float().cpu().numpy()


def test_tree_logits_are_those_of_each_path(ly, gpu):
    """Every node's logits equal the prefill's at the end of its path, over two
    rounds of drafting; one node alone is a decode step."""
    cfg, weights, gen = _model(ly, gpu)
    T = 150
    ids = gpu.randint(0, cfg.vocab_size, (T,), generator=gen, device="cuda")
    table = ly.rope_table(ly.rope_params(cfg.head_dim, cfg.rope_theta), T + 32, 0)
    c = ly.BoundedCache(cfg, T + 32, "cuda")
    full = ly.model_prefill(ids, weights, cfg, table[:T])
    assert gpu.equal(c.prefill(ids, weights, table), full)
    text = ids
    for parents, path in (([-1, 0, 0, 1, 1, 4, -1, 6], [0, 1, 4, 5]), ([-1, 0, 1, 0], [0, 3]),
                          ([-1], [0])):
        draft = gpu.randint(0, cfg.vocab_size, (len(parents),), generator=gen, device="cuda")
        logits = c.decode(draft, parents, weights, table)
        for i in range(len(parents)):
            chain = [i]
            while parents[chain[0]] >= 0:
                chain.insert(0, parents[chain[0]])
            seq = gpu.cat([text, draft[chain]])
            want = ly.model_prefill(seq, weights, cfg, table[:seq.numel()])[-1]
            assert norm_rel(_np(logits[i]), _np(want)) <= 2e-2, (parents, i)
        c.commit(path)
        text = gpu.cat([text, draft[path]])
        assert c.past == c.end == text.numel()
    # the committed caches are the prefill's
    ref = ly.new_cache(cfg, T + 32, "cuda")
    ly.model_prefill(text, weights, cfg, table[:text.numel()], ref)
    for (k, v), (rk, rv) in zip(c.caches, ref):
        n = text.numel()
        assert norm_rel(_np(k[:, :n]), _np(rk[:, :n])) <= 2e-2
        assert norm_rel(_np(v[:, :n]), _np(rv[:, :n])) <= 2e-2
    # and a decode step over them goes on from there
    nxt = gpu.randint(0, cfg.vocab_size, (1,), generator=gen, device="cuda")
    a = ly.model_decode_step(int(nxt), c.past, weights, cfg, table, c.caches)
    b = c.decode(nxt, [-1], weights, table)
    assert norm_rel(_np(b), _np(a)) <= 2e-2


def test_bounded_cache_holds_the_rows_it_says(ly, gpu):
    """Through drafting, commits and evictions each row holds the K and V of the
    token its position names, the protected tokens stay, and each query row's
    weight of one was given out in full."""
    cfg, weights, gen = _model(ly, gpu, heads=(4, 2))
    T, budget, sinks, recent = 200, 96, 4, 24
    ids = gpu.randint(0, cfg.vocab_size, (T,), generator=gen, device="cuda")
    table = ly.rope_table(ly.rope_params(cfg.head_dim, cfg.rope_theta), 512, 0)
    c = ly.BoundedCache(cfg, 240, "cuda")
    c.prefill(ids, weights, table, window=50)
    for w in c.weights:  # 50 tokens x 2 query heads per KV head
        total = _np(w).sum(-1)
        assert np.abs(total - 100).max() < 1e-3
    seen = [[(_np(k[0, :T]), _np(v[0, :T]))] for k, v in c.caches]  # rows by token, per layer
    for rnd in range(4):
        before = [_np(w).sum(-1) for w in c.weights]
        c.evict(budget, sinks=sinks, recent=recent)
        assert c.past == budget
        for li, ((k, v), p, w) in enumerate(zip(c.caches, c.positions, c.weights)):
            allk = np.concatenate([x for x, _ in seen[li]])
            allv = np.concatenate([y for _, y in seen[li]])
            assert len(allk) == c.end
            assert (_np(w[..., :budget]).sum(-1) <= before[li] + 1e-3).all()
            for h in range(cfg.num_key_value_heads):
                pos = p[0, h, :budget].cpu().numpy()
                assert len(set(pos.tolist())) == budget
                must = set(range(sinks)) | set(range(c.end - recent, c.end))
                assert must <= set(pos.tolist())
                np.testing.assert_array_equal(_np(k[0, :budget, h]), allk[pos, h])
                np.testing.assert_array_equal(_np(v[0, :budget, h]), allv[pos, h])
        for parents, path in (([-1, 0, 0, 2, 3, 1], [0, 2, 3, 4]), ([-1, -1, 1], [1, 2])):
            draft = gpu.randint(0, cfg.vocab_size, (len(parents),), generator=gen, device="cuda")
            logits = c.decode(draft, parents, weights, table)
            assert bool(gpu.isfinite(logits).all())
            at = c.past
            held = [_np(w[..., :at]).sum(-1) for w in c.weights]
            c.commit(path)
            for li, ((k, v), w) in enumerate(zip(c.caches, c.weights)):
                seen[li].append((_np(k[0, at:c.past]), _np(v[0, at:c.past])))
                total = _np(w[..., :c.past]).sum(-1)
                assert np.abs(total - held[li] - 2 * len(path)).max() < 1e-3


def test_bounded_cache_refuses(ly, gpu):
    cfg, weights, gen = _model(ly, gpu, layers=1)
    table = ly.rope_table(ly.rope_params(cfg.head_dim, cfg.rope_theta), 20, 0)
    c = ly.BoundedCache(cfg, 16, "cuda")
    ids = gpu.randint(0, cfg.vocab_size, (10,), generator=gen, device="cuda")
    with pytest.raises(ValueError, match="prompt"):
        c.prefill(gpu.cat([ids, ids]), weights, table)
    c.prefill(ids, weights, table)
    with pytest.raises(ValueError, match="capacity"):
        c.decode(ids[:7], [-1] * 7, weights, table)
    with pytest.raises(ValueError, match="parent"):
        c.decode(ids[:2], [-1], weights, table)
    c.decode(ids[:3], [-1, 0, 0], weights, table)
    for bad in ([1], [0, 1, 2], [0, 3], [2, 0]):
        with pytest.raises(ValueError, match="chain"):
            c.commit(bad)
    c.commit([0, 2])
    assert c.past == 12 and c.end == 12
    c.commit([])  # nothing drafted, nothing kept
    with pytest.raises(ValueError, match="chain"):
        c.commit([0])
    short = table[:13]
    with pytest.raises(ValueError, match="RoPE"):
        c.decode(ids[:2], [-1, 0], weights, short)
    c.evict(12)
    assert c.kept == 0  # nothing to do
