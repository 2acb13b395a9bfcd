"""layer.PagedCache: a model over paged 8-bit caches.  A layer is the composition
of the operators it is documented as; and the logits of prompts in pieces, ragged
batches, drafts and sequences that come and go are those of a float64 attention
over what the pools hold (norm-relative, the suite's bars: bf16 2e-2, fp32 1e-4)."""

import numpy as np
import pytest

from oracle import paged as op
from tests.conftest import norm_rel

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ly(gpu):
    from longctx100m_amd import layer

    return layer


def _model(ly, gpu, dtype, heads=(4, 2), d=128, layers=2):
    cfg = ly.ModelConfig(hidden_size=d * heads[0], num_heads=heads[0], num_key_value_heads=heads[1],
                         intermediate_size=512, num_layers=layers, vocab_size=1000, rope_theta=500000.0)
    gen = gpu.Generator(device="cuda")
    gen.manual_seed(37)
    return cfg, ly.init_model_weights(cfg, gen, "cuda", dtype=dtype, std=0.05), gen


def _np(t):
    return t.detach().float().cpu().numpy()


def _pool(p):
    return {"k": _np(p.k).astype(np.float64), "v": _np(p.v).astype(np.float64),
            "k_scale": _np(p.k_scale).astype(np.float64), "v_scale": _np(p.v_scale).astype(np.float64)}


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_layer_is_its_operators(ly, gpu, dtype):
    from longctx100m_amd import paged, rotary

    cfg, weights, gen = _model(ly, gpu, getattr(gpu, dtype))
    w, d, hq, hkv = weights["layers"][0], cfg.head_dim, 4, 2
    b, n = 3, 5
    x = gpu.randn(b * n, cfg.hidden_size, generator=gen, device="cuda").to(w["wo"].dtype)
    r = gpu.randn(b * n, cfg.hidden_size, generator=gen, device="cuda").to(x.dtype)
    i32 = dict(dtype=gpu.int32, device="cuda")
    table, past, counts = gpu.tensor([[0], [3], [2]], **i32), gpu.tensor([0, 7, 2], **i32), gpu.tensor([5, 3, 1], **i32)
    rot = rotary.Rotary(d, 500000.0)
    mine, other = paged.Pages(4, 16, hkv, d), paged.Pages(4, 16, hkv, d)
    x2, mlp = ly.layer_extend_paged(x, w, cfg, rot, mine, table, past, counts, residual=r)
    xin = gpu.empty_like(x)
    h = ly.rmsnorm(x, w["norm1"], cfg.rms_norm_eps, residual=r, residual_out=xin)
    qkv = ly.linear(h, w["wqkv"])
    at = (past.long()[:, None] + gpu.arange(n, device="cuda"))
    q = rotary.rotate(qkv[:, :hq * d].reshape(b, n, hq, d), at, rot)
    paged.append(other, table, past, qkv[:, hq * d:(hq + hkv) * d].reshape(b, n, hkv, d),
                 qkv[:, (hq + hkv) * d:].reshape(b, n, hkv, d), counts=counts, rotary=rot)
    a = paged.attention(q, other, table, past, counts=counts)[0]
    for name in ("k", "v", "k_scale", "v_scale"):
        assert gpu.equal(getattr(mine, name).view(gpu.uint8), getattr(other, name).view(gpu.uint8))
    want = gpu.empty_like(x)
    h2 = ly.rmsnorm(xin, w["norm2"], cfg.rms_norm_eps, residual=ly.linear(a.view(b * n, -1), w["wo"]), residual_out=want)
    gu = ly.linear(h2, w["wgu"])
    assert gpu.equal(x2, want)
    assert gpu.equal(mlp, ly.linear(ly.swiglu(gu[:, :512], gu[:, 512:]), w["wd"]))


@pytest.mark.parametrize("dtype,bar", [("bfloat16", 2e-2), ("float32", 1e-4)])
def test_logits_over_what_the_pools_hold(ly, gpu, dtype, bar):
    from longctx100m_amd import rotary

    cfg, weights, gen = _model(ly, gpu, getattr(gpu, dtype))
    hq, hkv, d = 4, 2, cfg.head_dim
    c = ly.PagedCache(cfg, pages=40, sequences=3, device="cuda", page_rows=16)
    rand = lambda n: gpu.randint(0, cfg.vocab_size, (n,), generator=gen, device="cuda")  # noqa: E731

    def want(slot, ids, past):
        """The logits of the last of ids, whose K and V are in the pools: its path
        through the layers alone, attending to the pools in float64."""
        x = gpu.nn.functional.embedding(ids, weights["embed"])
        res, n = None, ids.numel()
        table = np.array([c._pages[slot]])
        for w, p in zip(weights["layers"], c.pools):
            xin = gpu.empty_like(x)
            h = ly.rmsnorm(x, w["norm1"], cfg.rms_norm_eps, residual=res if res is not None else gpu.zeros_like(x),
                           residual_out=xin)
            qkv = ly.linear(h, w["wqkv"]).view(n, hq + 2 * hkv, d)
            q = rotary.rotate(qkv[:, :hq], past, c.rotary)
            pool = _pool(p)
            # the rows' K and V are those of the tokens, rounded to e4m3: half a step of 2^-3
            # relatively or 2^-9 of the scale, and the type's own error
            k = _np(rotary.rotate(qkv[:, hq:hq + hkv], past, c.rotary))
            v = _np(qkv[:, hq + hkv:])
            for i in range(n):
                page, row = table[0][(past + i) // 16], (past + i) % 16
                for got, true, s in ((pool["k"][page, :, row], k[i], pool["k_scale"][page]),
                                     (pool["v"][page, :, :, row], v[i], pool["v_scale"][page])):
                    off = np.abs(got * s[:, None] - true)
                    # (scales that later rows raised: rounded once more)
                    assert (off <= 2 * (2.0 ** -4 * np.abs(true) + 2.0 ** -10 * s[:, None]) + bar * np.abs(true).max()).all()
            out = op.attention(_np(q)[None], pool, table, [past], [n])[0]
            a = gpu.tensor(out, device="cuda").to(x.dtype).view(n, hq * d)
            x = gpu.empty_like(xin)
            h2 = ly.rmsnorm(xin, w["norm2"], cfg.rms_norm_eps, residual=ly.linear(a, w["wo"]), residual_out=x)
            gu = ly.linear(h2, w["wgu"])
            res = ly.linear(ly.swiglu(gu[:, :512], gu[:, 512:]), w["wd"])
        h = ly.rmsnorm(x, weights["final_norm"], cfg.rms_norm_eps, residual=res)
        return _np(ly.linear(h, weights["lm_head"]))[-1]

    def step(slots, counts):
        ids = [rand(n) for n in counts]
        past = [c.rows[s] for s in slots]
        got = _np(c.extend(slots, ids, weights))
        for g, s, t, p in zip(got, slots, ids, past):
            assert norm_rel(g, want(s, t, p)) <= bar

    a, b = c.open(), c.open()
    step([a, b], [70, 1])          # a prompt beside a single token
    step([b], [33])                # the rest of a prompt, over page ends
    step([a, b], [1, 1])           # a decode step
    step([b, a], [4, 5])           # drafts
    held = set(c._pages[a])
    c.close(a)
    d2, e = c.open(), c.open()
    step([d2, e, b], [100, 9, 1])  # the freed pages again, full of the old sequence's rows
    assert held & set(c._pages[d2])
    step([e], [1])
