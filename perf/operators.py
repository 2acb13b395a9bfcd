"""The KV-cache operators of longctx100m_amd.cache as measurable cases, with
their plain forms.

  tree     attention of a tree of drafted tokens over a cache (tree_attention):
           what a decoder layer runs to check drafted tokens
  weights  the attention weight each cached key receives, accumulated
           (key_weights): what decides which keys a bounded cache keeps
  evict    a cache cut to a budget of rows by those weights (evict)
  commit   the rows of the accepted tokens made a contiguous continuation of
           every layer's cache (commit)

A cache is [batch, capacity, kv_heads, head_dim]; its rows before the new
tokens are the sequence's past, ragged over the batch.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
HEADS = ((9, 3), (16, 16), (32, 8), (8, 2))


def listed():
    return [
        # Eight drafted tokens, short context: the smallest call, launches and latency.
        dict(name="tree_short", kind="tree", batch=1, tokens=8, past=500, hq=32, hkv=8, d=128,
             dtype="bf16", layout="rows"),
        # A draft tree of 26 nodes against a 16k context.
        dict(name="tree_16k", kind="tree", batch=1, tokens=26, past=16001, hq=32, hkv=8, d=128,
             dtype="bf16", layout="rows"),
        # A ragged batch of conversations of a GQA 9/3, head_dim 64 model, caches kept by head.
        dict(name="tree_batch_d64", kind="tree", batch=4, tokens=16, past=3001, hq=9, hkv=3, d=64,
             dtype="bf16", layout="heads"),
        # 64 drafted tokens over a 262,144-row cache of a GQA 32/8 layer: the largest.
        dict(name="tree_long", kind="tree", batch=1, tokens=64, past=262080, hq=32, hkv=8, d=128,
             dtype="bf16", layout="rows"),
        # The fp32 model of the parity setup, two sequences.
        dict(name="tree_fp32", kind="tree", batch=2, tokens=13, past=2047, hq=9, hkv=3, d=64,
             dtype="fp32", layout="rows"),
        # One new token's weights over a 262,144-row cache: a decode step of a bounded cache.
        dict(name="weights_token", kind="weights", batch=1, tokens=1, past=262143, hq=32, hkv=8,
             d=128, dtype="bf16", layout="rows", tree=False),
        # The weights that the last 512 tokens of a 32k prompt give, before its first eviction.
        dict(name="weights_prompt", kind="weights", batch=1, tokens=512, past=32000, hq=32, hkv=8,
             d=128, dtype="bf16", layout="rows", tree=False),
        # Checked drafts of a ragged fp32 batch.
        dict(name="weights_fp32", kind="weights", batch=3, tokens=13, past=2047, hq=9, hkv=3, d=64,
             dtype="fp32", layout="heads", tree=True),
        # A 262,144-token prompt's cache cut to 16,384 rows.
        dict(name="evict_prompt", kind="evict", batch=1, rows=262144, budget=16384, hkv=8, d=128,
             dtype="bf16", layout="rows", earlier=0),
        # Ragged conversations cut back to their budget after some 250 more tokens.
        dict(name="evict_again", kind="evict", batch=4, rows=4351, budget=4096, hkv=3, d=64,
             dtype="bf16", layout="rows", earlier=4000),
        # One sequence's accepted drafts, 24 layers of 8 KV heads.
        dict(name="commit_one", kind="commit", batch=1, tokens=64, past=8000, hkv=8, d=128,
             dtype="bf16", layers=24),
        # A batch's, fp32, 12 layers of the 3-head model.
        dict(name="commit_batch", kind="commit", batch=8, tokens=16, past=1001, hkv=3, d=64,
             dtype="fp32", layers=12),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over the logarithm, odd ones among them."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("tree", "tree", "weights", "weights", "evict", "commit"))
    hq, hkv = rng.choice(HEADS)
    c = dict(kind=kind, batch=_log(rng, 1, 8), hkv=hkv, d=rng.choice((64, 128)),
             dtype=rng.choice(("bf16", "bf16", "bf16", "fp32")))
    if kind == "commit":
        c.update(tokens=_log(rng, 1, 64), past=_log(rng, 1, 4000), layers=rng.randint(1, 24))
        return c
    c["layout"] = rng.choice(("rows", "heads"))
    if kind == "evict":
        most = (1 << 21) // (c["batch"] * hkv)
        c["rows"] = _log(rng, 64, min(262144, most))
        c["budget"] = _log(rng, 16, c["rows"])
        c["earlier"] = rng.choice((0, c["budget"] * rng.randint(1, 4) // 4))
        return c
    # Query rows x keys x heads of at most the largest listed case's (a thirtieth in fp32, whose
    # products run on the fp32 matrix cores).
    most = 64 * 32 * 262144 * 128 // (1 if c["dtype"] == "bf16" else 30)
    c.update(hq=hq, tokens=_log(rng, 1, 128 if kind == "tree" else 64))
    if kind == "weights":
        c["tree"] = rng.random() < 0.5
        if not c["tree"]:
            c["tokens"] = _log(rng, 1, min(4096, math.isqrt(most // (c["batch"] * hq * c["d"]))))
    most = min(most // (c["batch"] * c["tokens"] * hq * c["d"]), (1 << 21) // (c["batch"] * hkv))
    c["past"] = _log(rng, 1, max(1, min(262080, most - c["tokens"])))
    return c


def _lens(case, name="past"):
    """Rows of each sequence: the longest first, the last about half of it."""
    n, b = case[name], case["batch"]
    return [n - i * (n // 2) // b for i in range(b)]


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _cache(gen, case, rows):
    shape = (case["batch"], rows, case["hkv"], case["d"])
    if case.get("layout") == "heads":  # [batch, heads, rows, head_dim] in memory
        b, n, h, d = shape
        return _randn(gen, b, h, n, d).to(DTYPES[case["dtype"]]).transpose(1, 2)
    return _randn(gen, *shape).to(DTYPES[case["dtype"]])


def _parents(case, seed):
    """A draft tree: node 0 is the root, most nodes hang off one of the few
    nodes before them; the second sequence of every two lacks its last nodes."""
    gen = torch.Generator().manual_seed(seed)
    b, n = case["batch"], case["tokens"]
    i = torch.arange(n)
    back = 1 + (torch.rand(b, n, generator=gen) ** 2 * 6).long()
    p = torch.clamp(i - back, min=0)
    p[:, 0] = -1
    p[1::2, n - n // 4:] = -2
    return p.to(torch.int32).to(DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": dict(case)}
    dt = DTYPES[case["dtype"]]
    if case["kind"] in ("tree", "weights"):
        b, n, hq, hkv = case["batch"], case["tokens"], case["hq"], case["hkv"]
        cap = case["past"] + n
        s["past"] = torch.tensor(_lens(case), dtype=torch.int32, device=DEV)
        s["parents"] = _parents(case, seed) if case.get("tree", True) else None
        s["q"] = (2 * _randn(gen, b, n, hq, case["d"])).to(dt)
        s["k"] = _cache(gen, case, cap)
        if case["kind"] == "tree":
            s["v"] = _cache(gen, case, cap)
            s["out"] = torch.empty_like(s["q"])
            s["m"] = torch.empty(b, hq, n, device=DEV)
            s["l"] = torch.empty_like(s["m"])
        else:  # the statistics are the attention's, the weights those of the tokens before
            sc = _scores(s["q"], s["k"], _visible(s["past"], s["parents"], n, cap))
            m = sc.amax(-1)
            l = torch.exp(sc - torch.where(m == -math.inf, 0.0, m)[..., None]).sum(-1)
            s["m"], s["l"] = (_by_head(t, hq).contiguous() for t in (m, l))
            # Each token gives a head's keys a weight of 1 in all; as many again came before.
            s["weights"] = torch.exp(_randn(gen, b, hkv, cap)) * (n * (hq // hkv) / cap)
            s["out"] = torch.zeros_like(s["weights"])
    elif case["kind"] == "evict":
        b, rows, hkv = case["batch"], case["rows"], case["hkv"]
        lens = _lens(case, "rows")
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["k"], s["v"] = _cache(gen, case, rows), _cache(gen, case, rows)
        # Long-tailed weights, some of them zero (keys that nothing attends to).
        w = torch.exp(3 * _randn(gen, b, hkv, rows))
        s["weights"] = torch.where(torch.rand(w.shape, generator=gen, device=DEV) < 0.1, 0.0, w)
        # Rows of an earlier eviction hold tokens out of order: some of the first ones.
        earlier = min(case["earlier"], min(lens))
        s["kept"] = torch.full((b,), earlier, dtype=torch.int32, device=DEV)
        s["ends"] = s["lens"] + earlier
        at = torch.rand(b, hkv, 2 * earlier, generator=gen, device=DEV).argsort(-1)[..., :earlier]
        s["positions"] = torch.zeros(b, hkv, rows, dtype=torch.int32, device=DEV)
        s["positions"][..., :earlier] = at.to(torch.int32)
        s["sinks"], s["recent"] = min(4, case["budget"] // 8), case["budget"] // 8
        s["weights_out"] = torch.zeros_like(s["weights"])
        s["positions_out"] = torch.zeros_like(s["positions"])
        s["lens_out"] = torch.zeros_like(s["lens"])
    else:
        b, n, layers = case["batch"], case["tokens"], case["layers"]
        shape = (layers, b, case["past"] + n, case["hkv"], case["d"])
        s["k"], s["v"] = _randn(gen, *shape).to(dt), _randn(gen, *shape).to(dt)
        s["past"] = torch.tensor(_lens(case), dtype=torch.int32, device=DEV)
        # The accepted path: node 0 and some of the nodes after it, one to all but a few.
        depth = torch.rand(b, n, generator=gen, device=DEV) < 0.5
        depth[:, 0] = True
        nodes = torch.where(depth, torch.arange(n, device=DEV), n).sort(-1).values[:, :10]
        s["path"] = torch.where(nodes < n, nodes, -1).to(torch.int32).contiguous()
        s["lens_out"] = torch.zeros_like(s["past"])
    if own and case["kind"] in ("tree", "evict"):
        from longctx100m_amd import cache
        if case["kind"] == "tree":
            need = cache.tree_attention_workspace_bytes(s["q"], s["k"])
        else:
            need = cache.evict_workspace_bytes(s["k"])
        s["workspace"] = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
    if own and case["kind"] == "commit":
        from longctx100m_amd import cache
        s["layers"] = cache.Layers(list(s["k"]), list(s["v"]))
    return s


# ------------------------------------------------------------ plain forms --

def _by_head(x, hq):
    """[batch, kv_heads, tokens, group] -> [batch, heads, tokens]."""
    b, _, n, _ = x.shape
    return x.transpose(2, 3).reshape(b, hq, n)


def _visible(past, parents, n, cap):
    """[batch, tokens, capacity]: the rows each new token sees."""
    i = torch.arange(n, device=DEV)
    row = torch.arange(cap, device=DEV)
    if parents is None:
        return row <= past[:, None, None] + i[:, None]
    p = parents.long()[:, :, None]
    edge = ((p == i) & (i < i[:, None])).double()
    reach = torch.linalg.matrix_power(edge + torch.eye(n, device=DEV, dtype=torch.float64), n) > 0
    there = (reach & (parents == -1)[:, None, :]).any(-1)
    node = row - past.long()[:, None]
    above = reach.gather(2, node.clamp(0, n - 1)[:, None, :].expand(-1, n, -1))
    new = (node >= 0) & (node < n)
    return there[:, :, None] & torch.where(new[:, None, :], above, (node < 0)[:, None, :])


def _scores(q, k, visible):
    """Masked scaled scores [batch, kv_heads, tokens, group, capacity]."""
    b, n, hq, d = q.shape
    hkv = k.shape[2]
    qf = q.float().view(b, n, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)
    s = torch.matmul(qf, k.float().permute(0, 2, 3, 1).contiguous()) * d ** -0.5
    s = s.view(b, hkv, n, hq // hkv, -1)
    return s.masked_fill_(~visible[:, None, :, None, :], -math.inf)


def _tree_plain(s):
    q, k, v = s["q"], s["k"], s["v"]
    b, n, hq, d = q.shape
    hkv = k.shape[2]
    sc = _scores(q, k, _visible(s["past"], s["parents"], n, k.shape[1]))
    m = sc.amax(-1)
    p = sc.sub_(torch.where(m == -math.inf, 0.0, m)[..., None]).exp_()
    l = p.sum(-1)
    o = torch.matmul(p.view(b, hkv, n * (hq // hkv), -1),
                     v.float().permute(0, 2, 1, 3).contiguous()).view(b, hkv, n, hq // hkv, d)
    o = torch.where(l[..., None] > 0, o / l[..., None], 0.0)
    return [o.permute(0, 2, 1, 3, 4).reshape(b, n, hq, d).to(q.dtype), _by_head(m, hq),
            _by_head(l, hq)]


def _weights_plain(s):
    q, k = s["q"], s["k"]
    b, n, hq, _ = q.shape
    hkv, cap = k.shape[2], k.shape[1]
    m, l = (t.view(b, hkv, hq // hkv, n).transpose(2, 3)[..., None] for t in (s["m"], s["l"]))
    sc = _scores(q, k, _visible(s["past"], s["parents"], n, cap))
    p = sc.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    w = torch.where(l > 0, p / l, 0.0).sum((2, 3))
    row = torch.arange(cap, device=DEV)
    past = s["past"][:, None, None]
    w = torch.where(row < past, s["weights"], 0.0) + w
    return [torch.where(row < past + n, w, s["out"])]


def _evict_plain(s):
    w, k, v, budget = s["weights"], s["k"], s["v"], s["case"]["budget"]
    b, hkv, rows = w.shape
    row = torch.arange(rows, device=DEV)
    lens, ends = s["lens"][:, None, None], s["ends"][:, None, None]
    pos = torch.where(row < s["kept"][:, None, None], s["positions"], ends - lens + row)
    safe = (pos < s["sinks"]) | (pos >= ends - s["recent"])
    rank = torch.where(safe, math.inf, w)
    rank = torch.where(row < lens, rank, -math.inf)
    first = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    keep = torch.zeros(w.shape, dtype=torch.bool, device=DEV).scatter_(-1, first, True)
    keep &= row < lens
    # The j-th row below the budget that goes is replaced by the j-th row from it on that stays.
    far = torch.sort(keep & (row >= budget), dim=-1, descending=True, stable=True).indices
    hole = (~keep & (row < lens))[..., :budget]
    nth = (hole.cumsum(-1) - 1).clamp(min=0)
    src = torch.where(hole, far.gather(-1, nth), row[:budget])
    at = src.transpose(1, 2)[..., None].expand(-1, -1, -1, k.shape[3])
    k[:, :budget] = k.gather(1, at)
    v[:, :budget] = v.gather(1, at)
    n_out = lens.clamp(max=budget)
    left = row[:budget] < n_out
    wo, po = s["weights_out"].clone(), s["positions_out"].clone()
    wo[..., :budget] = torch.where(left, w.gather(-1, src), wo[..., :budget])
    po[..., :budget] = torch.where(left, pos.to(torch.int32).gather(-1, src), po[..., :budget])
    return [k, v, wo, po, s["lens"].clamp(max=budget)]


def _commit_plain(s):
    k, v, past, path = s["k"], s["v"], s["past"].long(), s["path"].long()
    count = (path >= 0).sum(-1)
    j = torch.arange(path.shape[1], device=DEV)
    b = torch.arange(path.shape[0], device=DEV)[:, None]
    # Places past the path's end copy their own row.
    src = past[:, None] + torch.where(path >= 0, path, torch.minimum(j, s["k"].shape[2] - 1
                                                                     - past[:, None]))
    dst = past[:, None] + torch.where(path >= 0, j, src - past[:, None])
    k[:, b, dst] = k[:, b, src]
    v[:, b, dst] = v[:, b, src]
    return [k, v, (past + count).to(torch.int32)]


def run(state):
    c = state["case"]
    if own:
        from longctx100m_amd import cache
        if c["kind"] == "tree":
            return list(cache.tree_attention(
                state["q"], state["k"], state["v"], state["past"], state["parents"],
                out=state["out"], m=state["m"], l=state["l"], workspace=state["workspace"]))
        if c["kind"] == "weights":
            return [cache.key_weights(state["q"], state["k"], state["past"], state["m"],
                                      state["l"], state["weights"], state["parents"],
                                      out=state["out"])]
        if c["kind"] == "evict":
            w, p, n = cache.evict(
                state["k"], state["v"], state["weights"], state["lens"], c["budget"],
                sinks=state["sinks"], recent=state["recent"], positions=state["positions"],
                kept=state["kept"], ends=state["ends"], weights_out=state["weights_out"],
                positions_out=state["positions_out"], lens_out=state["lens_out"],
                workspace=state["workspace"])
            return [state["k"], state["v"], w, p, n]
        n = cache.commit(state["layers"], state["past"], state["path"],
                         lens_out=state["lens_out"])
        return [state["k"], state["v"], n]
    return {"tree": _tree_plain, "weights": _weights_plain, "evict": _evict_plain,
            "commit": _commit_plain}[c["kind"]](state)


def work(case):
    b, hkv, d = case["batch"], case["hkv"], case["d"]
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] in ("tree", "weights"):
        n, hq = case["tokens"], case["hq"]
        keys = sum(x + n for x in _lens(case))
        # Pairs a mask leaves out count for a chain; a tree's are few beside the past.
        pairs = sum(n * x + (n * (n + 1) // 2 if not case.get("tree", True) else n)
                    for x in _lens(case))
        rows = b * n * hq
        if case["kind"] == "tree":
            return {"bytes": 2 * keys * hkv * d * e + 2 * rows * d * e + 8 * rows,
                    "flops": 4 * pairs * hq * d}
        return {"bytes": keys * hkv * (d * e + 8) + rows * (d * e + 8),
                "flops": 2 * pairs * hq * d}
    if case["kind"] == "evict":
        lens, budget = _lens(case, "rows"), case["budget"]
        # Rows below the budget that go: the protected eighth stays, of the rest a like share
        # to all rows'.
        moved = sum(0.875 * budget * (1 - min(1, budget / x)) for x in lens) * hkv
        held = sum(min(x, budget) for x in lens) * hkv
        return {"bytes": 4 * moved * d * e + 4 * sum(lens) * hkv + 8 * held,
                "flops": sum(lens) * hkv}
    moved = b * min(10, 1 + (case["tokens"] - 1) // 2)
    return {"bytes": 4 * case["layers"] * moved * hkv * d * e, "flops": 0}


# ------------------------------------------------------------- in 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("commit", "evict"):
        return None  # whole numbers, and copies of given values
    hq, hkv, n = case["hq"], case["hkv"], case["tokens"]
    g = hq // hkv

    def seen_by(parents):
        """[tokens, tokens]: the new tokens that each one sees, itself included; none
        where its chain of parents does not end at a root."""
        if parents is None:
            return torch.ones(n, n, dtype=torch.bool).tril()
        seen = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            chain = [i]
            while 0 <= parents[chain[-1]] < chain[-1]:
                chain.append(parents[chain[-1]])
            if parents[chain[-1]] == -1:
                seen[i, chain] = True
        return seen

    def by_head():
        """(sequence, its past, KV head, scores, mask), the rows by (query head, token)."""
        for b, past in enumerate(s["past"].tolist()):
            new = seen_by(None if s["parents"] is None else s["parents"][b].tolist())
            old = new.any(-1, keepdim=True).expand(n, past)
            seen = torch.cat([old, new], 1).to(DEV).repeat(g, 1)
            for h in range(hkv):
                rows = s["q"][b, :, h * g:(h + 1) * g].double().transpose(0, 1).reshape(g * n, -1)
                keys = s["k"][b, :past + n, h].double()
                yield b, past, h, (rows @ keys.t()) / math.sqrt(case["d"]), seen

    if case["kind"] == "tree":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        m = torch.full(s["m"].shape, -math.inf, dtype=torch.float64, device=DEV)
        l = torch.zeros(s["l"].shape, dtype=torch.float64, device=DEV)
        for b, past, h, sc, seen in by_head():
            sc = sc.masked_fill(~seen, -math.inf)
            top = sc.max(-1).values
            e = torch.where(seen, torch.exp(sc - top[:, None]), 0.0)
            tot = e.sum(-1)
            o = e @ s["v"][b, :past + n, h].double() / tot.clamp(min=1e-300)[:, None]
            m[b, h * g:(h + 1) * g], l[b, h * g:(h + 1) * g] = top.view(g, n), tot.view(g, n)
            out[b, :, h * g:(h + 1) * g] = o.view(g, n, -1).transpose(0, 1)
        return [out, m, l]
    w = s["out"].double()
    for b, past, h, sc, seen in by_head():
        m, l = (s[x][b, h * g:(h + 1) * g].double().reshape(-1, 1) for x in ("m", "l"))
        p = torch.where(seen & (l > 0), torch.exp(sc - m) / l, 0.0).sum(0)
        p[:past] += s["weights"][b, h, :past].double()
        w[b, h, :past + n] = p
    return [w]
