"""Rotary positions and the paged 8-bit KV cache as measurable cases, with their
plain forms.

  rotate  rotary positions of queries and keys, forward and backward
          (longctx100m_amd.rotary): pairs half a head apart or side by side, part
          of the head, frequencies scaled for long contexts, far positions
  append  new tokens' keys, rotated on the way, and values into a paged cache
          held in e4m3, their queries rotated beside (longctx100m_amd.paged.append)
  attend  attention of new tokens over such a cache (longctx100m_amd.paged.attention)

A page holds the K and V of page_rows tokens, [heads, rows, head_dim] and
[heads, head_dim, rows] in e4m3, and each head of it has one scale for K and
one for V: a power of two, the smallest that brings what the page has been
given to 448 at most.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
HEADS = ((9, 3), (16, 16), (32, 8), (8, 2))
YARN = dict(type="yarn", factor=32.0, original_max_position_embeddings=4096)
LLAMA3 = dict(type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
              original_max_position_embeddings=8192)
SCALING = {"default": None, "linear": dict(type="linear", factor=4.0), "llama3": LLAMA3, "yarn": YARN}


def listed():
    return [
        # The queries and keys of a decode step of eight conversations: launches and latency.
        dict(name="rotate_tokens", kind="rotate", tokens=8, heads=40, d=128, rotary=128,
             interleaved=False, scaling="llama3", far=8000, dtype="bf16", backward=False),
        # The queries and keys of a 32,768-token shard of a GQA 32/8 layer.
        dict(name="rotate_shard", kind="rotate", tokens=32768, heads=40, d=128, rotary=128,
             interleaved=False, scaling="default", far=100000000, dtype="bf16", backward=False),
        # Training at far positions, half of each head rotated, pairs side by side: the gradient.
        dict(name="rotate_back_part", kind="rotate", tokens=8191, heads=16, d=128, rotary=64,
             interleaved=True, scaling="yarn", far=100000000, dtype="bf16", backward=True),
        # The fp32 model's gradient of one odd-sized batch.
        dict(name="rotate_back_fp32", kind="rotate", tokens=1999, heads=9, d=64, rotary=64,
             interleaved=False, scaling="linear", far=2047, dtype="fp32", backward=True),
        # One new token of each of eight conversations.
        dict(name="append_tokens", kind="append", batch=8, tokens=1, past=8000, hq=32, hkv=8, d=128,
             rows=64, dtype="bf16", interleaved=False, scaling="llama3"),
        # Ragged drafts of a batch of the fp32 model, small pages.
        dict(name="append_fp32", kind="append", batch=24, tokens=13, past=2047, hq=9, hkv=3, d=64,
             rows=16, dtype="fp32", interleaved=True, scaling="default"),
        # A chunk of a prompt, which begins inside a page.
        dict(name="append_chunk", kind="append", batch=1, tokens=8192, past=5003, hq=32, hkv=8, d=128,
             rows=64, dtype="bf16", interleaved=False, scaling="yarn"),
        # One token over a short context: the smallest attention.
        dict(name="attend_short", kind="attend", batch=1, tokens=1, past=500, hq=32, hkv=8, d=128,
             rows=64, dtype="bf16"),
        # A decode step of 32 conversations of unequal length.
        dict(name="attend_batch", kind="attend", batch=32, tokens=1, past=8001, hq=32, hkv=8, d=128,
             rows=64, dtype="bf16"),
        # One token over a 262,144-row cache.
        dict(name="attend_long", kind="attend", batch=1, tokens=1, past=262143, hq=32, hkv=8, d=128,
             rows=128, dtype="bf16"),
        # 2,048 tokens of a prompt behind 16,000 of it: the most multiplications.
        dict(name="attend_chunk", kind="attend", batch=1, tokens=2048, past=16001, hq=32, hkv=8, d=128,
             rows=64, dtype="bf16"),
        # Drafts of the fp32 model, small pages.
        dict(name="attend_fp32", kind="attend", batch=2, tokens=13, past=2047, hq=9, hkv=3, d=64,
             rows=16, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over the logarithm, odd ones among them."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("rotate", "append", "attend", "attend"))
    hq, hkv = rng.choice(HEADS)
    d = rng.choice((64, 128))
    c = dict(kind=kind, d=d, dtype=rng.choice(("bf16", "bf16", "bf16", "fp32")))
    if kind == "rotate":
        most = 32768 * 40 * 128 * 2 // (d * (4 if c["dtype"] == "fp32" else 2))
        c.update(heads=rng.choice((hq, hkv, hq + hkv)), rotary=rng.choice((d, d, d // 2, d // 4)),
                 interleaved=rng.random() < 0.5, scaling=rng.choice(sorted(SCALING)),
                 far=_log(rng, 100, 100000000), backward=rng.random() < 0.5)
        c["tokens"] = _log(rng, 1, most // c["heads"])
        return c
    c.update(batch=_log(rng, 1, 64), hq=hq, hkv=hkv, rows=rng.choice((16, 32, 64, 128)))
    if kind == "append":
        c.update(tokens=_log(rng, 1, 8192 // c["batch"]), past=_log(rng, 1, 16000 // c["batch"] + 1),
                 interleaved=rng.random() < 0.5, scaling=rng.choice(sorted(SCALING)))
        if c["dtype"] == "fp32":
            c["tokens"] = (c["tokens"] + 1) // 2
        return c
    # Query rows x keys x heads of at most the largest listed case's (a tenth in fp32), rows of
    # the caches of at most the longest's.
    most = 2048 * 17024 * 32 * 128 // (1 if c["dtype"] == "bf16" else 10)
    c["tokens"] = _log(rng, 1, max(1, min(4096, math.isqrt(most // (c["batch"] * hq * d)))))
    most = min(most // (c["batch"] * c["tokens"] * hq * d), 262144 * 8 * 128 // (c["batch"] * hkv * d))
    c["past"] = _log(rng, 1, max(1, min(262143, most - c["tokens"])))
    return c


# ------------------------------------------------------------------ inputs --

def _lens(case):
    """Rows before the new tokens: the longest first, the last about half of it."""
    n, b = case["past"], case["batch"]
    return [n - i * (n // 2) // b for i in range(b)]


def _counts(case):
    """New tokens: all of them in the even sequences, some in the odd ones (of a
    decode step: one each)."""
    n = case["tokens"]
    return [n if i % 2 == 0 else max(1, n - 1 - i % 5) for i in range(case["batch"])]


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _pow2_scale(amax):
    """The smallest power of two s with amax <= 448 s, 2^-126 at least."""
    mant, e = torch.frexp(amax)
    e = torch.where(mant <= 0.875, e - 9, e - 8).clamp(min=-126)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, -126))


def _pool(gen, case, seed):
    """Pages that hold the sequences' rows in no order, and their table."""
    b, rows, hkv, d = case["batch"], case["rows"], case["hkv"], case["d"]
    need = [(x + case["tokens"] + rows - 1) // rows for x in _lens(case)]
    width, pages = max(need), sum(need) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:sum(need)]
    table = torch.full((b, width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s = {"table": table.to(DEV)}
    for name, shape in (("k", (pages, hkv, rows, d)), ("v", (pages, hkv, d, rows))):
        x = _randn(gen, *shape)
        s[name + "_scale"] = _pow2_scale(x.abs().amax((2, 3)))
        s[name + "_pages"] = (x / s[name + "_scale"][..., None, None]).to(torch.float8_e4m3fn)
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt, d = DTYPES[case["dtype"]], case["d"]
    s = {"case": dict(case)}
    if case["kind"] == "rotate":
        n = case["tokens"]
        # A run of positions up to `far`, the places of several sequences packed one behind another.
        start = max(0, case["far"] - n)
        s["positions"] = start + (torch.arange(n, device=DEV) * 7919) % max(1, min(n, case["far"]))
        s["x"] = _randn(gen, n, case["heads"], d).to(dt)
        s["out"] = torch.empty_like(s["x"])
    else:
        b, n, hq, hkv = case["batch"], case["tokens"], case["hq"], case["hkv"]
        s.update(_pool(gen, case, seed))
        s["past"] = torch.tensor(_lens(case), dtype=torch.int32, device=DEV)
        s["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device=DEV)
        if case["kind"] == "append":
            # The columns of a fused projection.
            qkv = _randn(gen, b, n, hq + 2 * hkv, d).to(dt)
            s["q"], s["k"], s["v"] = qkv.split((hq, hkv, hkv), 2)
            s["out"] = torch.zeros(b, n, hq, d, dtype=dt, device=DEV)
        else:
            s["q"] = (2 * _randn(gen, b, n, hq, d)).to(dt)
            s["out"] = torch.empty_like(s["q"])
            s["m"] = torch.empty(b, hq, n, device=DEV)
            s["l"] = torch.empty_like(s["m"])
    if case["kind"] != "attend":
        s["inv_freq"], s["factor"] = _frequencies(case)
        s["inv_freq"] = torch.tensor(s["inv_freq"], dtype=torch.float64, device=DEV)
    if own:
        from longctx100m_amd import paged, rotary
        if case["kind"] != "attend":
            s["rotary"] = rotary.Rotary(d, 500000.0, rotary_dim=case.get("rotary", d),
                                        interleaved=case["interleaved"],
                                        scaling=SCALING[case["scaling"]], device=DEV)
        if case["kind"] != "rotate":
            s["pages"] = paged.Pages.of(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
        if case["kind"] == "attend":
            need = paged.attention_workspace_bytes(s["q"], s["pages"], s["table"])
            s["workspace"] = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------------- plain forms --

def _frequencies(case):
    """Angle of each pair per position, and what multiplies cosine and sine."""
    dim, theta, sc = case.get("rotary", case["d"]), 500000.0, SCALING[case["scaling"]]
    f = [theta ** (-2.0 * i / dim) for i in range(dim // 2)]
    if sc is None:
        return f, 1.0
    s = sc["factor"]
    if sc["type"] == "linear":
        return [x / s for x in f], 1.0
    length = sc["original_max_position_embeddings"]
    if sc["type"] == "llama3":
        lo, hi = sc["low_freq_factor"], sc["high_freq_factor"]
        ramp = [(length * x / (2 * math.pi) - lo) / (hi - lo) for x in f]  # by turns in the context
        ramp = [min(1.0, max(0.0, r)) for r in ramp]
        return [x * (r + (1 - r) / s) for x, r in zip(f, ramp)], 1.0

    def index(turns):  # the pair that makes so many turns in the original context
        return dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(theta))

    lo, hi = max(0, math.floor(index(32.0))), min(dim - 1, math.ceil(index(1.0)))
    ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3))) for i in range(dim // 2)]
    return [x * (1 - r + r / s) for x, r in zip(f, ramp)], 0.1 * math.log(s) + 1.0


def _rotated(x, positions, s, backward=False):
    """x [..., heads, head_dim] turned by positions [...], in fp32."""
    case, half = s["case"], s["inv_freq"].numel()
    angle = positions.double()[..., None] * s["inv_freq"] * (-1 if backward else 1)
    cos = (angle.cos() * s["factor"]).float()[..., None, :]
    sin = (angle.sin() * s["factor"]).float()[..., None, :]
    xf = x.float()
    if case["interleaved"]:
        a, b = xf[..., 0:2 * half:2], xf[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = xf[..., :half], xf[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, xf[..., 2 * half:]), -1)


def _blocks(case, past, counts):
    """The pages that a call writes, [batch, some]: their places in the table, and
    for each row which new token it gets and whether it holds an earlier one.
    A sequence with fewer pages than others has its last one several times."""
    rows, n = case["rows"], case["tokens"]
    j = torch.arange((n + rows - 2) // rows + 1, device=DEV)
    past, end = past.long()[:, None], (past + counts).long()[:, None]
    at = torch.minimum(past // rows + j, (end - 1) // rows)
    token = at[..., None] * rows + torch.arange(rows, device=DEV) - past[..., None]
    return at, token, token < 0, (token >= 0) & (token < (end - past)[..., None])


def _append_plain(s):
    case, past, counts = s["case"], s["past"], s["counts"]
    b, n, hq, d = s["q"].shape
    i = torch.arange(n, device=DEV)
    positions = past[:, None] + i
    there = i < counts[:, None]
    q = _rotated(s["q"], positions, s).to(s["q"].dtype)
    s["out"].copy_(torch.where(there[..., None, None], q, s["out"]))
    at, token, earlier, new = _blocks(case, past, counts)
    page = s["table"].long().gather(1, at)
    seq = torch.arange(b, device=DEV)[:, None, None]
    for name, x in (("k", _rotated(s["k"], positions, s)), ("v", s["v"].float())):
        pages, scale = s[name + "_pages"], s[name + "_scale"]
        # [batch, some, heads, rows, d]
        x = x[seq, token.clamp(0, n - 1)].transpose(2, 3)
        byte = pages.view(torch.uint8)[page]
        old = byte.view(torch.float8_e4m3fn).float()
        if name == "v":
            old, byte = old.transpose(3, 4), byte.transpose(3, 4)
        is_new, is_old = new[:, :, None, :, None], earlier[:, :, None, :, None]
        was = torch.where(earlier.any(-1)[..., None], scale[page], 2.0 ** -126)
        amax = torch.where(is_new & x.isfinite(), x.abs(), 0.0).amax((3, 4))
        now = torch.maximum(was, _pow2_scale(amax))
        x = torch.where(is_new, x / now[..., None, None], old * (was / now)[..., None, None])
        x = torch.where(x.isfinite(), x, math.nan).to(torch.float8_e4m3fn).view(torch.uint8)
        x = torch.where(is_new | is_old, x, byte)
        pages.view(torch.uint8)[page] = x.transpose(3, 4).contiguous() if name == "v" else x
        scale[page] = now
    return [s["out"], s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]]


def _rows_of(s, name):
    """A sequence's K or V, [batch, heads, rows, d] in fp32."""
    page = s["table"].long().clamp(min=0)
    x = s[name + "_pages"].view(torch.uint8)[page].view(torch.float8_e4m3fn).float()
    x = x * s[name + "_scale"][page][..., None, None]
    if name == "v":
        x = x.transpose(3, 4)
    return x.transpose(1, 2).flatten(2, 3)


def _attend_plain(s):
    q, k, v = s["q"], _rows_of(s, "k"), _rows_of(s, "v")
    b, n, hq, d = q.shape
    hkv = k.shape[1]
    g = hq // hkv
    i = torch.arange(n, device=DEV)
    last = torch.where(i < s["counts"][:, None], s["past"][:, None] + i, -1)
    seen = torch.arange(k.shape[2], device=DEV) <= last[..., None]  # [batch, tokens, rows]
    qf = q.float().view(b, n, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, n * g, d)
    sc = torch.matmul(qf, k.transpose(2, 3).contiguous()).mul_(d ** -0.5).view(b, hkv, n, g, -1)
    sc.masked_fill_(~seen[:, None, :, None], -math.inf)
    m = sc.amax(-1)
    p = sc.sub_(torch.where(m == -math.inf, 0.0, m)[..., None]).exp_()
    l = p.sum(-1)
    v = torch.where((torch.arange(k.shape[2], device=DEV) <= last.amax(-1, True))[:, None, :, None], v, 0.0)
    o = torch.matmul(p.view(b, hkv, n * g, -1), v.contiguous()).view(b, hkv, n, g, d)
    o = torch.where(l[..., None] > 0, o / l[..., None], 0.0)
    by_head = [t.transpose(2, 3).reshape(b, hq, n) for t in (m, l)]
    return [o.permute(0, 2, 1, 3, 4).reshape(b, n, hq, d).to(q.dtype), *by_head]


def run(state):
    s, c = state, state["case"]
    if own:
        from longctx100m_amd import paged, rotary
        if c["kind"] == "rotate":
            turn = rotary.rotate_backward if c["backward"] else rotary.rotate
            return [turn(s["x"], s["positions"], s["rotary"], out=s["out"])]
        if c["kind"] == "append":
            q = paged.append(s["pages"], s["table"], s["past"], s["k"], s["v"], counts=s["counts"],
                             rotary=s["rotary"], q=s["q"], q_out=s["out"])
            return [q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]]
        return list(paged.attention(s["q"], s["pages"], s["table"], s["past"], counts=s["counts"],
                                    out=s["out"], m=s["m"], l=s["l"], workspace=s["workspace"]))
    if c["kind"] == "rotate":
        return [_rotated(s["x"], s["positions"], s, c["backward"]).to(s["x"].dtype)]
    return _append_plain(s) if c["kind"] == "append" else _attend_plain(s)


def work(case):
    d, e = case["d"], 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "rotate":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * d * e + 8 * case["tokens"], "flops": 3 * n * case["rotary"]}
    hq, hkv, counts, lens = case["hq"], case["hkv"], _counts(case), _lens(case)
    if case["kind"] == "append":
        n = sum(counts)
        return {"bytes": n * d * (2 * hq * e + 2 * hkv * (e + 1)), "flops": 3 * n * d * (hq + hkv)}
    rows = sum(counts) * hq
    keys = sum(x + c for x, c in zip(lens, counts))
    pairs = sum(c * x + c * (c + 1) // 2 for x, c in zip(lens, counts))
    return {"bytes": keys * hkv * (2 * d + 8 / case["rows"]) + rows * (2 * d * e + 8),
            "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------- in 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] != "attend":
        f, factor = _frequencies(case)

    def turned(x, positions, sign):
        """x [tokens, heads, head_dim] in 64 bits, pair by pair as a complex number."""
        x = x.double().clone()
        half = len(f)
        freq = torch.tensor(f, dtype=torch.float64, device=DEV)
        turn = torch.polar(torch.full((), factor, dtype=torch.float64, device=DEV).expand(len(positions), half),
                           sign * positions.double()[:, None] * freq)[:, None]
        one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else \
            (slice(0, half), slice(half, 2 * half))
        z = torch.complex(x[..., one].contiguous(), x[..., two].contiguous()) * turn
        x[..., one], x[..., two] = z.real, z.imag
        return x

    if case["kind"] == "rotate":
        return [turned(s["x"], s["positions"], -1 if case["backward"] else 1)]
    rows, d, hq, hkv = case["rows"], case["d"], case["hq"], case["hkv"]
    sequences = list(zip(_lens(case), _counts(case), s["table"].tolist()))
    if case["kind"] == "append":
        # The values that the codes stand for, in units of their scales, before they are rounded.
        out = s["out"].double()
        pages = {x: s[x + "_pages"].double() for x in "kv"}
        pages["v"] = pages["v"].transpose(2, 3)
        for b, (past, count, table) in enumerate(sequences):
            at = torch.arange(past, past + count, device=DEV)
            out[b, :count] = turned(s["q"][b, :count], at, 1)
            new = {"k": turned(s["k"][b, :count], at, 1), "v": s["v"][b, :count].double()}
            for p in range(past // rows, (past + count - 1) // rows + 1):
                lo, hi = max(past, p * rows), min(past + count, (p + 1) * rows)
                for x in "kv":
                    block = pages[x][table[p]]
                    given = new[x][lo - past:hi - past].transpose(0, 1)
                    scale = torch.exp2(torch.ceil(torch.log2(given.abs().amax((1, 2)) / 448)))
                    if lo > p * rows:
                        was = s[x + "_scale"][table[p]].double()
                        scale = torch.maximum(scale, was)
                        block[:, :lo - p * rows] *= (was / scale)[:, None, None]
                    block[:, lo - p * rows:hi - p * rows] = given / scale[:, None, None]
        return [out, pages["k"], pages["v"].transpose(2, 3).contiguous(), None, None]
    g, n = hq // hkv, case["tokens"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    m = torch.full(s["m"].shape, -math.inf, dtype=torch.float64, device=DEV)
    l = torch.zeros(s["l"].shape, dtype=torch.float64, device=DEV)
    for b, (past, count, table) in enumerate(sequences):
        ids = torch.tensor(table[:(past + count + rows - 1) // rows], device=DEV)
        seen = torch.arange(past + count, device=DEV) <= past + torch.arange(count, device=DEV)[:, None]
        for h in range(hkv):
            k = (s["k_pages"].view(torch.uint8)[ids, h].view(torch.float8_e4m3fn).double()
                 * s["k_scale"][ids, h].double()[:, None, None]).reshape(-1, d)[:past + count]
            v = (s["v_pages"].view(torch.uint8)[ids, h].view(torch.float8_e4m3fn).double()
                 * s["v_scale"][ids, h].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:past + count]
            for e in range(g):
                sc = (s["q"][b, :count, h * g + e].double() @ k.t()) / math.sqrt(d)
                sc = sc.masked_fill_(~seen, -math.inf)
                top = sc.max(-1).values
                p = sc.sub_(top[:, None]).exp_()
                tot = p.sum(-1)
                out[b, :count, h * g + e] = (p @ v) / tot[:, None]
                m[b, h * g + e, :count], l[b, h * g + e, :count] = top, tot
    return [out, m, l]
