"""A paged KV cache in 8 bits: appending tokens, their keys rotated on the way,
and attention over it (lc_paged_* of include/longctx100m_attn.h).

The reference keeps no cache (src/longctx100m/distributed_infer.py:185-219
recomputes the prefill for every token); ``layer.new_cache`` and ``cache`` keep
one sequence's, or a batch's, in rows of their own.  Here many sequences share a
pool of pages (:class:`Pages`) and take them as they grow, at half of bf16's
bytes: e4m3 codes, with a power-of-two scale for each page and KV head.

``table`` (int32 ``[B, W]``, on the GPU) lists each sequence's pages: row r of its
cache is row r % rows of page table[b, r // rows].  An entry outside the pool is
no page.  ``past`` (int32 ``[B]``) counts the rows before the call's new tokens, a
negative one marks a batch slot without a sequence; ``counts`` (int32 ``[B]``)
tells how many of the call's N tokens a sequence has (None: all).  New token i
is row and position past + i.  :func:`append` writes the new rows, after which
:func:`attention` lets each token see the rows up to its own.

Everything runs on the current stream of the tensors' device, nothing
synchronises, and tables and lengths are read on the device only, so a
captured graph can be replayed with others.  The kernels of an attention are
chosen by the table's width: where a bound on the rows is known, pass
``table[:, :bound].contiguous()``.  Calls that overlap need a ``workspace`` each
(without one, a tensor of the current stream is allocated).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .cache import _buf, _call, _opt, _workspace
from .ring_attention import _dtype_code
from .rotary import Rotary, heads_of

PAGE_ROWS = (16, 32, 64, 128)


def _check_scales(k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    scale = torch.stack((k_scale, v_scale))
    bits = scale.view(torch.int32)
    # A sign, a mantissa, or an exponent above 2^120's, which the largest finite values take.
    bad = ((bits & -0x7f800001) != 0) | (bits > 247 << 23)
    bad &= scale == scale
    if bool(bad.any()):
        which, page, head = bad.nonzero()[0].tolist()
        raise ValueError(f"{'kv'[which]}_scale[{page}, {head}] = {float(scale[which, page, head])} is no power of two "
                         "from 2^-126 to 2^120 (nor 0 or NaN, of a page that is not in use)")


class Pages:
    """The pool of a layer: ``k`` [pages, Hkv, rows, D] and ``v`` [pages, Hkv, D, rows]
    in float8_e4m3fn, ``k_scale`` and ``v_scale`` [pages, Hkv] fp32.  A row's K is its
    codes times its page's scale, which is a power of two (csrc/e4m3.h has why); those of
    pages not in use may be 0 or NaN.  The attributes cannot be set: another pool is another
    ``Pages``."""

    def __init__(self, pages: int, rows: int, kv_heads: int, head_dim: int, device="cuda"):
        def codes(*shape):
            return torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)

        self._set(codes(pages, kv_heads, rows, head_dim), codes(pages, kv_heads, head_dim, rows),
                  torch.zeros(pages, kv_heads, device=device), torch.zeros(pages, kv_heads, device=device))

    @classmethod
    def of(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> "Pages":
        """A pool in tensors that are there already.  Scales of another kind, such as amax /
        448, are refused: the kernels take their exponents alone.  (This waits for the GPU,
        and is left out while a graph is captured.)"""
        p = cls.__new__(cls)
        p._set(k, v, k_scale, v_scale)
        if not (k.is_cuda and torch.cuda.is_current_stream_capturing()):
            _check_scales(k_scale, v_scale)
        return p

    def _set(self, k, v, k_scale, v_scale):
        for t in (k, v, k_scale, v_scale):
            if not isinstance(t, torch.Tensor) or not t.is_contiguous():
                raise ValueError("a pool is contiguous tensors")
        if k.dim() != 4 or v.dim() != 4 or any(t.dtype is not torch.float8_e4m3fn for t in (k, v)):
            raise ValueError("pages must be float8_e4m3fn tensors [pages, kv_heads, rows, head_dim] and "
                             "[pages, kv_heads, head_dim, rows]")
        n, h, rows, d = k.shape
        if v.shape != (n, h, d, rows) or any(t.shape != (n, h) or t.dtype is not torch.float32
                                             for t in (k_scale, v_scale)):
            raise ValueError("v must be [pages, kv_heads, head_dim, rows], and the scales fp32 [pages, kv_heads]")
        if any(t.device != k.device for t in (v, k_scale, v_scale)):
            raise ValueError("a pool lives on one device")
        if rows not in PAGE_ROWS:
            raise ValueError(f"a page has {PAGE_ROWS} rows, got {rows}")
        if max(n, h, d) >= 2 ** 31 or min(n, h, d) == 0:
            raise ValueError(f"a pool of shape {tuple(k.shape)}")
        self.__dict__.update(k=k, v=v, k_scale=k_scale, v_scale=v_scale, count=n, kv_heads=h, rows=rows, head_dim=d)

    def __setattr__(self, name, value):  # the checks above hold for these tensors
        raise AttributeError(f"{name} of a pool cannot be set: Pages.of makes a pool of other tensors")

    # Asked of the tensors at every call: a copied or unpickled pool has its own.
    @property
    def _ptrs(self) -> Tuple[int, int, int, int]:
        return self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr()

    def device(self) -> int:
        device = self.k.get_device()
        if device < 0:
            raise ValueError("tensors must live on the GPU (device pointers are passed to HIP)")
        return device


def _describe(pages: Pages, table: torch.Tensor, b: int, n: int, heads_q: int, dtype: int) -> _lib.Paged:
    if not isinstance(table, torch.Tensor) or table.dim() != 2:
        raise ValueError("table must be a [batch, pages of a sequence] tensor")
    width = table.shape[1]
    if max(b, n, heads_q, width) >= 2 ** 31:
        raise ValueError(f"{n} tokens of {heads_q} heads in {b} sequences: a size is beyond 32 bits")
    return _lib.Paged(b, n, heads_q, pages.kv_heads, pages.head_dim, dtype, pages.count, pages.rows, width, 0)


def _lengths(table, past, counts, desc: _lib.Paged, dev: int) -> Tuple[int, int, Optional[int]]:
    b = (desc.batch,)
    return (_buf(table, (desc.batch, desc.table_width), torch.int32, dev, "table"),
            _buf(past, b, torch.int32, dev, "past"), _opt(counts, b, torch.int32, dev, "counts"))


def _rows(t, shape: Tuple[int, ...], dtype, dev: int, name: str) -> _lib.Rows:
    if not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype is not dtype or t.get_device() != dev:
        raise ValueError(f"{name} must be a {dtype} tensor {shape} on cuda:{dev}")
    return heads_of(t, shape, name)


def append(pages: Pages, table: torch.Tensor, past: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
           counts: Optional[torch.Tensor] = None, rotary: Optional[Rotary] = None,
           q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Appends the new tokens' k and v [B, N, Hkv, D] (bf16 or fp32, any strides with
    contiguous D, e.g. columns of a fused projection) to the pages, k rotated to
    positions past + i by ``rotary`` (whose rotary_dim is a multiple of 16 here).  With
    ``q`` [B, N, Hq, D] the tokens' queries are rotated too and returned (``q_out``,
    contiguous, may be q; padded tokens' rows in it are left alone, and are not written
    in one made here).  No gradients: they are lost here.

    The pages that new rows lie in must be their sequence's alone.  Their scales
    rise as needed, which rounds codes of earlier rows in them again: to the
    same value, but for values below 2^-6 of the scale.  Infinities and NaN are
    stored as NaN."""
    dev = pages.device()
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise ValueError("k must be a [batch, tokens, heads, head_dim] tensor")
    b, n = k.shape[:2]
    dtype, d = k.dtype, pages.head_dim
    shape = (b, n, pages.kv_heads, d)
    ks, vs = _rows(k, shape, dtype, dev, "k"), _rows(v, shape, dtype, dev, "v")
    hq = 0
    qs = qp = qo = None
    if q is not None:
        if not isinstance(q, torch.Tensor) or q.dim() != 4:
            raise ValueError("q must be a [batch, tokens, heads, head_dim] tensor")
        hq = q.shape[2]
        shape = (b, n, hq, d)
        qs = _rows(q, shape, dtype, dev, "q")
        if q_out is None:
            q_out = torch.empty(shape, dtype=dtype, device=q.device)
        qp, qo = q.data_ptr(), _buf(q_out, shape, dtype, dev, "q_out")
    elif q_out is not None:
        raise ValueError("q_out comes with q")
    desc = _describe(pages, table, b, n, hq, _dtype_code(k))
    if b == 0 or n == 0:
        return q_out
    _call(dev, _lib.load().lc_paged_append, desc, rotary.on(dev) if rotary is not None else None,
          *_lengths(table, past, counts, desc, dev), qp, qs, qo, k.data_ptr(), ks, v.data_ptr(), vs, *pages._ptrs)
    return q_out


def _queries(q, pages: Pages, dev: int) -> None:
    if not isinstance(q, torch.Tensor) or q.dim() != 4 or not q.is_contiguous() or q.get_device() != dev:
        raise ValueError(f"q must be a contiguous [batch, tokens, heads, head_dim] tensor on cuda:{dev}")
    if q.shape[3] != pages.head_dim:
        raise ValueError("q and the pages must agree in head_dim")


def attention_workspace_bytes(q: torch.Tensor, pages: Pages, table: torch.Tensor) -> int:
    """Workspace of :func:`attention` for queries, pools and tables of these shapes."""
    _queries(q, pages, pages.device())
    b, n, hq, _ = q.shape
    return int(_lib.load().lc_paged_attn_workspace_bytes(_describe(pages, table, b, n, hq, _dtype_code(q))))


def attention(q: torch.Tensor, pages: Pages, table: torch.Tensor, past: torch.Tensor, *,
              counts: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
              m: Optional[torch.Tensor] = None, l: Optional[torch.Tensor] = None,
              workspace: Optional[torch.Tensor] = None):
    """Attention of N new tokens of each sequence, appended before, over the rows up
    to their own: one token, drafts, or a whole prompt.

    q [B, N, Hq, D] (bf16 or fp32); returns (out [B, N, Hq, D] in q's type, m, l
    [B, Hq, N] fp32), the statistics as those of ``ring_attention.fwd_shard``.
    Padded tokens, and those that see no row, have out = 0, m = -inf, l = 0.
    bf16 queries round the probabilities to bf16 for the product with v, fp32
    ones do not."""
    dev = pages.device()
    _queries(q, pages, dev)
    b, n, hq, _ = q.shape
    stats = (b, hq, n)
    out = torch.empty_like(q) if out is None else out
    m = torch.empty(stats, dtype=torch.float32, device=dev) if m is None else m
    l = torch.empty(stats, dtype=torch.float32, device=dev) if l is None else l
    ptrs = (q.data_ptr(), *pages._ptrs, _buf(out, q.shape, q.dtype, dev, "out"),
            _buf(m, stats, torch.float32, dev, "m"), _buf(l, stats, torch.float32, dev, "l"))
    desc = _describe(pages, table, b, n, hq, _dtype_code(q))
    if b == 0 or n == 0:
        return out, m, l
    lib = _lib.load()
    workspace = _workspace(workspace, lib.lc_paged_attn_workspace_bytes, desc, dev)
    _call(dev, lib.lc_paged_attn, desc, *_lengths(table, past, counts, desc, dev), *ptrs, workspace.data_ptr(),
          workspace.numel() * workspace.element_size())
    return out, m, l
