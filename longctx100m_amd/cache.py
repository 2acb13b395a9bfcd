"""Operators on KV caches: attention of a tree of drafted tokens, the attention
weight that cached rows receive, eviction by it, and the commit of accepted
tokens (the lc_cache_* entries of include/longctx100m_attn.h).

The reference keeps no cache (src/longctx100m/distributed_infer.py:185-219
recomputes the prefill for every token); these continue where
``ring_attention.decode`` stands: one step checks many drafted tokens, and a
cache stays within a budget.

A cache is a pair of ``[B, C, Hkv, D]`` tensors K and V of the same strides
(``layer.new_cache`` makes such), D contiguous; ``x.transpose(1, 2)`` of a
``[B, Hkv, C, D]`` tensor will do.  ``past`` (int32 ``[B]``, on the GPU) counts
the rows of each sequence that hold earlier tokens, in any order; a negative
one marks a batch slot without a sequence.  The new tokens' K and V are in rows
``past + i``, written by the caller.  ``parents`` (int32 ``[B, N]``) makes them
a tree: -1 hangs token i off the past, p < i off token p, anything else is
padding; None is a chain.

Kernels are chosen by the capacity: of a cache that is far from full, pass
``k[:, :bound]`` and ``v[:, :bound]`` to :func:`tree_attention` where a bound on the
rows, new tokens included, is known.

Everything runs on the current stream of the tensors' device, nothing
synchronises, and lengths, trees and paths are read on the device only, so a
captured graph can be replayed with others.  Calls that overlap need a
``workspace`` each (without one, a tensor of the current stream is allocated).
"""

from __future__ import annotations

import ctypes
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from .ring_attention import _dtype_code

MAX_TOKENS = _lib.LC_CACHE_MAX_TOKENS


def _call(device: int, fn, *args) -> None:
    """fn(*args, stream) with the tensors' device current, as HIP launches want it."""
    if torch._C._cuda_getDevice() == device:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc:
        _lib.check(rc)


def _buf(t, shape, dtype, device: int, name: str) -> int:
    """The address of a contiguous tensor of exactly this shape, type and device."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != shape or \
            t.get_device() != device or not t.is_contiguous():
        what = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t)
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} "
                         f"on cuda:{device}, got {what}")
    return t.data_ptr()


def _opt(t, shape, dtype, device: int, name: str) -> Optional[int]:
    return None if t is None else _buf(t, shape, dtype, device, name)


def _int32(x: int, name: str) -> int:
    """An argument of the C ABI's int32_t, which ctypes would cut to its low bits."""
    x = int(x)
    if not -2 ** 31 <= x < 2 ** 31:
        raise ValueError(f"{name} is beyond 32 bits: {x}")
    return x


def _kv(k: torch.Tensor, v: Optional[torch.Tensor]) -> int:
    """Checks a cache; returns its device."""
    for t, name in ((k, "k"), (v, "v")):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError("expected torch tensors")
        if not t.is_cuda:
            raise ValueError("tensors must live on the GPU (device pointers are passed to HIP)")
        if t.dim() != 4 or t.stride(3) != 1:
            raise ValueError(f"{name} must be a cache [batch, rows, kv_heads, head_dim] with "
                             "contiguous head_dim")
    if v is not None and (v.shape != k.shape or v.stride() != k.stride() or v.dtype is not k.dtype
                          or v.get_device() != k.get_device()):
        raise ValueError("k and v must have the same shape, strides, type and device")
    return k.get_device()


def _describe(k: torch.Tensor, tokens: int, heads_q: int, precise: bool = False) -> _lib.Cache:
    b, c, hkv, d = k.shape
    sb, sr, sh, _ = k.stride()
    if max(b, c, hkv, d, tokens, heads_q) >= 2 ** 31:  # as _int32
        raise ValueError(f"{tokens} tokens of {heads_q} heads over a cache {tuple(k.shape)}: "
                         "a size is beyond 32 bits")
    return _lib.Cache(b, tokens, c, heads_q, hkv, d, _dtype_code(k),
                      _lib.LC_FLAG_PRECISE if precise else 0,
                      # the stride of a dimension of one is never used, and may be anything
                      sb if b > 1 else 0, sr if c > 1 else 0, sh if hkv > 1 else 0)


def _queries(q: torch.Tensor, k: torch.Tensor) -> Tuple[int, int, int, int]:
    if not isinstance(q, torch.Tensor) or q.dim() != 4 or not q.is_contiguous() or \
            q.dtype is not k.dtype or q.get_device() != k.get_device():
        raise ValueError("q must be a contiguous [batch, tokens, heads, head_dim] tensor of the "
                         "cache's type and device")
    if q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError("q and the cache must agree in batch and head_dim")
    return q.shape


def tree_attention_workspace_bytes(q: torch.Tensor, k: torch.Tensor, precise: bool = False) -> int:
    """Workspace of :func:`tree_attention` for queries and caches of these shapes."""
    c = _describe(k, q.shape[1], q.shape[2], precise)
    return int(_lib.load().lc_cache_attn_workspace_bytes(c))


def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, past: torch.Tensor,
                   parents: Optional[torch.Tensor] = None, *, out: Optional[torch.Tensor] = None,
                   m: Optional[torch.Tensor] = None, l: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None, precise: bool = False):
    """Attention of N <= 256 new tokens of each sequence over its past, their
    chains of parents and themselves.

    q [B, N, Hq, D]; returns (out [B, N, Hq, D] in q's type, m, l [B, Hq, N]
    fp32), the statistics as those of ``ring_attention.fwd_shard``.  Padded
    tokens have out = 0, m = -inf, l = 0.  bf16 caches of head_dim 64 or 128 round
    the past's probabilities to bf16 for the product with v; ``precise`` takes
    bf16 inputs through the fp32-math kernels, which do not."""
    dev = _kv(k, v)
    b, n, hq, d = _queries(q, k)
    stats = (b, hq, n)
    out = torch.empty_like(q) if out is None else out
    m = torch.empty(stats, dtype=torch.float32, device=dev) if m is None else m
    l = torch.empty(stats, dtype=torch.float32, device=dev) if l is None else l
    ptrs = (_buf(past, (b,), torch.int32, dev, "past"),
            _opt(parents, (b, n), torch.int32, dev, "parents"), q.data_ptr(), k.data_ptr(),
            v.data_ptr(), _buf(out, q.shape, q.dtype, dev, "out"),
            _buf(m, stats, torch.float32, dev, "m"), _buf(l, stats, torch.float32, dev, "l"))
    lib = _lib.load()
    c = _describe(k, n, hq, precise)
    workspace = _workspace(workspace, lib.lc_cache_attn_workspace_bytes, c, dev)
    _call(dev, lib.lc_cache_attn, c, *ptrs, workspace.data_ptr(),
          workspace.numel() * workspace.element_size())
    return out, m, l


def _workspace(workspace, size, c: _lib.Cache, dev: int) -> torch.Tensor:
    if workspace is None:
        return torch.empty(max(size(c), 1), dtype=torch.uint8, device=dev)
    if not workspace.is_contiguous() or workspace.get_device() != dev:
        raise ValueError(f"workspace must be a contiguous tensor on cuda:{dev}")
    return workspace


def key_weights(q: torch.Tensor, k: torch.Tensor, past: torch.Tensor, m: torch.Tensor,
                l: torch.Tensor, weights: Optional[torch.Tensor] = None,
                parents: Optional[torch.Tensor] = None, *, out: Optional[torch.Tensor] = None,
                precise: bool = False) -> torch.Tensor:
    """The attention weight that each cached row receives from the new tokens,
    added to ``weights``: [B, Hkv, C] fp32, summed over the query heads of a KV
    head.  Query rows with m = -inf or an l that is not above 0 give nothing.

    m, l [B, Hq, N] are the statistics of the tokens' attention
    (:func:`tree_attention`, or a forward over the same rows).  Rows < past get
    weights + w (weights None: w), the tokens' own rows w, and rows behind them
    keep what ``out`` holds; without ``out`` a tensor of zeros is made.  ``out``
    may be ``weights``.  N is limited to 256 with parents only."""
    dev = _kv(k, None)
    b, n, hq, d = _queries(q, k)
    shape, stats = (b, k.shape[2], k.shape[1]), (b, hq, n)
    out = torch.zeros(shape, dtype=torch.float32, device=dev) if out is None else out
    ptrs = (_buf(past, (b,), torch.int32, dev, "past"),
            _opt(parents, (b, n), torch.int32, dev, "parents"), q.data_ptr(), k.data_ptr(),
            _buf(m, stats, torch.float32, dev, "m"), _buf(l, stats, torch.float32, dev, "l"),
            _opt(weights, shape, torch.float32, dev, "weights"),
            _buf(out, shape, torch.float32, dev, "out"))
    _call(dev, _lib.load().lc_cache_weights, _describe(k, n, hq, precise), *ptrs)
    return out


def evict_workspace_bytes(k: torch.Tensor) -> int:
    """Workspace of :func:`evict` for caches of this shape."""
    return int(_lib.load().lc_cache_evict_workspace_bytes(_describe(k, 0, 0)))


def evict(k: torch.Tensor, v: torch.Tensor, weights: torch.Tensor, lens: torch.Tensor, budget: int,
          *, sinks: int = 0, recent: int = 0, positions: Optional[torch.Tensor] = None,
          kept: Optional[torch.Tensor] = None, ends: Optional[torch.Tensor] = None,
          weights_out: Optional[torch.Tensor] = None,
          positions_out: Optional[torch.Tensor] = None, lens_out: Optional[torch.Tensor] = None,
          workspace: Optional[torch.Tensor] = None):
    """Cuts each sequence's cache to at most ``budget`` rows per KV head, in place.

    Of the ``lens`` [B] rows the ``sinks`` first and ``recent`` last positions
    stay, then the rows of the largest ``weights`` [B, Hkv, C] (ties: the lower
    row; NaN last).  Kept rows below ``budget`` stay where they are, the others
    fill the holes, so a cache that is a little over costs a few rows' copies.
    Each KV head keeps its own rows; their order is not that of the tokens.

    A later eviction of the same cache takes what this one returns, (weights,
    positions, lens): ``positions`` [B, Hkv, C] int32 and ``kept`` = lens tell
    where the rows of the earlier eviction belong, and ``ends`` [B] how many
    tokens the sequence has had (rows behind ``kept`` were appended in order,
    the last of them at position ends - 1).

    ``weights_out`` and ``positions_out`` may be their inputs; they are written up to
    lens_out.  Without them tensors of zeros are made."""
    dev = _kv(k, v)
    b, c, hkv, d = k.shape
    shape = (b, hkv, c)
    weights_out = torch.zeros(shape, dtype=torch.float32, device=dev) \
        if weights_out is None else weights_out
    positions_out = torch.zeros(shape, dtype=torch.int32, device=dev) \
        if positions_out is None else positions_out
    lens_out = torch.empty(b, dtype=torch.int32, device=dev) if lens_out is None else lens_out
    i32, f32 = torch.int32, torch.float32
    ptrs = (_buf(lens, (b,), i32, dev, "lens"), _opt(kept, (b,), i32, dev, "kept"),
            _opt(ends, (b,), i32, dev, "ends"), k.data_ptr(), v.data_ptr(),
            _buf(weights, shape, f32, dev, "weights"),
            _opt(positions, shape, i32, dev, "positions"),
            _buf(weights_out, shape, f32, dev, "weights_out"),
            _buf(positions_out, shape, i32, dev, "positions_out"),
            _buf(lens_out, (b,), i32, dev, "lens_out"))
    lib = _lib.load()
    desc = _describe(k, 0, 0)
    workspace = _workspace(workspace, lib.lc_cache_evict_workspace_bytes, desc, dev)
    _call(dev, lib.lc_cache_evict, desc, _int32(budget, "budget"), _int32(sinks, "sinks"),
          _int32(recent, "recent"), *ptrs,
          workspace.data_ptr(), workspace.numel() * workspace.element_size())
    return weights_out, positions_out, lens_out


class Layers:
    """The caches of a model's layers, of one shape and stride, checked once for
    :func:`commit`: ``Layers(ks, vs)``, or ``Layers.of(caches)`` for the (K, V)
    pairs of ``layer.new_cache``.  Holds the tensors."""

    def __init__(self, ks: Sequence[torch.Tensor], vs: Sequence[torch.Tensor]):
        self.ks, self.vs = list(ks), list(vs)
        if not self.ks or len(self.ks) != len(self.vs):
            raise ValueError("Layers needs one k and one v per layer")
        first = self.ks[0]
        _kv(first, None)
        like = (first.shape, first.stride(), first.dtype, first.get_device())
        if any((t.shape, t.stride(), t.dtype, t.get_device()) != like for t in self.ks + self.vs):
            raise ValueError("the caches must have the same shape, strides, type and device")
        if len({t.data_ptr() for t in self.ks + self.vs}) < 2 * len(self.ks):
            raise ValueError("a cache is listed twice: its rows would be moved twice")
        self._k, self._ka = _lib.ptr_array([t.data_ptr() for t in self.ks])
        self._v, self._va = _lib.ptr_array([t.data_ptr() for t in self.vs])

    @classmethod
    def of(cls, caches: Sequence[Tuple[torch.Tensor, torch.Tensor]]) -> "Layers":
        return cls([k for k, _ in caches], [v for _, v in caches])


def commit(layers: Layers, past: torch.Tensor, path: torch.Tensor, *,
           lens_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Moves the K and V rows of an accepted path of drafted tokens to the rows
    that continue the past, in every layer's cache: row past + path[j] to
    past + j.  path [B, P] int32 holds token numbers in ascending order and
    ends at the first -1.  Returns the new lengths, past + the path's length."""
    k = layers.ks[0]
    dev, b = k.get_device(), k.shape[0]
    if not isinstance(path, torch.Tensor) or path.dim() != 2:
        raise ValueError("path must be a [batch, tokens] tensor")
    lens_out = torch.empty(b, dtype=torch.int32, device=dev) if lens_out is None else lens_out
    ptrs = (_buf(past, (b,), torch.int32, dev, "past"),
            _buf(path, (b, path.shape[1]), torch.int32, dev, "path"),
            _buf(lens_out, (b,), torch.int32, dev, "lens_out"))
    _call(dev, _lib.load().lc_cache_commit, _describe(k, path.shape[1], 0), len(layers.ks),
          layers._k, layers._v, *ptrs)
    return lens_out


def tree_depths(parents: Sequence[int]) -> List[int]:
    """Depth of each node of a tree given on the host: 0 for a node that hangs off
    the past, -1 for padding.  A drafted token's position is the number of
    tokens before the tree plus its depth."""
    depths: List[int] = []
    for i, p in enumerate(parents):
        if p == -1:
            depths.append(0)
        else:
            depths.append(depths[p] + 1 if 0 <= p < i and depths[p] >= 0 else -1)
    return depths
