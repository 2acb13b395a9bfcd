"""Rotary positions at any positions, forward and backward (lc_rotary_* of
include/longctx100m_layer.h).

``layer.rope_apply`` is the reference's rotation
(rust/longctx100m-model/src/rope.rs:101-127): whole heads, pairs half a head
apart, a table of consecutive positions whose angles are fp32 products, off by
a radian at 10^7.  Here

  * positions are given (any int64, in any order), or follow from a first one;
  * pairs lie half the rotated part apart, or side by side (``interleaved``);
  * the first ``rotary_dim`` dims of a head turn, the others stay;
  * angles are 64-bit fractions of a turn: right to 2^-38 of a turn at 10^8;
  * the backward pass is there, and autograd takes it.

A :class:`Rotary` holds what a model's rotation is; kernels run on the current
stream of the tensors' device and nothing synchronises.
"""

from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .cache import _call
from .ring_attention import _dtype_code


def frequencies(rotary_dim: int, theta: float, scaling: Optional[dict] = None) -> Tuple[List[float], float]:
    """(inverse frequencies, factor of cos and sin) of a config's rope_theta and
    rope_scaling, in 64 bits.

    f_i = theta^(-2i / rotary_dim).  ``scaling`` types, with s = ``factor``:
      linear  f / s;
      llama3  f / s for pairs that make fewer than low_freq_factor turns in
              original_max_position_embeddings, f for more than
              high_freq_factor, linear in the turns between;
      yarn    f for pairs that make more than beta_fast (32) turns in
              original_max_position_embeddings, f / s for fewer than beta_slow
              (1), linear in the pair's index between, and a factor of
              attention_factor (0.1 ln s + 1) (YaRN, Peng et al. 2023).
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not theta > 1.0:  # (NaN too)
        raise ValueError(f"theta must be above 1, got {theta}")
    f = [theta ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if not scaling:
        return f, 1.0
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "default":
        return f, 1.0
    s = float(scaling.get("factor", 1.0))
    if not s > 0.0:
        raise ValueError(f"the scaling factor must be positive, got {s}")
    if kind == "linear":
        return [x / s for x in f], 1.0
    if kind not in ("llama3", "yarn"):
        raise ValueError(f"unsupported RoPE type {kind!r}")
    if "original_max_position_embeddings" not in scaling:
        raise ValueError(f"{kind} RoPE needs the original context length")
    length = float(scaling["original_max_position_embeddings"])
    if not length > 0.0:
        raise ValueError(f"the original context length must be positive, got {length}")
    if kind == "llama3":
        if "low_freq_factor" not in scaling or "high_freq_factor" not in scaling:
            raise ValueError("llama3 RoPE needs low/high frequency factors")
        lo, hi = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not hi > lo:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        keep = [(length * x / (2 * math.pi) - lo) / (hi - lo) for x in f]
        keep = [min(1.0, max(0.0, x)) for x in keep]
        return [x * k + x / s * (1.0 - k) for x, k in zip(f, keep)], 1.0
    fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
    if not fast > slow > 0.0:
        raise ValueError("beta_fast must be above beta_slow, and that above 0")

    def pair_of(turns: float) -> float:  # length f_i = 2 pi turns
        return rotary_dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(theta))

    lo = max(0, math.floor(pair_of(fast)))
    hi = min(rotary_dim - 1, math.ceil(pair_of(slow)))
    keep = [min(1.0, max(0.0, 1.0 - (i - lo) / max(hi - lo, 1e-3))) for i in range(len(f))]
    given = scaling.get("attention_factor")
    factor = float(given) if given is not None else 0.1 * math.log(s) + 1.0 if s > 1.0 else 1.0
    return [x * k + x / s * (1.0 - k) for x, k in zip(f, keep)], factor


class Rotary:
    """A model's rotation: ``Rotary(head_dim, theta)`` with ``rotary_dim`` (all of the
    head), ``interleaved`` pairs and ``scaling`` as :func:`frequencies` takes it, or
    with ``inv_freq`` (and ``factor``) given instead.  Keeps the frequencies on
    ``device``.  The attributes cannot be set: another rotation is another ``Rotary``."""

    def __init__(self, head_dim: int, theta: float = 10000.0, *, rotary_dim: Optional[int] = None,
                 interleaved: bool = False, scaling: Optional[dict] = None,
                 inv_freq: Optional[Sequence[float]] = None, factor: Optional[float] = None, device="cuda"):
        head_dim = int(head_dim)
        if inv_freq is not None:
            if scaling is not None:
                raise ValueError("inv_freq comes in place of scaling")
            inv_freq, own = [float(x) for x in inv_freq], 1.0
            if rotary_dim is not None and rotary_dim != 2 * len(inv_freq):
                raise ValueError("inv_freq needs rotary_dim / 2 values")
            rotary_dim = 2 * len(inv_freq)
        else:
            rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
            inv_freq, own = frequencies(rotary_dim, float(theta), scaling)
        if not 0 < head_dim <= 256 or not 0 < rotary_dim <= head_dim:
            raise ValueError(f"rotary_dim ({rotary_dim}) must be positive and at most head_dim "
                             f"({head_dim}), and that at most 256")
        n = rotary_dim // 2
        turns = (ctypes.c_uint64 * n)()
        _lib.check(_lib.load().lc_rotary_turns(n, (ctypes.c_double * n)(*inv_freq), turns))
        # (two's complement: torch has no arithmetic on uint64, nor needs any here)
        host = torch.tensor([x - (x >> 63 << 64) for x in turns], dtype=torch.int64)
        self.__dict__.update(head_dim=head_dim, rotary_dim=rotary_dim, interleaved=bool(interleaved),
                             inv_freq=inv_freq, factor=own if factor is None else float(factor),
                             turns=host.to(device))
        self._describe()

    def _describe(self) -> None:
        self.__dict__["_c"] = _lib.Rotary(self.head_dim, self.rotary_dim, self.interleaved, self.factor)

    # A copy has a description of its own (which could not be copied: it holds a pointer).
    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k != "_c"}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._describe()

    def __setattr__(self, name, value):  # turns follow from the rest
        raise AttributeError(f"{name} of a rotation cannot be set: make another Rotary")

    @classmethod
    def of(cls, rope: _lib.Rope, device="cuda") -> "Rotary":
        """The rotation of ``layer.rope_params``, with the reference's fp32 frequencies
        (rope.rs:15-99): what a model's RoPE table holds, but for the table's fp32
        angles.  The reference's llama3 profile takes every wavelength as 2 pi
        (rope.rs:70), so ``Rotary(.., scaling=..)`` has other frequencies there."""
        n = rope.head_dim // 2
        inv, cos_factor = (ctypes.c_float * max(n, 1))(), ctypes.c_float()
        _lib.check(_lib.load().lc_rope_inv_freq(ctypes.byref(rope), ctypes.addressof(inv),
                                                ctypes.addressof(cos_factor)))
        if cos_factor.value != 1.0:
            raise ValueError("the reference's attention_factor scales cos alone: not a rotation")
        by = rope.factor if rope.type == 1 else 1.0
        return cls(rope.head_dim, inv_freq=[x / by for x in inv], device=device)

    def on(self, device: int) -> _lib.Rotary:
        """The rotation as the C ABI takes it, for tensors of that GPU."""
        if self.turns.get_device() != device:
            raise ValueError(f"the rotary frequencies live on {self.turns.device}, not on cuda:{device}")
        self._c.turns = self.turns.data_ptr()
        return self._c


def heads_of(t: torch.Tensor, shape: Sequence[int], name: str) -> _lib.Rows:
    """Strides of a tensor of this shape, [batch, tokens, heads, head_dim] or [tokens,
    heads, head_dim], for the C ABI."""
    # The stride of a dimension of one is never used, and may be anything.
    if len(shape) == 4:
        b, n, h, d = shape
        sb, sn, sh, sd = t.stride()
        rows = _lib.Rows(sb if b > 1 else 0, sn if n > 1 else 0, sh if h > 1 else 0)
    else:
        n, h, d = shape
        sn, sh, sd = t.stride()
        rows = _lib.Rows(0, sn if n > 1 else 0, sh if h > 1 else 0)
    if sd != 1 and d > 1:
        raise ValueError(f"{name} must have contiguous head_dim")
    return rows


def _turn(x: torch.Tensor, positions: Union[torch.Tensor, int], rotary: Rotary, out: Optional[torch.Tensor],
          inverse: int) -> torch.Tensor:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("tensors must live on the GPU (device pointers are passed to HIP)")
    shape, dev = x.shape, x.get_device()
    if len(shape) not in (3, 4) or shape[-1] != rotary.head_dim:
        raise ValueError(f"rows must be [(batch,) tokens, heads, {rotary.head_dim}], got {tuple(shape)}")
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
    elif not isinstance(out, torch.Tensor) or out.shape != shape or out.dtype is not x.dtype or \
            out.get_device() != dev:
        raise ValueError("out must have the shape, type and device of the rows")
    b, n, h = (1, shape[0], shape[1]) if len(shape) == 3 else shape[:3]
    if isinstance(positions, torch.Tensor):
        if positions.dtype is not torch.int64 or positions.shape != shape[:-2] or \
                positions.get_device() != dev or not positions.is_contiguous():
            raise ValueError(f"positions must be a contiguous int64 tensor {tuple(shape[:-2])} on cuda:{dev}, "
                             "or the first one's number")
        at, pos0 = positions.data_ptr(), 0
    else:
        at, pos0 = None, int(positions)
        if not -2 ** 62 <= pos0 < 2 ** 62:
            raise ValueError(f"the first position is beyond 62 bits: {pos0}")
    if max(b, n, h) >= 2 ** 31:
        raise ValueError(f"a size of {tuple(shape)} is beyond 32 bits")
    if h == 0:
        return out
    _call(dev, _lib.load().lc_rotary_apply, rotary.on(dev), _dtype_code(x), b, n, h, at, pos0, inverse,
          x.data_ptr(), heads_of(x, shape, "x"), out.data_ptr(), heads_of(out, shape, "out"))
    return out


class _Rotate(torch.autograd.Function):
    """The rotation, or its transpose (inverse = 1), each of which is the other's gradient."""

    @staticmethod
    def forward(ctx, x, positions, rotary, inverse):
        at = isinstance(positions, torch.Tensor)
        ctx.save_for_backward(*[positions] if at else [])
        ctx.args = None if at else positions, rotary, inverse
        return _turn(x, positions, rotary, None, inverse)

    @staticmethod
    def backward(ctx, grad):
        first, rotary, inverse = ctx.args
        positions = ctx.saved_tensors[0] if first is None else first
        if grad.stride(-1) != 1:  # (of a sum: one element for all)
            grad = grad.contiguous()
        return _Rotate.apply(grad, positions, rotary, 1 - inverse), None, None, None


def _with_graph(x, positions, rotary, out, inverse: int) -> torch.Tensor:
    if out is not None:
        raise ValueError("rows that need a gradient are not rotated into out: leave it away, or use torch.no_grad()")
    return _Rotate.apply(x, positions, rotary, inverse)


def rotate(x: torch.Tensor, positions: Union[torch.Tensor, int], rotary: Rotary, *,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turns the rows x [(batch,) tokens, heads, head_dim] (bf16 or fp32, any strides
    with contiguous head_dim) to ``positions``: int64 [(batch,) tokens] on the GPU,
    or the number of each sequence's first one.  ``out`` may be x.  Differentiable in x
    where no ``out`` is given."""
    if getattr(x, "requires_grad", False) and torch.is_grad_enabled():
        return _with_graph(x, positions, rotary, out, 0)
    return _turn(x, positions, rotary, out, 0)


def rotate_backward(grad: torch.Tensor, positions: Union[torch.Tensor, int], rotary: Rotary, *,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of :func:`rotate`'s x from that of its result (which autograd calls by
    itself)."""
    if getattr(grad, "requires_grad", False) and torch.is_grad_enabled():
        return _with_graph(grad, positions, rotary, out, 1)
    return _turn(grad, positions, rotary, out, 1)
