"""Rotary positions for attention queries and keys, forward and backward, one launch each.

    rotary = Rotary(64)                       # values turned per head, base 10000
    q, k = rotary(q, k)                       # (batch, heads, length, head_dim)
    q, k = rotary(q, k, positions=cached)     # continue at position `cached`
    q, k = rotary(q, k, positions=ids)        # integer tensor (length) or (batch, length)

Pair j of a head at position p turns by p w_j, w_j = base^(-2j / dim); the pair is
(2j, 2j + 1) where ``interleaved``, else (j, j + dim / 2); values from ``dim`` on pass
through.  Angles are formed in 64 bits: at position p off by at most |p| 2^-55 of a turn
(base >= 1), which up to 2^29 is no more than their rounding to 24 bits for cos and sin
(2^-26 of a turn).  Any strides with neighbouring values of a head next to each other are
read as they are (views of a fused projection, (batch, length, heads, head_dim) memory).
float32, bfloat16 and float16, CUDA tensors of one device.  Forward-mode derivatives raise.
"""
from __future__ import annotations

import math
import operator
import struct
from array import array
from dataclasses import dataclass

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib
from .cuda import _CODE, _followed, _hooked, _launch

MAX_DIM = 512


@dataclass(frozen=True)
class RotaryScaling:
    """Frequencies for contexts ``factor`` times as long as the trained one.

    * ``"linear"``: every frequency divided by ``factor`` (position interpolation);
    * ``"ntk"``: base multiplied by factor^(dim / (dim - 2)), so the slowest pair is
      divided by ``factor`` and the fastest is kept;
    * ``"yarn"``: per frequency, by the turns r it makes over ``original_len``: kept where
      r >= ``fast``, divided by ``factor`` where r <= ``slow``, and the mean of both
      weighted by (r - slow) / (fast - slow) between; the turned values are multiplied by
      ``magnitude`` (0.1 ln(factor) + 1 where that is None).
    """
    kind: str
    factor: float
    original_len: int | None = None
    fast: float = 32.0
    slow: float = 1.0
    magnitude: float | None = None

    def __post_init__(self):
        if self.kind not in ("linear", "ntk", "yarn"):
            raise ValueError(f"rotary scaling must be linear, ntk or yarn, not {self.kind!r}")
        if not (math.isfinite(self.factor) and self.factor >= 1):
            raise ValueError(f"rotary scaling factor must be at least 1, not {self.factor}")
        if self.kind == "yarn":
            if self.original_len is None or self.original_len < 1:
                raise ValueError("yarn scaling needs original_len, the trained context length")
            if not 0 <= self.slow < self.fast:
                raise ValueError("yarn scaling needs 0 <= slow < fast")


def _frequencies(dim, base, s):
    """(radians per position of each pair in 64 bits, factor on the turned values)."""
    if s is not None and s.kind == "ntk":
        if dim == 2:
            raise ValueError("ntk scaling needs dim > 2")
        base = base * s.factor ** (dim / (dim - 2))
    freq = base ** (-np.arange(0, dim, 2, dtype=np.float64) / dim)
    if s is None or s.kind == "ntk":
        return freq, 1.0
    if s.kind == "linear":
        return freq / s.factor, 1.0
    turns = s.original_len * freq / (2 * math.pi)
    keep = np.clip((turns - s.slow) / (s.fast - s.slow), 0.0, 1.0)
    magnitude = 0.1 * math.log(s.factor) + 1.0 if s.magnitude is None else s.magnitude
    return freq * keep + freq / s.factor * (1 - keep), magnitude


class Rotary:
    """Rotary positions over the first ``dim`` values of each head (module docstring)."""

    def __init__(self, dim, base=10000.0, *, interleaved=False, scaling=None):
        if dim < 2 or dim % 2 or dim > MAX_DIM:
            raise ValueError(f"rotary dim must be even and within 2..{MAX_DIM}, not {dim}")
        if not (math.isfinite(base) and base > 0):
            raise ValueError(f"rotary base must be positive, not {base}")
        self.dim, self.base, self.interleaved, self.scaling = dim, float(base), bool(interleaved), scaling
        self.frequencies, self.magnitude = _frequencies(dim, self.base, scaling)
        self._turns = array("d")
        self._turns.frombytes((self.frequencies / (2 * math.pi)).tobytes())

    def __call__(self, q, k=None, positions=None):
        """The turned q, or (q, k): new tensors of the same shape, type and order in
        memory.  ``positions``: None counts from 0, an int from there, an integer tensor
        gives each token's, (length) or (batch, length)."""
        if q.dim() != 4 or q.shape[3] < self.dim or (k is not None and k.dim() != 4):
            raise ValueError("q and k must be (batch, heads, length, head_dim) with at least "
                             f"{self.dim} values a head, not {tuple(q.shape)}"
                             + ("" if k is None else f", {tuple(k.shape)}"))
        if q.dtype not in _CODE:
            raise TypeError(f"unsupported dtype {q.dtype}")
        if k is not None and (k.dtype != q.dtype or k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:]):
            raise ValueError(f"q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} must share "
                             "batch, length, head_dim and dtype")
        start = 0
        if isinstance(positions, torch.Tensor):
            if positions.dtype not in (torch.int32, torch.int64):
                raise TypeError(f"positions must be int32 or int64, not {positions.dtype}")
            if positions.dim() not in (1, 2) or positions.shape[-1] != q.shape[2] or \
                    (positions.dim() == 2 and positions.shape[0] not in (1, q.shape[0])):
                raise ValueError(f"positions {tuple(positions.shape)} do not fit q {tuple(q.shape)}")
        elif positions is not None:
            start, positions = operator.index(positions), None
            if abs(start) >= 1 << 52:
                raise ValueError(f"position {start} is out of range")
        index = q.get_device()
        if not q.is_cuda or (k is not None and k.get_device() != index) or \
                (positions is not None and positions.get_device() != index):
            raise RuntimeError("scao_b200: q, k and positions must be on one CUDA device (no CPU path)")
        if _followed() or torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            out = _Turn.apply((self, False, start, index), positions, q, k)
        else:
            out = _run(self, False, positions, start, index, (q, k))
        return out[0] if k is None else tuple(out)


# ScaoRotary, field by field: two addresses each of the inputs and the results, their
# strides (batch, head, token of both), turns and positions, the positions' strides and
# start, heads of both, eight numbers, the factor
_ARGS = struct.Struct("@4P12q2P3q10ifi")
_NONE = (0, 0, (0, 0, 0), (0, 0, 0), 0)


def _strides(t):
    """Batch, head and token strides; 0 where there is one only."""
    (b, h, n, _), (sb, sh, sn, _) = t.shape, t.stride()
    return (sb if b > 1 else 0, sh if h > 1 else 0, sn if n > 1 else 0)


def _run(rotary, inverse, positions, start, index, tensors):
    """The turned tensors (None stays None)."""
    outs, kept, parts = [], [], []
    for x in tensors:
        if x is None:
            outs.append(None)
            parts.append(_NONE)
            continue
        if x.stride(3) != 1:
            x = x.contiguous()
        y = torch.empty_like(x)
        if y.stride(3) != 1:
            y = torch.empty_like(x, memory_format=torch.contiguous_format)
        parts.append((x.data_ptr(), y.data_ptr(), _strides(x), _strides(y), x.shape[1]))
        outs.append(y)
        kept.append(x)
    if not kept:
        return outs
    x = kept[0]
    at, wide, sb, sn = 0, 0, 0, 0
    if positions is not None:
        at, wide = positions.data_ptr(), positions.dtype == torch.int64
        sn = positions.stride(-1) if positions.shape[-1] > 1 else 0
        sb = positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0
    (qs, qd, qss, qds, qh), (ks, kd, kss, kds, kh) = parts
    b, _, n, hd = x.shape
    args = _ARGS.pack(qs, ks, qd, kd, *qss, *kss, *qds, *kds, rotary._turns.buffer_info()[0], at, sb, sn,
                      start, qh, kh, _CODE[x.dtype], b, n, hd, rotary.dim, rotary.interleaved, wide, inverse,
                      rotary.magnitude, 0)
    _launch("scao_rotary", index, _lib.lib().scao_rotary, args)
    return outs


class _Turn(torch.autograd.Function):
    """The rotation, or its transpose (``inverse``), which is its gradient."""

    @staticmethod
    def forward(ctx, how, positions, q, k):
        ctx.how = how
        if positions is not None:
            ctx.places = (positions.get_device(), positions.dtype, positions.shape) if _hooked() else None
            ctx.save_for_backward(positions)
        ctx.set_materialize_grads(False)
        rotary, inverse, start, index = how
        return tuple(_run(rotary, inverse, positions, start, index, (q, k)))

    @staticmethod
    def backward(ctx, gq, gk):
        rotary, inverse, start, index = ctx.how
        saved = ctx.saved_tensors
        positions = saved[0] if saved else None
        if positions is not None and ctx.places is not None and \
                ctx.places != (positions.get_device(), positions.dtype, positions.shape):
            raise RuntimeError("rotary: the positions came back with another size, type or device")
        _, _, need_q, need_k = ctx.needs_input_grad
        gq, gk = gq if need_q else None, gk if need_k else None
        if torch.is_grad_enabled() or forward_ad._current_level >= 0:   # differentiable again
            gq, gk = _Turn.apply((rotary, not inverse, start, index), positions, gq, gk)
        else:
            gq, gk = _run(rotary, not inverse, positions, start, index, (gq, gk))
        return None, None, gq, gk
