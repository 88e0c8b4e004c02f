"""Gated feed-forward product, forward and backward, on the tensor cores.

    h = gated_ff(x, w_gate, w_up, activation="silu")     # act(x w_gate^T) * (x w_up^T)

``x`` is (..., d), the weights are (ff, d) as ``torch.nn.Linear`` keeps them, h is
(..., ff), all bfloat16 or all float16 (under CUDA autocast they are cast to its type)
with 32-bit sums.  The activation is "silu", "gelu" or "gelu_tanh".  Both projections,
the activation and the product are one kernel; where a gradient will be taken it also
keeps both projections' results in 32 bits (8 bytes for each value of h).

Any sizes; rows that are a multiple of 16 bytes apart are read as they lie, others are
copied first.  ``GatedFeedForward`` is the block with its output projection.
"""
from __future__ import annotations

import ctypes

import torch
import torch.nn as nn

from . import _lib
from .cuda import _CODE, _on_cuda, _stream

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def _rows(t):
    """``t`` (2-D) as the kernels read it: neighbouring values of a row adjacent, rows a
    multiple of 16 bytes apart, the first on 16 bytes."""
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and \
            (t.shape[0] == 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1])):
        return t
    n = t.shape[1]
    p = torch.zeros(t.shape[0], (n + 7) // 8 * 8, dtype=t.dtype, device=t.device)
    p[:, :n] = t
    return p[:, :n]


def _pitch(t):
    """Row pitch in values; of a single row any that is allowed."""
    return t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 7) // 8 * 8


def _args(x, w_gate, w_up, act):
    a = _lib.GatedFfArgs()
    a.x, a.w_gate, a.w_up = x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr()
    a.ldx, a.ldg, a.ldu = _pitch(x), _pitch(w_gate), _pitch(w_up)
    a.rows, a.d, a.ff, a.dtype, a.act = x.shape[0], x.shape[1], w_gate.shape[0], _CODE[x.dtype], act
    return a


class _GatedFF(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act, train):
        dev, L = x.device, _lib.lib()
        rows, ff = x.shape[0], w_gate.shape[0]
        h = torch.empty(rows, ff, dtype=x.dtype, device=dev)
        saved = None
        if train:
            saved = torch.empty(int(L.scao_gated_ff_saved_bytes(rows, ff)), dtype=torch.uint8, device=dev)
        if rows:
            ins = _rows(x), _rows(w_gate), _rows(w_up)
            a = _args(*ins, act)
            a.h, a.saved = h.data_ptr(), saved.data_ptr() if train else None
            with torch.cuda.device(dev):
                _lib.check(L.scao_gated_ff_forward(ctypes.byref(a), _stream(dev)), "scao_gated_ff_forward")
        if train:
            ctx.act = act
            ctx.save_for_backward(x, w_gate, w_up, saved)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, saved = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dev, L = x.device, _lib.lib()
        rows = x.shape[0]
        new = torch.empty if rows else torch.zeros
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        dwg, dwu = (new(w_gate.shape, dtype=x.dtype, device=dev) if need_w else None for _ in range(2))
        if rows:
            ins = _rows(x), _rows(w_gate), _rows(w_up)
            a = _args(*ins, ctx.act)
            if dh.stride(1) != 1:
                dh = dh.contiguous()
            ws = torch.empty(int(L.scao_gated_ff_workspace_bytes(a.rows, a.d, a.ff)), dtype=torch.uint8,
                             device=dev)
            a.dh, a.lddh, a.saved, a.workspace = dh.data_ptr(), dh.stride(0), saved.data_ptr(), ws.data_ptr()
            a.dx = dx.data_ptr() if need_x else None
            a.dw_gate, a.dw_up = (dwg.data_ptr(), dwu.data_ptr()) if need_w else (None, None)
            with torch.cuda.device(dev):
                _lib.check(L.scao_gated_ff_backward(ctypes.byref(a), _stream(dev)), "scao_gated_ff_backward")
        return dx, dwg, dwu, None, None


def gated_ff(x, w_gate, w_up, activation="silu"):
    """act(x w_gate^T) * (x w_up^T): module docstring.  Differentiable once in x and the
    weights."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, not {activation!r}")
    if torch.is_autocast_enabled("cuda"):
        t = torch.get_autocast_dtype("cuda")
        x, w_gate, w_up = (v.to(t) if v.is_floating_point() and v.dtype != torch.float64 else v
                           for v in (x, w_gate, w_up))
    if w_gate.dim() != 2 or w_gate.shape != w_up.shape or x.dim() < 1 or x.shape[-1] != w_gate.shape[1]:
        raise ValueError(f"x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)} and w_up {tuple(w_up.shape)} "
                         "must be (..., d), (ff, d) and (ff, d)")
    if min(w_gate.shape) < 1:
        raise ValueError(f"w_gate {tuple(w_gate.shape)} has no values")
    if x.dtype not in (torch.bfloat16, torch.float16) or w_gate.dtype != x.dtype or w_up.dtype != x.dtype:
        raise TypeError("x, w_gate and w_up must all be bfloat16 or all float16 (or be cast by CUDA "
                        f"autocast), not {x.dtype}, {w_gate.dtype}, {w_up.dtype}")
    if x.numel() // x.shape[-1] >= 1 << 31 or max(w_gate.shape) >= 1 << 23:
        raise ValueError("gated_ff takes fewer than 2^31 rows and widths below 2^23")
    _on_cuda(x, w_gate, w_up)
    train = torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad)
    h = _GatedFF.apply(x.reshape(-1, x.shape[-1]), w_gate, w_up, act, train)
    return h.view(*x.shape[:-1], w_gate.shape[0])


class GatedFeedForward(nn.Module):
    """A decoder layer's gated feed-forward block, without biases:
    out(act(gate(x)) * up(x))."""

    def __init__(self, d_model, d_ff, activation="silu", device=None, dtype=None):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, not {activation!r}")
        kw = dict(bias=False, device=device, dtype=dtype)
        self.activation = activation
        self.gate = nn.Linear(d_model, d_ff, **kw)
        self.up = nn.Linear(d_model, d_ff, **kw)
        self.out = nn.Linear(d_ff, d_model, **kw)

    def forward(self, x):
        return self.out(gated_ff(x, self.gate.weight, self.up.weight, self.activation))
