"""Gated feed-forward product, forward and backward, on the tensor cores.

    h = gated_ff(x, w_gate, w_up, activation="silu")     # act(x w_gate^T) * (x w_up^T)

``x`` is (..., d), the weights are (ff, d) as ``torch.nn.Linear`` keeps them, h is
(..., ff), all bfloat16 or all float16 (under CUDA autocast they are cast to its type)
with 32-bit sums; the weights' gradients have the weights' type (under autocast they are
rounded to its type first and widened).  float32 without autocast raises.  The activation is "silu", "gelu" or "gelu_tanh".  Both projections,
the activation and the product are one kernel; where a gradient will be taken it also
keeps both projections' results in 24 bits (6 bytes for each value of h, in whole blocks
of 128 rows x 128 columns: one row keeps what 128 do).

Any sizes; rows that are a multiple of 16 bytes apart are read as they lie, others are
copied first.  ``GatedFeedForward`` is the block with its output projection.
"""
from __future__ import annotations

import operator
import struct
from array import array

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _lib
from .cuda import _CODE, _followed, _hooked, _launch

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


_DTYPE, _DEVICE = operator.attrgetter("dtype"), torch.Tensor.get_device

# ScaoGatedFf: ten addresses, four row pitches, six numbers
_ARGS = struct.Struct("@10P4q6i")


def _operands(tensors):
    """The 2-D ``tensors`` as the kernels read them (neighbouring values of a row adjacent,
    rows a multiple of 16 bytes apart, the first on 16 bytes; copies, in one launch,
    where they lie otherwise): ([tensor, address, row pitch, whether a copy] of each,
    whether any was copied)."""
    out, table, kept = [], [], []
    for t in tensors:
        n, p = t.shape[1], t.data_ptr()
        if p & 15 == 0:
            if n & 7 == 0 and t.is_contiguous():
                out.append((t, p, n, False))
                continue
            if t.stride(1) == 1 or n == 1:
                pitch = t.stride(0) if t.shape[0] > 1 else (n + 7) & ~7
                if pitch & 7 == 0 and pitch >= n:
                    out.append((t, p, pitch, False))
                    continue
        if t.stride(1) != 1:
            t = t.contiguous()
            kept.append(t)
        wide = t.new_empty((t.shape[0], (n + 63) & ~63))      # rows of whole 128-byte lines
        table += (t.data_ptr(), wide.data_ptr(), t.shape[0], n, t.stride(0))
        out.append((wide, wide.data_ptr(), wide.shape[1], True))
    if table:
        table = array("q", table)
        _launch("scao_gated_ff_pack", tensors[0].get_device(), _lib.lib().scao_gated_ff_pack,
                table.buffer_info()[0], len(table) // 5)
    return out, bool(table)


def _forward(x, w_gate, w_up, act, train):
    """(h, what the gradient reads or None, the copy of each operand or None, () without any)."""
    L, rows, (ff, d) = _lib.lib(), x.shape[0], w_gate.shape
    h = x.new_empty((rows, ff))
    saved, copies = None, ()
    if train:
        saved = x.new_empty(L.scao_gated_ff_saved_bytes(rows, ff) >> 1)     # 16-bit places
    if rows:
        ins, copied = _operands((x, w_gate, w_up))
        args = _ARGS.pack(ins[0][1], ins[1][1], ins[2][1], h.data_ptr(), saved.data_ptr() if train else 0,
                          0, 0, 0, 0, 0, ins[0][2], ins[1][2], ins[2][2], 0,
                          rows, d, ff, _CODE[x.dtype], act, 0)
        _launch("scao_gated_ff_forward", x.get_device(), L.scao_gated_ff_forward, args)
        if copied and train:
            copies = [i[0] if i[3] else None for i in ins]
    return h, saved, copies


def _from_hooks(dh, ins, saved, places, copies):
    """``saved`` where the kernels can read it; raises where hooks handed back something else
    than was saved."""
    (x, w_gate, w_up), kept = ins, (dh, *ins, saved)
    if copies:
        kept += tuple(c for c in copies if c is not None)
    good = len(set(map(_DTYPE, kept))) == 1 == len(set(map(_DEVICE, kept))) and saved.numel() == places and \
        dh.shape == (x.shape[0], w_gate.shape[0]) and w_gate.shape == w_up.shape and x.shape[1] == w_gate.shape[1]
    for t, c in zip(ins, copies):
        good = good and (c is None or c.shape == (t.shape[0], (t.shape[1] + 63) & ~63))
    if not good:
        raise RuntimeError("gated_ff: a saved tensor came back with another size, type or device")
    return saved.clone(memory_format=torch.contiguous_format) \
        if saved.data_ptr() & 15 or not saved.is_contiguous() else saved


def _backward(x, w_gate, w_up, saved, dh, act, need_x, need_w, copies):
    """(dx, dw_gate, dw_up), None where not needed."""
    L, rows, (ff, d) = _lib.lib(), x.shape[0], w_gate.shape
    dx = x.new_empty((rows, d)) if need_x else None
    new = x.new_empty if rows else x.new_zeros
    dwg, dwu = (new((ff, d)), new((ff, d))) if need_w else (None, None)
    if rows:
        ins = (x, w_gate, w_up)
        if copies:
            ins = [t if c is None else c for t, c in zip(ins, copies)]
        ins, _ = _operands(ins)
        if dh.stride(1) != 1:
            dh = dh.contiguous()
        ws = x.new_empty((L.scao_gated_ff_workspace_bytes(rows, d, ff, need_x | need_w << 1) + 1) >> 1)
        at = [0 if t is None else t.data_ptr() for t in (dx, dwg, dwu)]
        args = _ARGS.pack(ins[0][1], ins[1][1], ins[2][1], 0, saved.data_ptr(), dh.data_ptr(), *at,
                          ws.data_ptr(), ins[0][2], ins[1][2], ins[2][2], dh.stride(0),
                          rows, d, ff, _CODE[x.dtype], act, 0)
        _launch("scao_gated_ff_backward", x.get_device(), L.scao_gated_ff_backward, args)
    return dx, dwg, dwu


class _Once(torch.autograd.Function):
    """A gradient taken under create_graph: it depends on ``sources``, and asking for
    that dependence raises instead of passing for a constant."""

    @staticmethod
    def forward(ctx, grad, *sources):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("gated_ff is differentiable once: its gradient has no gradient")


class _GatedFF(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act):
        h, saved, copies = _forward(x, w_gate, w_up, act, True)
        ctx.act, ctx.hooked = act, _hooked()
        ctx.save_for_backward(x, w_gate, w_up, saved, *copies)
        return h

    @staticmethod
    def backward(ctx, dh):
        need, (x, w_gate, w_up, saved, *copies) = ctx.needs_input_grad, ctx.saved_tensors
        if ctx.hooked:
            places = _lib.lib().scao_gated_ff_saved_bytes(dh.shape[0], dh.shape[1]) >> 1
            saved = _from_hooks(dh, (x, w_gate, w_up), saved, places, copies)
        grads = _backward(x, w_gate, w_up, saved, dh, ctx.act, need[0], need[1] or need[2], copies)
        if torch.is_grad_enabled() or forward_ad._current_level >= 0:
            grads = [None if g is None else _Once.apply(g, x, w_gate, w_up, dh) for g in grads]
        return *grads, None


def gated_ff(x, w_gate, w_up, activation="silu"):
    """act(x w_gate^T) * (x w_up^T): module docstring.  Differentiable once in x and the
    weights; forward-mode derivatives raise."""
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
    if not x.is_cuda or w_gate.get_device() != x.get_device() or w_up.get_device() != x.get_device():
        raise RuntimeError("scao_b200: x, w_gate and w_up must be on one CUDA device (no CPU path)")
    flat = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if _followed() or torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        h = _GatedFF.apply(flat, w_gate, w_up, act)
    else:
        h = _forward(flat, w_gate, w_up, act, False)[0]
    return h if x.dim() == 2 else h.view(*x.shape[:-1], w_gate.shape[0])


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
