"""Global gradient norm and clipping, over any number of gradients in two launches.

``clip_grad_norm_``, ``get_total_norm`` and ``clip_grads_with_norm_`` do what the
functions of the same names in ``torch.nn.utils`` do and return the norm as a float32
scalar on the gradients' device; nothing waits for the GPU.  Refused, where those take it:
norms of other orders than 1, 2 and inf, float64 and sparse gradients, gradients on the
CPU or on several devices, gradients that share memory, a negative ``max_norm``, and the
argument ``foreach``.  Gradients may mix float32, bfloat16 and float16, sizes and alignments.
Sums are held in 64 bits over the whole range of float32, the same inputs give the
same bits, and each value is scaled in 32 bits and rounded to its type.  Gradients within the threshold are
not written (strided ones that do not fill a range of memory are: with their own values).  CUDA tensors of one device only; errors raise.
"""
from __future__ import annotations

import math
from array import array
from operator import attrgetter

import torch
from torch._C import _is_tracing
from torch.autograd import forward_ad

from . import _lib
from .cuda import _CODE, _launch

_KIND = {1.0: 0, 2.0: 1, math.inf: 2}
_DTYPES = set(_CODE)
SHARED = "two gradients share memory: each can be scaled only once"
_DTYPE, _LAYOUT, _GRAD = attrgetter("dtype"), attrgetter("layout"), attrgetter("grad")


def _layout(t):
    """(dense, overlapping) of a strided tensor: its values fill a range of memory /
    two of its elements may share an address."""
    expected, dense = 1, True
    for stride, size in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n != 1):
        if stride < expected:
            return False, True
        dense = dense and stride == expected
        expected += stride * (size - 1)
    return dense, False


def _places(t):
    """Where a tensor's bytes lie: (first address, [(count, stride in bytes)] from the widest
    stride on, bytes of an unbroken run, bytes from the first to behind the last)."""
    size = run = t.element_size()
    steps = []
    for stride, n in sorted((st * size, n) for n, st in zip(t.shape, t.stride()) if n != 1):
        if not steps and stride == run:
            run *= n
        else:
            steps.append((n, stride))
    return t.data_ptr(), steps[::-1], run, run + sum((n - 1) * st for n, st in steps)


def _meet(p, a, run_a, span_a, q, b, run_b, span_b):
    """Whether two tensors, neither of which overlaps itself, share a byte (``_places`` of
    both).  A step's span is at most its stride, so with equal strides only the neighbouring
    shifts of one against the other can meet; else the wider steps are taken one by one, where
    they reach the other tensor."""
    if p + span_a <= q or q + span_b <= p:
        return False
    if not a and not b:
        return True
    if not a or (b and b[0][1] > a[0][1]):
        p, a, run_a, span_a, q, b, run_b, span_b = q, b, run_b, span_b, p, a, run_a, span_a
    n, stride = a[0]
    a, span_a = a[1:], span_a - (n - 1) * stride
    low, high = 0, n - 1
    if b and b[0][1] == stride:
        m, b, span_b = b[0][0], b[1:], span_b - (b[0][0] - 1) * stride
        low -= m - 1
    # steps i for which [p + i stride, + span_a) meets [q, q + span_b)
    low, high = max(low, (q - p - span_a) // stride + 1), min(high, (q + span_b - p - 1) // stride)
    return any(_meet(p + i * stride, a, run_a, span_a, q, b, run_b, span_b) for i in range(low, high + 1))


def _refuse_sharing(tensors, strided):
    """Raises where one of the ``strided`` tensors (by number) shares memory with another."""
    places = sorted(((*_places(t), i in strided) for i, t in enumerate(tensors) if t.numel()),
                    key=lambda x: x[0])
    near = []
    for p, steps, run, span, loose in places:
        near = [x for x in near if x[0] + x[3] > p]
        if any((loose or x[4]) and _meet(*x[:4], p, steps, run, span) for x in near):
            raise ValueError(SHARED)
        near.append((p, steps, run, span, loose))


def _refuse(tensors):
    """Raises for the first tensor that is not a strided one of a supported type on the
    device of the others."""
    for t in tensors:
        if t.layout != torch.strided:
            raise TypeError(f"unsupported gradient layout {t.layout}")
        if t.dtype not in _CODE:
            raise TypeError(f"unsupported gradient dtype {t.dtype}")
        if t.device != tensors[0].device:
            raise ValueError("the gradients must be on one device, not "
                             f"{tensors[0].device} and {t.device}")


def _table(tensors, write):
    """(rows of the C table, tensors behind them, [(strided gradient, its packed copy)],
    device number).  Strided gradients that are not dense are packed for the call; tensors
    that will be written must not share memory."""
    n, index = len(tensors), tensors[0].get_device()
    if _is_tracing():
        raise RuntimeError("the gradients' norm and clipping cannot be traced")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("gradients with forward-mode tangents are not clipped")
    get, dtypes = torch.Tensor, set(map(_DTYPE, tensors))
    if index < 0 or not dtypes <= _DTYPES or set(map(get.get_device, tensors)) != {index} or \
            set(map(_LAYOUT, tensors)) != {torch.strided}:
        _refuse(tensors)
    codes = [_CODE[dtypes.pop()]] * n if len(dtypes) == 1 else [_CODE[t.dtype] for t in tensors]
    packed, strided = [], set()
    if not all(map(get.is_contiguous, tensors)):
        tensors = list(tensors)
        for i, t in enumerate(tensors):
            if t.is_contiguous():
                continue
            dense, overlapping = _layout(t)
            if overlapping and write:
                raise ValueError("a gradient shares memory with itself (an expanded view): "
                                 "it cannot be scaled in place")
            if not dense:
                strided.add(i)
        if write and strided:
            _refuse_sharing(tensors, strided)
        for i in strided:
            t, tensors[i] = tensors[i], tensors[i].detach().contiguous()
            packed.append((t, tensors[i]))
    rows = [0] * (3 * n)
    rows[0::3] = list(map(get.data_ptr, tensors))
    rows[1::3] = list(map(get.numel, tensors))
    rows[2::3] = codes
    table = array("q", rows)
    if write:
        rc = _lib.lib().scao_grads_overlap(table.buffer_info()[0], n)
        if rc == 1:
            raise ValueError(SHARED)
        _lib.check(rc, "scao_grads_overlap")
    if not tensors[0].is_cuda:
        raise RuntimeError("scao_b200: gradients must be CUDA tensors (no CPU path)")
    return table, tensors, packed, index


def _kind(norm_type):
    kind = _KIND.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type must be 1, 2 or inf, not {norm_type}")
    return kind


def _max_norm(max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be at least 0, not {max_norm}")
    return max_norm


def _grads(parameters):
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return [g for g in map(_GRAD, parameters) if g is not None]


def _refuse_nonfinite(total, norm_type):
    if not bool(torch.isfinite(total)):
        raise RuntimeError(f"the total norm of order {norm_type} of the gradients is not finite, "
                           "so they cannot be clipped; pass error_if_nonfinite=False to scale "
                           "by it all the same")


def _outputs(tensors):
    """(the norm, the workspace) of the gradients."""
    t, size = tensors[0], _lib.lib().scao_grad_norm_workspace_bytes(len(tensors))
    return t.new_empty((), dtype=torch.float32), t.new_empty(size, dtype=torch.uint8)


def _finish(grads, packed):
    """What an in-place operation on the gradients ends with."""
    for g, copy in packed:
        with torch.no_grad():
            g.copy_(copy)
    try:
        torch.autograd.graph.increment_version(grads)
    except RuntimeError:            # inference tensors have no version
        torch.autograd.graph.increment_version([g for g in grads if not g.is_inference()])


def get_total_norm(tensors, norm_type=2.0, error_if_nonfinite=False):
    """The norm of all values of ``tensors`` (a tensor or an iterable) as if they were
    one vector: a float32 scalar on their device.  ``norm_type`` is 1, 2 or inf;
    no tensors give 0, a NaN anywhere gives NaN.  ``error_if_nonfinite`` waits for the
    GPU and raises where the norm is inf or NaN."""
    kind = _kind(norm_type)
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    n = len(tensors)
    table, kept, _, index = _table(tensors, write=False)
    total, ws = _outputs(kept)
    _launch("scao_grad_norm", index, _lib.lib().scao_grad_norm, table.buffer_info()[0], n, kind,
            ws.data_ptr(), total.data_ptr())
    if error_if_nonfinite:
        _refuse_nonfinite(total, norm_type)
    return total


def clip_grads_with_norm_(parameters, max_norm, total_norm):
    """Scales the gradients of ``parameters`` (a tensor or an iterable) in place by
    min(1, max_norm / (total_norm + 1e-6)); ``total_norm`` is a scalar tensor on their
    device, as ``get_total_norm`` returns it (or reduced over ranks)."""
    max_norm = _max_norm(max_norm)
    grads = _grads(parameters)
    if not grads or max_norm == math.inf:
        return
    table, kept, packed, index = _table(grads, write=True)
    if total_norm.numel() != 1 or total_norm.get_device() != index:
        raise ValueError("total_norm must be one number on the gradients' device")
    total = total_norm.detach().to(torch.float32)
    _launch("scao_grad_clip", index, _lib.lib().scao_grad_clip, table.buffer_info()[0], len(grads),
            max_norm, total.data_ptr())
    _finish(grads, packed)


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Clips the gradients of ``parameters`` (a tensor or an iterable) in place so that
    their norm, taken over all of them as one vector, is at most ``max_norm``:
    g <- g min(1, max_norm / (norm + 1e-6)).  Returns the norm before clipping, a
    float32 scalar on their device.  ``norm_type`` is 1, 2 or inf; an infinite
    ``max_norm`` leaves the gradients as they are; a norm that is NaN makes every
    gradient NaN unless ``error_if_nonfinite``, which waits for the GPU and raises
    before anything is scaled.  Two gradients that share memory are refused."""
    kind, max_norm = _kind(norm_type), _max_norm(max_norm)
    grads = _grads(parameters)
    if not grads:
        return torch.tensor(0.0)
    if max_norm == math.inf:
        return get_total_norm(grads, norm_type, error_if_nonfinite)
    n, L = len(grads), _lib.lib()
    table, kept, packed, index = _table(grads, write=True)
    at = table.buffer_info()[0]
    total, ws = _outputs(kept)
    if error_if_nonfinite:
        _launch("scao_grad_norm", index, L.scao_grad_norm, at, n, kind, ws.data_ptr(), total.data_ptr())
        _refuse_nonfinite(total, norm_type)
        _launch("scao_grad_clip", index, L.scao_grad_clip, at, n, max_norm, total.data_ptr())
    else:
        _launch("scao_grad_norm_clip", index, L.scao_grad_norm_clip, at, n, kind, max_norm, ws.data_ptr(),
                total.data_ptr())
    _finish(grads, packed)
    return total
