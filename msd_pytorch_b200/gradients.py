"""The global norm of many gradient tensors, and clipping by it.

The reference's training step has no clipping (``learn``, msd_model.py:183-196); a network that
is trained with it needs the norm over some hundred small tensors every step.  All tensors of a
device go through one call of the C ABI whatever their number, sizes and types.
"""
import array
from operator import attrgetter

import torch

from . import _lib
from .losses import _has_tangent, _scratch

NORM_TYPES = {2.0: 0, float("inf"): 1}


# A training step asks for some hundred small tensors every time: attributes are gathered one at a
# time by mapping the methods themselves, at 0.04 us each.
_Tensor = torch.Tensor
_dtype_of = attrgetter("dtype")


def _norm_code(norm_type):
    code = NORM_TYPES.get(float(norm_type))
    if code is None:
        raise ValueError("the norm type must be 2 or inf, got %r" % (norm_type,))
    return code


def _dense(t):
    """Whether the elements of ``t`` fill one stretch of memory, each place once."""
    if t.is_contiguous():
        return True
    expect = 1
    for st, size in sorted((st, size) for st, size in zip(t.stride(), t.shape) if size != 1):
        if st != expect:
            return False
        expect = st * size
    return True


def _check_list(tensors, op):
    """Device and types of the tensors."""
    if _has_tangent(*tensors):
        raise RuntimeError("%s: forward-mode derivatives are not offered" % op)
    indices = set(map(_Tensor.get_device, tensors))
    if min(indices) < 0:
        raise RuntimeError("%s: expected CUDA tensors (there is no CPU implementation)" % op)
    dtypes = list(map(_dtype_of, tensors))
    for dtype in set(dtypes):
        if dtype not in _lib.GRAD_DTYPES:
            raise RuntimeError("%s: expected float32, float64, bfloat16 or float16 tensors, got %s" % (op, dtype))
    if len(indices) > 1:
        raise RuntimeError("%s: expected all tensors on one device, got devices %s" % (op, sorted(indices)))
    return tensors[0].device, dtypes


def _spans(pointers, out_pointers, sizes, dtypes):
    """The ``msd_span_t`` array of dense tensors: data, out, size and (32-bit) type of each."""
    n = len(pointers)
    table = array.array("q", bytes(32 * n))
    table[0::4] = array.array("q", pointers)
    table[1::4] = array.array("q", out_pointers)
    table[2::4] = array.array("q", sizes)
    if dtypes.count(dtypes[0]) == n:
        table[3::4] = array.array("q", (_lib.GRAD_DTYPES[dtypes[0]],)) * n
    else:
        table[3::4] = array.array("q", map(_lib.GRAD_DTYPES.__getitem__, dtypes))
    return (_lib.MsdSpan * n).from_buffer(table)


def _norm_tensor(dtypes, dev):
    wide = dtypes.count(torch.float64) == len(dtypes)
    norm = torch.empty((), dtype=torch.float64 if wide else torch.float32, device=dev)
    return norm, (None, norm.data_ptr()) if wide else (norm.data_ptr(), None)


def total_norm(tensors, norm_type=2.0):
    """The norm of all values of ``tensors`` taken together, as a 0-dimensional tensor on their
    device (float32; float64 if every tensor is float64).  ``norm_type``: 2 or inf.  A number to look at
    or to clip by: no gradient flows through it."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    code = _norm_code(norm_type)
    if not tensors:
        return torch.zeros(())
    dev, dtypes = _check_list(tensors, "total_norm")
    data = tensors if all(map(_Tensor.is_contiguous, tensors)) else [t if _dense(t) else t.contiguous() for t in tensors]
    pointers = list(map(_Tensor.data_ptr, data))
    spans = _spans(pointers, pointers, list(map(_Tensor.numel, data)), dtypes)
    norm, (n32, n64) = _norm_tensor(dtypes, dev)
    ws = _scratch(_lib.lib.msd_grad_norm_workspace_bytes(len(data)), dev)
    _lib.check(_lib.lib.msd_grad_norm(spans, len(data), code, n32, n64, ws.data_ptr(), ws.numel(), dev.index, _lib.stream_of(dev)))
    return norm


def clip_norm_(tensors, max_norm, norm_type=2.0, error_if_nonfinite=False, out=None):
    """Scales ``tensors`` by ``min(1, max_norm / (norm + 1e-6))``, where ``norm`` is their
    :func:`total_norm`, and returns the norm.  In place, or, with ``out``, into the tensors listed
    there, with ``tensors`` left as they are: same types and shapes (contiguous ones may differ in
    shape, slices of a flat buffer for instance), no overlap with the input other than being the
    same tensors.  A tensor that appears twice is refused: it would be scaled twice.

    Nothing waits for the GPU unless ``error_if_nonfinite`` is set, which raises a RuntimeError for a norm
    that is infinite or NaN and leaves the tensors unscaled."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    code = _norm_code(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("max_norm must be zero or more, got %r" % max_norm)
    if out is not None:
        out = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(out) != len(tensors):
            raise ValueError("clip_norm_: expected %d output tensors, got %d" % (len(tensors), len(out)))
    if not tensors:
        return torch.zeros(())
    dev, dtypes = _check_list(tensors, "clip_norm_")
    sizes = list(map(_Tensor.numel, tensors))
    dense = all(map(_Tensor.is_contiguous, tensors))
    if out is not None:
        out_dev, out_dtypes = _check_list(out, "clip_norm_")
        dense = dense and all(map(_Tensor.is_contiguous, out))
        if out_dev != dev:
            raise RuntimeError("clip_norm_: expected outputs on %s, got %s" % (dev, out_dev))
        if out_dtypes != dtypes or list(map(_Tensor.numel, out)) != sizes or not (dense or all(o.shape == t.shape for t, o in zip(tensors, out))):
            raise RuntimeError("clip_norm_: expected outputs of the tensors' types and sizes (and shapes, unless all are contiguous)")
    targets = tensors if out is None else out
    target_pointers = list(map(_Tensor.data_ptr, targets))
    if len(set(target_pointers)) != len(target_pointers):
        seen = [p for p, n in zip(target_pointers, sizes) if n]  # empty tensors have no place of their own
        if len(set(seen)) != len(seen):
            raise RuntimeError("clip_norm_: the same tensor appears twice")
    if error_if_nonfinite:
        norm = total_norm(tensors, norm_type)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError("clip_norm_: the total norm of order %s is not finite (%s), so the tensors were not clipped" % (float(norm_type), norm.item()))
    data, written = tensors, targets
    if not dense:
        # values in one stretch of memory each, outputs laid out like their inputs
        data = [t if _dense(t) else t.contiguous() for t in tensors]
        written = [o if (o is t and d is t) or (_dense(o) and o.stride() == d.stride()) else torch.empty_strided(d.shape, d.stride(), dtype=d.dtype, device=dev)
                   for t, d, o in zip(tensors, data, targets)]
        target_pointers = list(map(_Tensor.data_ptr, written))
    spans = _spans(target_pointers if data is written else list(map(_Tensor.data_ptr, data)), target_pointers, sizes, dtypes)
    norm, (n32, n64) = _norm_tensor(dtypes, dev)
    ws = _scratch(_lib.lib.msd_grad_norm_workspace_bytes(len(data)), dev)
    with torch.no_grad():
        _lib.check(_lib.lib.msd_clip_grad_norm(spans, len(data), max_norm, code, n32, n64, ws.data_ptr(), ws.numel(), dev.index, _lib.stream_of(dev)))
        if written is not targets:
            for w, o in zip(written, targets):
                if w is not o:
                    o.copy_(w)
        # written by address: graphs that saved one of them have to know
        torch.autograd.graph.increment_version(targets)
    return norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """:func:`clip_norm_` of the gradients of ``parameters`` (those that have one), in place: the
    calling convention of ``torch.nn.utils.clip_grad_norm_``, but each parameter at most once."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    return clip_norm_([p.grad for p in parameters if p.grad is not None], max_norm, norm_type, error_if_nonfinite)
