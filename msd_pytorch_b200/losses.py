"""Losses that work on a linear layer's input instead of its output.

``linear_cross_entropy`` is the final 1x1 layer, log-softmax and negative log-likelihood of a
segmentation network (msd_segmentation_model.py:64-66 and msd_module.py:60-88 of the reference)
as one operator: the logits, ``labels`` values per voxel, are formed tile by tile on the chip and
never stored.  It serves a large vocabulary over rows of features as well.
"""
import array
import functools

import torch
import torch.autograd.forward_ad as fwAD
from torch.autograd.function import once_differentiable

from . import _lib

REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _features(x):
    """``(batch, channels, voxels, stride_batch, stride_channel, stride_voxel)`` of features
    ``[N, C, *spatial]`` or rows ``[T, C]``; None if the spatial axes have no common stride."""
    if x.dim() == 2:
        return 1, x.shape[1], x.shape[0], 0, x.stride(1), x.stride(0)
    if x.is_contiguous() and x.numel():
        n, c = x.shape[:2]
        voxels = x.numel() // (n * c)
        if voxels > 1:
            return n, c, voxels, c * voxels, voxels, 1
    voxels, stride = 1, None
    for size, st in zip(reversed(x.shape[2:]), reversed(x.stride()[2:])):
        if size == 1:
            continue
        if stride is None:
            stride = st
        elif st != voxels * stride:
            return None
        voxels *= size
    return x.shape[0], x.shape[1], voxels, x.stride(0), x.stride(1), 1 if stride is None else stride


def _describe(x, geometry):
    f = _lib.MsdFeatures()
    f.data = x.data_ptr()
    f.batch, f.channels, f.voxels, f.stride_batch, f.stride_channel, f.stride_voxel = geometry
    return f


@functools.lru_cache(maxsize=1024)
def _sizes(code, geometry, weight_alignment, labels):
    """``(single pass, bytes left to the backward call, scratch bytes forward, backward)`` of a shape."""
    features = _lib.MsdFeatures()
    features.data = 256
    features.batch, features.channels, features.voxels, features.stride_batch, features.stride_channel, features.stride_voxel = geometry
    weight = 256 + weight_alignment  # the library asks for its alignment only
    return (bool(_lib.lib.msd_linear_xent_single_pass(code, features, labels)), _lib.lib.msd_linear_xent_saved_bytes(code, features, weight, labels),
            _lib.lib.msd_linear_xent_workspace_bytes(code, features, weight, labels, 0),
            _lib.lib.msd_linear_xent_workspace_bytes(code, features, weight, labels, 1))


def _scratch(op_bytes, device):
    """Scratch of one call, from the caching allocator: a captured graph gets memory of its own."""
    return torch.empty(op_bytes, dtype=torch.uint8, device=device)


def _check(input, weight, bias, target, reduction):
    if reduction not in REDUCTIONS:
        raise ValueError("linear_cross_entropy: the reduction must be one of %s, got %r" % (sorted(REDUCTIONS), reduction))
    if not input.is_cuda:
        raise RuntimeError("linear_cross_entropy: expected CUDA tensors (there is no CPU implementation)")
    dtype, device = input.dtype, input.device
    _lib.loss_dtype_code(dtype)
    shape, wshape = input.shape, weight.shape
    if len(shape) < 2:
        raise RuntimeError("linear_cross_entropy: expected features [N, C, *spatial] or [T, C], got %d dimension(s)" % len(shape))
    if len(wshape) < 2 or wshape[1] != shape[1] or any(s != 1 for s in wshape[2:]):
        raise RuntimeError("linear_cross_entropy: expected a weight [labels, %d] (or a 1x1 kernel of these channels), got %s" % (shape[1], tuple(wshape)))
    if wshape[0] < 1 or wshape[1] < 1:
        raise RuntimeError("linear_cross_entropy: expected at least one label and one channel")
    if target.dim() != len(shape) - 1 or target.shape[0] != shape[0] or target.shape[1:] != shape[2:]:
        raise RuntimeError("linear_cross_entropy: expected a target of shape %s, got %s" % ((shape[0], *shape[2:]), tuple(target.shape)))
    if target.dtype != torch.int64:
        raise RuntimeError("linear_cross_entropy: expected int64 targets, got %s" % target.dtype)
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != wshape[0]):
        raise RuntimeError("linear_cross_entropy: expected a bias of %d values, got %s" % (wshape[0], tuple(bias.shape)))
    if weight.dtype != dtype or (bias is not None and bias.dtype != dtype):
        raise RuntimeError("linear_cross_entropy: expected all tensors to have the same scalar type")
    for t in (weight, bias, target):
        if t is not None and t.device != device:
            raise RuntimeError("linear_cross_entropy: expected all tensors on %s, got one on %s" % (device, t.device))


def _index(ignore_index):
    index = int(ignore_index)
    if not -2 ** 63 <= index < 2 ** 63:
        raise ValueError("linear_cross_entropy: ignore_index must be a 64-bit integer, got %d" % index)
    return index


def xent_forward_(x, geometry, weight, bias, target, ignore_index, reduction, keep):
    """``(loss, saved)`` through the C ABI; the arguments have passed the checks and are dense."""
    dev = x.device
    code = _lib.loss_dtype_code(x.dtype)
    features = _describe(x, geometry)
    loss = torch.empty(target.shape if reduction == "none" else (), dtype=torch.float32, device=dev)
    w = weight.data_ptr()
    _, kept, scratch, _ = _sizes(code, geometry, w % 16, weight.shape[0])
    saved = _scratch(kept, dev) if keep else None
    ws = _scratch(scratch, dev)
    _lib.check(_lib.lib.msd_linear_xent_forward(code, features, w, None if bias is None else bias.data_ptr(), target.data_ptr(),
                                                weight.shape[0], ignore_index, REDUCTIONS[reduction], loss.data_ptr(),
                                                None if saved is None else saved.data_ptr(), kept, ws.data_ptr(), scratch, dev.index,
                                                _lib.stream_of(dev)))
    return loss, saved


def xent_backward_(x, geometry, weight, bias, target, ignore_index, reduction, saved, grad_loss, grad_x, grad_x_geometry, grad_weight, grad_bias):
    """Writes the wanted gradients (None: not wanted)."""
    dev = x.device
    code = _lib.loss_dtype_code(x.dtype)
    features = _describe(x, geometry)
    gx = None if grad_x is None else _describe(grad_x, grad_x_geometry)
    scratch = _sizes(code, geometry, weight.data_ptr() % 16, weight.shape[0])[3]
    ws = _scratch(scratch, dev)
    _lib.check(_lib.lib.msd_linear_xent_backward(code, features, weight.data_ptr(), None if bias is None else bias.data_ptr(), target.data_ptr(),
                                                 weight.shape[0], ignore_index, REDUCTIONS[reduction], saved.data_ptr(), saved.numel(), grad_loss.data_ptr(), gx,
                                                 None if grad_weight is None else grad_weight.data_ptr(),
                                                 None if grad_bias is None else grad_bias.data_ptr(), ws.data_ptr(), ws.numel(), dev.index,
                                                 _lib.stream_of(dev)))


def xent_step_(x, geometry, weight, bias, target, ignore_index, reduction, grad_x, grad_x_geometry, grad_weight, grad_bias):
    """``(loss, saved)``, and the wanted gradients written for an upstream gradient of 1."""
    dev = x.device
    code = _lib.loss_dtype_code(x.dtype)
    features = _describe(x, geometry)
    gx = None if grad_x is None else _describe(grad_x, grad_x_geometry)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    _, kept, _, scratch = _sizes(code, geometry, weight.data_ptr() % 16, weight.shape[0])
    saved = _scratch(kept, dev)
    ws = _scratch(scratch, dev)
    _lib.check(_lib.lib.msd_linear_xent_step(code, features, weight.data_ptr(), None if bias is None else bias.data_ptr(), target.data_ptr(),
                                             weight.shape[0], ignore_index, REDUCTIONS[reduction], loss.data_ptr(), saved.data_ptr(), saved.numel(), gx,
                                             None if grad_weight is None else grad_weight.data_ptr(),
                                             None if grad_bias is None else grad_bias.data_ptr(), ws.data_ptr(), ws.numel(), dev.index,
                                             _lib.stream_of(dev)))
    return loss, saved


def single_pass(x, geometry, labels):
    """Whether :func:`xent_step_` takes these features."""
    return _sizes(_lib.loss_dtype_code(x.dtype), geometry, 0, labels)[0]


def _empty_gradient(x, x_geometry):
    """``(tensor, geometry)`` for the gradient of features: in their own layout, or dense where that
    has no geometry or voxels side by side would be lost."""
    grad = torch.empty_like(x)
    geometry = x_geometry if grad.stride() == x.stride() else _features(grad)
    if geometry is None or (x_geometry[5] == 1 and geometry[5] != 1):
        grad = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        geometry = _features(grad)
    return grad, geometry


def capturing(x):
    """Whether work on the current stream, and so on ``x``, is being captured into a graph."""
    return x.is_cuda and torch.cuda.is_current_stream_capturing()


def scale_(tensors, factor):
    """Multiplies dense tensors in place with the float32 value of ``factor`` (0-dimensional, on the device)."""
    table = array.array("q")
    for t in tensors:
        p = t.data_ptr()
        table.extend((p, p, t.numel(), _lib.GRAD_DTYPES[t.dtype]))
    spans = (_lib.MsdSpan * len(tensors)).from_buffer(table)
    dev = factor.device
    _lib.check(_lib.lib.msd_scale_tensors(spans, len(tensors), factor.data_ptr(), dev.index, _lib.stream_of(dev)))


def _has_tangent(*tensors):
    """Whether one of the tensors carries a forward-mode derivative."""
    return fwAD._current_level >= 0 and any(t is not None and fwAD.unpack_dual(t).tangent is not None for t in tensors)


def _operands(input, weight, bias, target):
    """The arguments as the library takes them, and the features' geometry."""
    geometry = _features(input)
    if geometry is None:
        input = input.contiguous()
        geometry = _features(input)
    return input, weight.contiguous(), None if bias is None else bias.contiguous(), target.contiguous(), geometry


def _saved_for(layout, input, geometry, weight, bias, target, ignore_index, reduction, saved):
    """What the forward call left for these operands; computed again if its operands lay differently in
    memory (``layout``: their geometry and the weight's alignment, on which kernel and contents depend)."""
    if layout == (geometry, weight.data_ptr() % 16):
        return saved.contiguous()
    return xent_forward_(input, geometry, weight, bias, target, ignore_index, reduction, True)[1]


class LinearCrossEntropyFunction(torch.autograd.Function):
    """With few labels over float32 images or volumes the gradients are computed in the forward pass,
    with the loss: x, which everything is bound by, is then read once instead of twice.  The
    backward pass multiplies them with the upstream gradient (nothing to do for 1) and hands
    them out; a second backward pass of a kept graph computes them again, and so does one that is captured
    when the forward pass was not (its replays would multiply the same values again and again)."""

    @staticmethod
    def forward(ctx, input, weight, bias, target, ignore_index, reduction):
        input, weight, bias, target, geometry = _operands(input, weight, bias, target)
        need = ctx.needs_input_grad
        ctx.grads = None
        if reduction != "none" and single_pass(input, geometry, weight.shape[0]):
            grad_x, grad_geometry = _empty_gradient(input, geometry) if need[0] else (None, None)
            grad_weight = torch.empty_like(weight) if need[1] else None
            grad_bias = torch.empty_like(bias) if bias is not None and need[2] else None
            loss, saved = xent_step_(input, geometry, weight, bias, target, ignore_index, reduction, grad_x, grad_geometry, grad_weight, grad_bias)
            ctx.grads, ctx.captured = (grad_x, grad_weight, grad_bias), capturing(input)
        else:
            loss, saved = xent_forward_(input, geometry, weight, bias, target, ignore_index, reduction, True)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        ctx.layout = geometry, weight.data_ptr() % 16
        ctx.save_for_backward(input, weight, bias, target, saved)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        input, weight, bias, target, saved = ctx.saved_tensors
        grads, ctx.grads = ctx.grads, None
        if grads is not None and (ctx.captured or not capturing(input)):
            scale_([g for g in grads if g is not None], grad_loss)
            return (*grads, None, None, None)
        # hooks on saved tensors may hand them back in another layout
        input, weight, bias, target, geometry = _operands(input, weight, bias, target)
        saved = _saved_for(ctx.layout, input, geometry, weight, bias, target, ctx.ignore_index, ctx.reduction, saved)
        need = ctx.needs_input_grad
        grad_x, grad_geometry = _empty_gradient(input, geometry) if need[0] else (None, None)
        grad_weight = torch.empty_like(weight) if need[1] else None
        grad_bias = torch.empty_like(bias) if bias is not None and need[2] else None
        xent_backward_(input, geometry, weight, bias, target, ctx.ignore_index, ctx.reduction, saved, grad_loss.contiguous(), grad_x, grad_geometry,
                       grad_weight, grad_bias)
        return grad_x, grad_weight, grad_bias, None, None, None


def linear_cross_entropy(input, weight, bias, target, ignore_index=-100, reduction="mean"):
    """Cross entropy of ``input @ weight.T + bias`` against ``target``, without storing the logits.

    ``input``: features ``[N, C, *spatial]`` (images, volumes) or ``[T, C]`` (rows), float32,
    bfloat16 or float16, any strides.  ``weight``: ``[labels, C]``, or the ``[labels, C, 1, ...]``
    of a 1x1 convolution.  ``bias``: ``[labels]`` or None.  ``target``: int64 labels of the input's
    shape without the channel axis; ``ignore_index`` leaves a token out of the loss and all
    gradients, whatever its features hold.  ``reduction``: "mean" (over the tokens that count),
    "sum" or "none".

    The loss is float32 for every input type: products of bfloat16 and float16 values are exact, those of
    float32 values are off by less than their own rounding (magnitudes below 1e-32 count as up to 2^-126 less),
    sums, exponentials and logarithms are float32.  Gradients have their tensors' types and are the
    same bits in every run.  With bfloat16 and float16 features the softmax gradient of a token
    (probability minus one for its label) is rounded to that type before it is multiplied with weight and
    features, unless there are at most 16 labels over images or volumes; float16 holds it down to 2^-38 of the
    upstream gradient, and in three pieces of 8 bits for reduction "none".  As in ``torch.nn.functional.cross_entropy`` a mean over no tokens is
    NaN; a target that names no label makes the loss and the gradients that its token reaches NaN
    instead of ending the process."""
    _check(input, weight, bias, target, reduction)
    ignore_index = _index(ignore_index)
    wanted = torch.is_grad_enabled() and (input.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad))
    if not wanted and not _has_tangent(input, weight, bias):  # a tangent goes to autograd, which refuses it
        input, weight, bias, target, geometry = _operands(input, weight, bias, target)
        return xent_forward_(input, geometry, weight, bias, target, ignore_index, reduction, False)[0]
    return LinearCrossEntropyFunction.apply(input, weight, bias, target, ignore_index, reduction)
