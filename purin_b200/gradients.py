"""Global gradient norm over many tensors, and clipping.

Gradients through a projection jump where its active set changes, so training through
the layer clips them.  Both functions read all tensors in one launch, whatever their
number, sizes and types, and never wait for the device.
"""

from __future__ import annotations

import torch

from purin_b200 import _native_ops as _ops


def _tensors(what, tensors):
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        raise ValueError(f"{what}: no tensors")
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: expected tensors, got {type(t).__name__}")
    _ops.require_cuda(what, *tensors)
    for t in tensors:
        _ops.require_floating(what, "tensors", t)
    return tensors


def _dense(t):
    """True if the tensor's elements fill a range of memory (in any order of dimensions)."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((st, si) for st, si in zip(t.stride(), t.shape) if si != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def gradient_norm(tensors):
    """``sqrt(sum of x^2)`` over all elements of ``tensors``, a 0-d tensor on their device.

    float32, or float64 if one of the tensors is; partial sums are joined in float64.  Not
    differentiable: the norm of tensors that need a gradient raises in a backward.
    """
    tensors = _tensors("gradient_norm", tensors)
    if not all(map(_dense, tensors)):
        tensors = [t if _dense(t) else t.contiguous() for t in tensors]
    return _ops.load().gradients(tensors, tensors, False, 0.0, 0.0)


def clip_gradients(tensors, max_norm, *, out=None, eps=1e-6):
    """Scale ``tensors`` by ``min(1, max_norm / (norm + eps))``; returns the norm.

    In place, or into ``out`` (tensors of the same shapes and types); no output may share
    memory with another tensor.  Autograd records neither the scaling nor the norm.

    The norm is that before clipping.  If it is NaN, so are all clipped values; an infinite value
    makes the norm infinite, itself NaN and the finite values zero: ask ``isfinite`` of the norm to
    skip a step.  The values are scaled by the norm in float64, so of finite values whose norm
    passes float32 the clipped ones are right and only the returned norm is infinite.
    """
    what = "clip_gradients"
    tensors = _tensors(what, tensors)
    max_norm, eps = float(max_norm), float(eps)
    if not max_norm >= 0.0:
        raise ValueError(f"{what}: max_norm must be nonnegative, got {max_norm}")
    if not eps >= 0.0:
        raise ValueError(f"{what}: eps must be nonnegative, got {eps}")
    if out is None:
        outs = tensors
        fits = [_dense(t) for t in tensors]
    else:
        outs = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(outs) != len(tensors):
            raise ValueError(f"{what}: {len(tensors)} tensors but {len(outs)} outputs")
        for t, o in zip(tensors, outs):
            if not t.is_same_size(o) or o.dtype != t.dtype or o.get_device() != t.get_device():
                raise ValueError(f"{what}: an output differs from its tensor in shape, type or device")
        fits = [t.is_contiguous() and o.is_contiguous() or _dense(t) and t.stride() == o.stride()
                for t, o in zip(tensors, outs)]
    if all(fits):
        return _ops.load().gradients(tensors, outs, True, max_norm, eps)
    # Tensors with gaps, or laid out differently from their outputs, go through copies.
    with torch.no_grad():
        dense = [t if f else t.contiguous() for t, f in zip(tensors, fits)]
        made = [o if f else torch.empty_like(d) for o, d, f in zip(outs, dense, fits)]
        norm = _ops.load().gradients(dense, made, True, max_norm, eps)
        for o, m, f in zip(outs, made, fits):
            if not f:
                o.copy_(m)
    return norm
