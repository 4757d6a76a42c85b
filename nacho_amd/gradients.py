"""What becomes of a step's gradients before they are used: their common norm, and clipping.

Tensors are float32, float16 or bfloat16 in any mixture, on one device; entries that are None
(parameters without a gradient) are passed over.  The squares are summed in float64, in a fixed
order.

Calls are asynchronous on torch's current stream, read nothing back and may be captured in a
graph.  There is no CPU fallback.  Neither has a gradient: a norm of tensors that require one
refuses its backward pass, both refuse tangents of forward mode, and clipping is no part of a history.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from .blocks import _MOST_SCALE, _TYPES, _call, _device_of, _has_derivatives


def _list(tensors, name):
    if isinstance(tensors, torch.Tensor):
        return [tensors]
    return list(tensors)


def _device(tensors):
    for t in tensors:
        if t is not None:
            return _device_of(t, "tensors[0]" if t is tensors[0] else "tensors")
    raise ValueError("tensors: expected at least one")


def _check(tensors, name, device, dtypes=_TYPES):
    for i, t in enumerate(tensors):
        if t is None:
            continue
        if _device_of(t, f"{name}[{i}]") != device:
            raise ValueError(f"operands on different devices: {device} and {t.device}")
        if t.layout != torch.strided:
            raise TypeError(f"{name}[{i}]: expected a strided tensor, got {t.layout}")
        if t.dtype not in dtypes:
            raise TypeError(f"{name}[{i}]: expected dtype {' or '.join(map(str, dtypes))}, got "
                            f"{t.dtype}")


def _dense(t):
    """Whether a tensor's elements are next to each other, in some order of its dimensions."""
    expected = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return t.numel() == 0
        expected *= size
    return True


def _norm(device, held, tensors):
    got = _call("grad_norm", device, held)
    if got is None:
        _check(tensors, "tensors", device)
        raise ValueError("gpu_grad_norm: refused operands")
    return got


class _GradNorm(torch.autograd.Function):
    """(Refuses tangents, as a function without jvp.)"""

    @staticmethod
    def forward(ctx, device, *held):
        return _norm(device, held, held)

    @staticmethod
    def backward(ctx, dnorm):
        raise RuntimeError("gpu_grad_norm has no gradient: detach the tensors or the norm")


def gpu_grad_norm(tensors) -> torch.Tensor:
    """The root of the sum of the squares of all elements of a tensor or of many, float32, on the
    device.  Not differentiable: of tensors that require a gradient, its backward pass raises."""
    tensors = _list(tensors, "tensors")
    device = _device(tensors)
    held = tuple(t for t in tensors if t is not None)
    if _has_derivatives(*held):
        _check(tensors, "tensors", device)
        return _GradNorm.apply(device, *held)
    return _norm(device, held, tensors)


def gpu_clip_grad_norm(tensors, max_norm: float, out=None) -> torch.Tensor:
    """Scale tensors (gradients, not the parameters that have them) so that their common norm is at
    most max_norm, and give the norm that they had (float32, on the device): every element times
    min(1, max_norm / (norm + 1e-6)).

    In place, or into the tensors of `out`, of the same shapes, each of its tensor's type or
    float32 (as an optimiser's own copies are).  A tensor that is written has to have its elements
    next to each other, in any order of its dimensions, and share no memory with another's.  A norm
    of infinity makes finite elements 0 and infinite ones no numbers; one that is no number makes
    all of them that.  max_norm may be infinity: nothing is scaled.  Not differentiable: what is
    written has the history that it had, and the norm none."""
    tensors = _list(tensors, "tensors")
    device = _device(tensors)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be 0 or more, got {max_norm}")
    limit = float(max_norm)
    if _MOST_SCALE < limit < float("inf"):
        raise ValueError(f"max_norm must be infinity or finite in float32, got {max_norm}")
    outs = tensors if out is None else _list(out, "out")
    if len(outs) != len(tensors) or any((a is None) != (b is None)
                                        for a, b in zip(tensors, outs)):
        raise ValueError(f"out: expected a tensor for each of the {len(tensors)}, got {len(outs)}")
    if forward_ad._current_level >= 0:
        for t in (*tensors, *outs):
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("gpu_clip_grad_norm has no jvp: tensors with tangents")
    got = _call("clip_grad_norm", device, tuple(t for t in tensors if t is not None),
                tuple(t for t in outs if t is not None), limit)
    if got is None:
        _refuse_clip(tensors, outs, device, out is None)
    return got


def _refuse_clip(tensors, outs, device, in_place):
    _check(tensors, "tensors", device)
    name = "tensors" if in_place else "out"
    for i, o in enumerate(outs):
        if o is not None and o.requires_grad and o.is_leaf:
            raise ValueError(f"{name}[{i}] is a leaf that requires a gradient: expected the "
                             "gradients (parameter.grad), not the parameters")
    for i, (t, o) in enumerate(zip(tensors, outs)):
        if t is None or (in_place and _dense(t)):
            continue
        if in_place:
            raise ValueError(f"tensors[{i}]: expected elements next to each other, got strides "
                             f"{t.stride()} of shape {tuple(t.shape)}")
        _check([o], f"out of tensors[{i}]", device, (t.dtype, torch.float32))
        if o.shape != t.shape:
            raise ValueError(f"out[{i}]: expected shape {tuple(t.shape)}, got {tuple(o.shape)}")
        if not _dense(o):
            raise ValueError(f"out[{i}]: expected elements next to each other, got strides "
                             f"{o.stride()} of shape {tuple(o.shape)}")
    raise ValueError("tensors that are written share memory")
