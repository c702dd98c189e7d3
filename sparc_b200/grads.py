"""The global norm of a model's gradients, and clipping by it, on the kernels of csrc/grad_norm.cu:
two launches for all tensors together, no copy to the host. In data-parallel training it follows
the gradient exchange of `ddp.py`: every rank then holds the same sums, and gets the same norm and
the same clipped gradients bit for bit.

    norm = sqrt(sum of g^2 over every element of every tensor)
    g   <- g min(1, max_norm / (norm + eps))

Gradients are float32 or bfloat16 CUDA tensors of one device. The norm is a float32 tensor with
one element, right also where a square would overflow or underflow in float32. A norm that is NaN
makes every gradient NaN; whether to skip such a step is the caller's decision.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib


def _check(tensors, what, like=None):
    """Shape checks first (ValueError), then dtypes (TypeError), then the device (no CPU path)."""
    for i, t in enumerate(tensors):
        if t.layout != torch.strided:
            raise TypeError(f"{what} expects dense tensors, got {t.layout}")
        if like is not None and (t.shape != like[i].shape or t.dtype != like[i].dtype):
            raise ValueError(f"{what} expects out to match the gradients' shapes and dtypes")
    for t in tensors:
        _lib.dtype_code(t.dtype)
    for t in tensors:
        _lib.require_cuda(t, "every gradient")
        if t.device != tensors[0].device:
            raise RuntimeError(f"{what} expects tensors of one device, got {tensors[0].device} and {t.device}")


def _call(grads, out, max_norm, eps):
    L = _lib.lib()
    n = len(grads)
    dev = grads[0].device
    norm = torch.empty((), dtype=torch.float32, device=dev)
    nbytes = L.sparc_grad_clip_workspace_bytes(n)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
    a = _lib.GradClipArgs((ctypes.c_void_p * n)(*[g.data_ptr() for g in grads]),
                          None if out is None else (ctypes.c_void_p * n)(*[o.data_ptr() for o in out]),
                          (ctypes.c_longlong * n)(*[g.numel() for g in grads]),
                          (ctypes.c_int * n)(*[_lib.dtype_code(g.dtype) for g in grads]), n, max_norm, eps,
                          norm.data_ptr(), ws.data_ptr(), nbytes)
    with _lib.on_device(dev):
        _lib.check(L.sparc_grad_clip(ctypes.byref(a), _lib.stream_handle(dev)), "sparc_grad_clip")
    return norm


@torch.no_grad()
def grad_norm(grads) -> torch.Tensor:
    """The norm of all elements of `grads` (an iterable of tensors) together: float32, one element."""
    grads = list(grads)
    if not grads:
        raise ValueError("grad norm expects at least one tensor")
    _check(grads, "grad norm")
    return _call([g.contiguous() for g in grads], None, 0.0, 0.0)


@torch.no_grad()
def clip_grads(grads, max_norm: float, out=None, eps: float = 1e-6) -> torch.Tensor:
    """Scale `grads` by min(1, max_norm / (norm + eps)) in place, or into the tensors `out` (same
    shapes and dtypes; the gradients then stay as they are); returns their norm before that.
    Every tensor may be given once, and no output may overlap another tensor."""
    grads = list(grads)
    if not grads:
        raise ValueError("clip grads expects at least one tensor")
    if not (max_norm >= 0.0 and eps >= 0.0):
        raise ValueError("max_norm and eps must not be negative")
    _check(grads, "clip grads")
    target = grads
    if out is not None:
        target = list(out)
        if len(target) != len(grads):
            raise ValueError("clip grads expects one output for each gradient")
        _check(target, "clip grads", grads)
        if target[0].device != grads[0].device:
            raise RuntimeError("clip grads expects out on the gradients' device")
    # the kernels take dense arrays: others go through a copy
    src = [g.contiguous() for g in grads]
    dst = [s if o is g and s is not g else o if o.is_contiguous() else torch.empty_like(s)
           for g, s, o in zip(grads, src, target)]
    norm = _call(src, dst, float(max_norm), float(eps))
    for d, o in zip(dst, target):
        if d is not o:
            o.copy_(d)
    return norm


def clip_grad_norm_(parameters, max_norm: float, eps: float = 1e-6) -> torch.Tensor:
    """Clip the gradients of `parameters` (a tensor or an iterable; those without a gradient are
    skipped, one given twice counts once) in place by their global norm; returns the norm."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = list({id(p): p.grad for p in parameters if p.grad is not None}.values())
    if not grads:
        return torch.tensor(0.0)
    return clip_grads(grads, max_norm, eps=eps)
