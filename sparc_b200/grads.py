"""The global norm of a model's gradients, and clipping by it, on the kernels of csrc/grad_norm.cu:
two launches for all tensors together, no copy to the host. In data-parallel training it follows
the gradient exchange of `ddp.py`: every rank then holds the same sums, and gets the same norm and
the same clipped gradients bit for bit.

    norm = sqrt(sum of g^2 over every element of every tensor)
    g   <- g min(1, max_norm / (norm + eps))

Gradients are float32 or bfloat16 CUDA tensors of one device. The norm is a float32 tensor with
one element, right also where a square would overflow or underflow in float32. A norm that is NaN
makes every gradient NaN; whether to skip such a step is the caller's decision. No gradient goes
through norm or scaling, and a tensor with a forward-mode tangent is refused (NotImplementedError).
"""
from __future__ import annotations

import torch

from . import torch_ops


def grad_norm(grads) -> torch.Tensor:
    """The norm of all elements of `grads` (an iterable of tensors) together: float32, one element."""
    return torch_ops.call("grad_clip", list(grads), [], False, 0.0, 0.0)


def clip_grads(grads, max_norm: float, out=None, eps: float = 1e-6) -> torch.Tensor:
    """Scale `grads` by min(1, max_norm / (norm + eps)) in place, or into the tensors `out` (same
    shapes and dtypes; the gradients then stay as they are); returns their norm before that.
    Every tensor may be given once, and no output may overlap another tensor."""
    grads = list(grads)
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError("clip grads expects one output for each gradient")
    return torch_ops.call("grad_clip", grads, out or [], True, max_norm, eps)


def clip_grad_norm_(parameters, max_norm: float, eps: float = 1e-6) -> torch.Tensor:
    """Clip the gradients of `parameters` (a tensor or an iterable; those without a gradient are
    skipped, one given twice counts once) in place by their global norm; returns the norm."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = list({id(p): p.grad for p in parameters if p.grad is not None}.values())
    if not grads:
        return torch.tensor(0.0)
    return clip_grads(grads, max_norm, eps=eps)
