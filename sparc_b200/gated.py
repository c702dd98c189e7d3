"""Gated linear recurrence h_t = a_t h_{t-1} + sqrt(1 - a_t^2) s(write_t) x_t with
a_t = exp(-exp(nu_log) s(retention_t)), s the logistic function: per channel a retention rate (as
SPARCMixer's nu_log) that every token's retention gate scales, and an input that its write gate
scales and sqrt(1 - a_t^2) keeps at the state's own variance. The scans of `real.py` take a and
b ready-made; here the gates are part of the kernels, and so are the gradients through them.

``gated_scan`` is the training and prefill form, ``gated_scan_step`` the one-token form for
decoding. x and the two gates are float32 or bfloat16 (one dtype), [B, T, D] with adjacent
channels in any batch and token strides: the three may be columns of one projection, and are read
in place. nu_log and the states are float32, and so is the arithmetic.

``segment_pos`` ([B, T] integers, as SPARCMixer's) restarts the recurrence at every token whose
position is 0 (packed sequences): nothing of the earlier segment is kept, not its infinities or
NaN either. The token's write keeps its factor sqrt(1 - a_t^2).

Both are operators of csrc_torch/train_ops.cpp, which checks the arguments (shapes: ValueError,
dtypes: TypeError, a forward-mode tangent: NotImplementedError, a tensor that is not on the GPU:
RuntimeError) and calls the kernels of csrc/gated_scan.cu on the current stream.
"""
from __future__ import annotations

import torch

from . import torch_ops


def gated_scan(x: torch.Tensor, retention_gate: torch.Tensor, write_gate: torch.Tensor, nu_log: torch.Tensor,
               state: torch.Tensor | None = None, segment_pos: torch.Tensor | None = None,
               return_last: bool = False):
    """The recurrence over [B, T, D]: y [B, T, D] in x's dtype, or with `return_last` (y, last)
    with the state after the last token, float32 [B, D]. Starts from `state` ([B, D]) or zero.
    Differentiable (once) with respect to x, the gates, nu_log and the state, through y and last."""
    out = torch_ops.call("gated_scan", x, retention_gate, write_gate, nu_log, state, segment_pos, return_last)
    return tuple(out) if return_last else out[0]


def gated_scan_step(x: torch.Tensor, retention_gate: torch.Tensor, write_gate: torch.Tensor, nu_log: torch.Tensor,
                    state: torch.Tensor, segment_pos: torch.Tensor | None = None):
    """One token: x and the gates [B, D], the state [B, D]; returns (y [B, D] in x's dtype, the new
    state, float32). Without autograd, as ``sparc_decode_step``; a length-1 ``gated_scan`` with the
    state is the differentiable form. `segment_pos` ([B]) restarts the rows whose position is 0."""
    return torch_ops.call("gated_scan_step", x, retention_gate, write_gate, nu_log, state, segment_pos)
